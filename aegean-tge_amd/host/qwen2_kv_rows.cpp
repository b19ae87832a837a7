// The driver's layer call on rows of 16 bits (e4m3 caches).
#include "../csrc/tge_layer.h"
#include "qwen2_kv_handles.hpp"

namespace tge::models {

void Qwen2KvPath::layer_rows(int layer, const tge_append_rows_args& store,
                             const tge_attention_rows_args& attend, void* stream) {
  if (!begun_) throw std::runtime_error("layer: no step begun");
  if (layer < 0 || layer >= config_.layers) {
    throw std::invalid_argument("layer: layer out of range");
  }
  check(tge::layer_rows(batch_, pool_, layer, store, attend, stream), "layer");
}

}  // namespace tge::models

extern "C" {

int tge_qwen2_kv_layer_rows(tge_qwen2_kv* m, int layer, const tge_append_rows_args* store,
                            const tge_attention_rows_args* attend, void* stream) {
  if (!m || !store || !attend) return TGE_ERR_INVALID;
  return guarded([&] { m->impl.layer_rows(layer, *store, *attend, stream); });
}

}  // extern "C"
