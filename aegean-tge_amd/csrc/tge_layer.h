// The driver's way into the C ABI's layer calls. Internal to libtge_kv.so.
#pragma once

#include "tge_kv.h"

namespace tge {

int layer_rows(const tge_batch* batch, tge_kv_pool* pool, int layer, const tge_append_rows_args& store,
               const tge_attention_rows_args& attend, void* stream);

}  // namespace tge
