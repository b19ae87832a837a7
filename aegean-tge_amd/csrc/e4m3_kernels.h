// Kernel parameters and launchers of the e4m3 cache. Internal to libtge_kv.so.
#pragma once

#include <hip/hip_runtime.h>

#include "e4m3_common.h"
#include "tge_records.h"

namespace tge {

// Rows of q, k, v and out: element type (enum tge_row_type) and elements
// between rows. Row bases and strides are multiples of 16 bytes.
struct E4m3Append {
  const void* k;
  const void* v;
  long k_stride, v_stride;
  int row_type;
  char* blocks;      // layer base
  uint32_t* scales;  // bf16 pair of each block
  const E4m3Tile* tiles;
  int n_tiles;
  int kv_heads;
  int dims;   // the head's dims
  int width;  // block width
  // bias + rotation (rope_cos null: rows are stored as they are)
  const void* q;
  void* q_out;
  long q_stride, q_out_stride;
  const RowRec* rows;
  int n_rows;
  int q_heads;
  const float* q_bias;
  const float* k_bias;
  const float* v_bias;
  const float* rope_cos;
  const float* rope_sin;
  int rope_fma;
};

struct E4m3Attn {
  const char* blocks;
  const uint32_t* scales;
  const E4m3Item* items;  // workgroup i starts with item i
  const int* tables;
  const E4m3Merge* merges;
  int* counters;  // arrivals of each merge record, zero between launches
  const void* q;
  void* out;
  long q_stride, out_stride;
  int row_type;
  int kv_heads;
  int group;
  int dims;
  float scale_log2;  // softmax scale * log2(e)
  float* part_o;     // [parts][part_rows][width]
  float* part_ml;    // [parts][part_rows][2]
  int part_rows;
};

struct E4m3Gather {
  const char* blocks;
  const uint32_t* scales;
  const int* table;  // device
  int count;
  int kv_heads;
  int dims;
  int width;
  uint8_t* k_rows;
  uint8_t* v_rows;
  uint16_t* k_scales;
  uint16_t* v_scales;
};

hipError_t launch_e4m3_append(const E4m3Append& p, hipStream_t stream);
hipError_t launch_e4m3_gather(const E4m3Gather& p, hipStream_t stream);
hipError_t launch_e4m3_attention(int width, int groups, const E4m3Attn& p, hipStream_t stream);
// Workgroups that a compute unit holds at once.
int e4m3_groups_per_cu(int width);

}  // namespace tge
