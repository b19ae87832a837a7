// The e4m3 cache (pool format TGE_KV_E4M3): block layout, codec, plan records
// and kernel parameters, shared by the planner, the C ABI and the kernels.
//
// A page block is 16 tokens of one KV head at the block width W (64, 128 or
// 256 dims; dims past the head's own are zero codes): 16*W K codes, then 16*W
// V codes, one contiguous run of HBM, 4096 B at W = 128. The layer's blocks
// are followed by one bf16 pair (K scale, V scale) for each block. Every scale is 2^e with
// -15 <= e <= 7, so a stored value code * 2^e is exact in f16 and the
// matrix-core operands are made with one conversion for two values
// (v_cvt_scalef32_pk_f16_fp8).
//
// Order inside a part, chosen for v_mfma_f32_32x32x16_f16 with K as the A
// operand of S^T = K.Q^T and V^T as the A operand of O^T = V^T.P^T, where a
// lane (c = lane & 31, h = lane >> 5) of the score tile holds row c and the
// tokens 8b + 4h + e. Piece i of lane l sits at byte i*1024 + l*16:
//   K: lane = ((d/16)&3)*16 + t,  j = (d/64)*16 + (d&15)
//      (16 dims of one token lie together: two operands of 8 dims)
//   V: lane = (t/4)*16 + (d&15),  j = ((d/16)&1)*(W/8) + (d/32)*4 + (t&3)
//      (4 tokens of a dim, then the same of the dims 32 further on)
//   byte = (j/16)*1024 + lane*16 + j%16
// 16 lanes with 16 bytes each make up 256 contiguous bytes in either part, so
// the LDS reads of a copied block have no bank conflicts.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#define TGE_HD __host__ __device__
#else
#define TGE_HD
#endif

namespace tge {

constexpr int kE4m3MinExp = -15, kE4m3MaxExp = 7;
constexpr float kE4m3Max = 448.0f;

TGE_HD inline int e4m3_k_index(int t, int d) {
  const int lane = ((d >> 4) & 3) * 16 + t, j = (d >> 6) * 16 + (d & 15);
  return (j >> 4) * 1024 + lane * 16 + (j & 15);
}
TGE_HD inline int e4m3_v_index(int t, int d, int width) {
  const int lane = (t >> 2) * 16 + (d & 15), j = ((d >> 4) & 1) * (width >> 3) + (d >> 5) * 4 + (t & 3);
  return (j >> 4) * 1024 + lane * 16 + (j & 15);
}
constexpr int e4m3_block_bytes(int width) { return 2 * 16 * width; }

// The smallest exponent with m <= 448 * 2^e, within the stored range, for a
// non-negative m given by its bits (448 = 1.75 * 2^8; subnormals and zero
// come out at the lower end, infinity at the upper one).
TGE_HD inline int e4m3_exponent(uint32_t bits) {
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kE4m3MinExp ? kE4m3MinExp : e > kE4m3MaxExp ? kE4m3MaxExp : e;
}

// ---- plan records ----------------------------------------------------------
// The new rows of one session that fall into one page.
struct E4m3Tile {
  int page;
  int row;    // first row of k/v
  int slot;   // its slot in the page
  int count;  // rows
  int pos;    // position of the first row
  int pad[3];
};

// One piece of attention work: up to 32*rw rows of one (session, KV head)
// against a range of its pages. Row r is global row row0 + r of the group:
// query (row0 + r) / group, head kv_head*group + (row0 + r) % group.
struct E4m3Item {
  int kv_head;
  int page_begin;  // logical page range [page_begin, page_end)
  int page_end;
  int part;        // partial slot, or -1: the item writes the output
  int row0;
  int rows;
  int ctx;
  int q_row;
  int table_off;
  int merge;       // merge record of a split tile, or -1
  int rw;          // row-waves: 1, 2 or 4 waves of 32 rows; 4 / rw waves share the pages
  int once;        // 1: no other item reads these blocks (cache policy of the loads)
  int next;        // the workgroup's next item, or -1
  int pad[3];
};
static_assert(sizeof(E4m3Item) == 16 * sizeof(int), "E4m3Item is read as 16 ints");

// A cut tile: the last of its pieces to arrive merges them all.
struct E4m3Merge {
  int first_part;
  int n_parts;
  int rows;
  int row0;     // which tile it is: for checks of a plan (the kernel knows from
  int kv_head;  // the arriving piece)
  int q_row;
  int pad[2];
};

constexpr int kE4m3Rows = 128;  // rows of a tile at most

}  // namespace tge
