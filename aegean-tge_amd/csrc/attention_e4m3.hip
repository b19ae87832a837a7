// Attention over the e4m3 cache: decode, verification of drafted tokens and
// prompt chunks in one kernel.
//
// A workgroup is four waves. An item is a tile of 32*RW rows, (query, head)
// pairs of one session and KV head, against a range of the session's pages:
// RW waves hold 32 rows each, and 4/RW such groups share the pages, taking
// tiles of TP pages in turn. RW is 1 where rows are few (decode: every wave
// streams pages of its own, nothing waits for another wave), and larger where
// many rows meet the same pages (each page block is copied to LDS once for
// all waves of a group).
//
// Page blocks go from HBM straight to LDS (buffer_load ... lds, a contiguous
// KiB each) into a ring, and from there into matrix-core operands: per 32
// tokens (two pages) and wave
//   S^T = K.Q^T   v_mfma_f32_32x32x16_f16: lane (c, h) holds row c and tokens
//                 8b + 4h + e; K codes become f16 with their block's scale in
//                 one conversion for two values
//   online softmax in the log2 domain: a row's base is an integer and moves
//                 only when a score passes it by more than 8, so rescaling is
//                 rare and exact; weights are f16 (at most 2^8), their sum
//                 is taken from the rounded weights, in fp32
//   O^T += V^T.P^T  the same instruction: P is already in operand order, and
//                 V's order in the page gives lane (c, h) the same tokens
// No value crosses lanes until a tile ends.
#include "attn_common.h"
#include "e4m3_kernels.h"
#include "tge_kv.h"

namespace tge {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

#define MFMA32x32x16(a, b, c) __builtin_amdgcn_mfma_f32_32x32x16_f16((a), (b), (c), 0, 0, 0)

// Launch shape at a block width.
template <int W>
struct E4m3Cfg {
  static constexpr int BLOCK = e4m3_block_bytes(W);
  static constexpr int PER_CU = W > 128 ? 1 : W > 64 ? 2 : 3;  // workgroups (= waves per SIMD)
  static constexpr int TP(int rw) { return rw == 4 ? 4 : 2; }  // pages of a tile
  static constexpr int NB(int rw) { return rw == 1 ? 2 : 4; }  // ring slots of a group
  static constexpr int RING = 16 * BLOCK;                      // (4 / rw) * NB * TP blocks
  static_assert(4 * NB(1) * TP(1) == 16 && 2 * NB(2) * TP(2) == 16 && NB(4) * TP(4) == 16, "ring size");
};

template <int W>
struct E4m3Shared {
  alignas(16) char ring[E4m3Cfg<W>::RING];  // at a tile's end: the waves' accumulators
  int ids[kE4m3ItemPages];                  // the item's pages: block numbers
  uint32_t scales[kE4m3ItemPages];          // and their scale pairs
  long out_at[kE4m3Rows];                   // element offset of each row in out
  float ml[2][4][32];                       // per wave: base, sum
  float sum[kE4m3Rows];
  float base[kE4m3Rows];
  int flag;
};

// Eight codes (two dwords) times a power of two as eight f16.
__device__ __forceinline__ half8_t e4m3x8(uint32_t a, uint32_t b, float scale) {
  const half2_t x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, false);
  const half2_t y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, true);
  const half2_t z = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, false);
  const half2_t w = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, true);
  return half8_t{x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}

// Eight q values from element `at` times c, as f16.
__device__ __forceinline__ half8_t load_q8(const void* q, long at, int type, float c) {
  float x[8];
  if (type == TGE_ROWS_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(q) + at);
    const float4 a = p[0], b = p[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const u32x4_t w = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(q) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (type == TGE_ROWS_BF16) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const half2_t h = bitcast<half2_t>(w[i]);
        x[2 * i] = (float)h[0];
        x[2 * i + 1] = (float)h[1];
      }
    }
  }
  half8_t r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (_Float16)(x[i] * c);
  return r;
}

// Four outputs, rounded to nearest even for 16-bit rows.
__device__ __forceinline__ void store_out4(void* out, long at, int type, float4_t v) {
  if (type == TGE_ROWS_F32) {
    *reinterpret_cast<float4_t*>(static_cast<float*>(out) + at) = v;
  } else {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      b[i] = type == TGE_ROWS_BF16 ? bitcast<uint16_t>((__bf16)v[i]) : bitcast<uint16_t>((_Float16)v[i]);
    *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(out) + at) = u32x2_t{b[0] | b[1] << 16, b[2] | b[3] << 16};
  }
}

// Copy the page block `n` to LDS at `slot`.
template <int W, int POLICY>
__device__ __forceinline__ void fetch_block(char* slot, const char* blocks, int n, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BLOCK = E4m3Cfg<W>::BLOCK;
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(blocks + (size_t)n * BLOCK, BLOCK);
#pragma unroll
  for (int i = 0; i < BLOCK / 1024; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(slot + i * 1024), 16, i * 1024 + lane * 16, 0, 0,
                                             POLICY);
#endif
}

// A wave's rows against pages.
template <int W>
struct E4m3Rows {
  static constexpr int KS = W / 32;  // pieces of 16 dims a lane holds (two operands each)
  static constexpr int NT = W / 32;  // 32-dim output tiles
  half8_t q[KS][2];                  // row c, dims 32u + 16h + 8x ..
  f32x16_t o[NT];
  float base, thr, sum;              // of the row; `sum` over the lane's own tokens
  int lim;                           // the row's last visible position within the item
  int first_lim, last_lim;           // over the wave's rows (wave-uniform)

  // Tokens [16 * page, 16 * page + 32) from the two blocks at `slot`.
  __device__ __forceinline__ void pair(const char* slot, uint32_t sa, uint32_t sb, int page, int lane) {
    constexpr int BLOCK = E4m3Cfg<W>::BLOCK;
    const int c = lane & 31, h = lane >> 5;
    const float ks = __uint_as_float((c & 16 ? sb : sa) << 16);
    const char* kp = slot + (c >> 4) * BLOCK + h * 256 + (c & 15) * 16;
    f32x16_t s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = -base;
#pragma unroll
    for (int u = 0; u < KS; ++u) {
      const u32x4_t k = *reinterpret_cast<const u32x4_t*>(kp + u * 512);
      s = MFMA32x32x16(e4m3x8(k[0], k[1], ks), q[u][0], s);
      s = MFMA32x32x16(e4m3x8(k[2], k[3], ks), q[u][1], s);
    }
    if (page * 16 + 31 > first_lim) {  // (wave-uniform: positions that some row does not see)
      const int p0 = page * 16 + 4 * h;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (p0 + 8 * (r >> 2) + (r & 3) > lim) s[r] = -INFINITY;
    }
    float m = max3f(s[0], s[1], s[2]);
#pragma unroll
    for (int r = 3; r < 15; r += 2) m = max3f(m, s[r], s[r + 1]);
    m = max3f(m, s[15], s[15]);
    if (__builtin_expect(__any(m > thr), 0)) {
      const float top = fmaxf(m, __shfl_xor(m, 32));
      const bool grow = top > thr;
      const float delta = grow ? ceilf(top) : 0.0f;  // (integer steps keep the base integral)
      const float alpha = grow && thr != -INFINITY ? pow2i(-delta) : 1.0f;
      base += delta;
      thr = grow ? kLazyMax : thr;
      s -= delta;
      sum *= alpha;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] *= alpha;
    }
    half8_t p[2];
    const half2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const f32x2_t e = {__builtin_amdgcn_exp2f(s[r]), __builtin_amdgcn_exp2f(s[r + 1])};
      const half2_t w = __builtin_convertvector(e, half2_t);
      sum = __builtin_amdgcn_fdot2(w, ones, sum, false);
      p[r >> 3][r & 7] = w[0];
      p[r >> 3][(r & 7) + 1] = w[1];
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float vs = __uint_as_float((b ? sb : sa) & 0xffff0000u);
      const char* vp = slot + b * BLOCK + 16 * W + (h * 16 + (c & 15)) * 16;
      uint32_t x[NT], y[NT];  // tokens 4h .. and 8 + 4h .. of dims 32i + c
      if constexpr (W == 64) {
        const u32x2_t a = *reinterpret_cast<const u32x2_t*>(vp + (c >> 4) * 8);
        const u32x2_t d = *reinterpret_cast<const u32x2_t*>(vp + (c >> 4) * 8 + 512);
        x[0] = a[0]; x[1] = a[1]; y[0] = d[0]; y[1] = d[1];
      } else {
        const char* vq = vp + (c >> 4) * (8 * W);
#pragma unroll
        for (int k = 0; k < NT / 4; ++k) {
          const u32x4_t a = *reinterpret_cast<const u32x4_t*>(vq + k * 1024);
          const u32x4_t d = *reinterpret_cast<const u32x4_t*>(vq + k * 1024 + 512);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[4 * k + i] = a[i];
            y[4 * k + i] = d[i];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] = MFMA32x32x16(e4m3x8(x[i], y[i], vs), p[b], o[i]);
    }
  }
};

__device__ __forceinline__ E4m3Item load_item(const E4m3Item* items, int i) {
  const sconst_int* w = (const sconst_int*)(items + i);
  E4m3Item t;
  t.kv_head = w[0];
  t.page_begin = w[1];
  t.page_end = w[2];
  t.part = w[3];
  t.row0 = w[4];
  t.rows = w[5];
  t.ctx = w[6];
  t.q_row = w[7];
  t.table_off = w[8];
  t.merge = w[9];
  t.rw = w[10];
  t.once = w[11];
  return t;
}

// Chunk c (4 dims) of row r in the staged accumulators: 16-byte chunks are
// permuted within a row so that 32 rows fall on different banks.
template <int W>
__device__ __forceinline__ int staged(int r, int c) {
  return r * W * 4 + ((c ^ (r & (W / 4 - 1))) << 4);
}

template <int W, int RW>
__device__ __forceinline__ void run_item(const E4m3Attn& p, E4m3Shared<W>& sh, const E4m3Item& it) {
  using C = E4m3Cfg<W>;
  constexpr int KS = 4 / RW, TP = C::TP(RW), NB = C::NB(RW), MINE = TP / RW;  // pages a wave copies per tile
  constexpr int LOADS = MINE * C::BLOCK / 1024;
  static_assert(MINE >= 1, "every wave copies a page");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave % RW, ks = wave / RW;
  const int c = lane & 31, h = lane >> 5;
  const int npages = it.page_end - it.page_begin;
  const int ntiles = (npages + TP - 1) / TP;
  const int turns = (ntiles + KS - 1) / KS;

  // ---- the item's block numbers and rows
  for (int j = threadIdx.x; j < npages; j += 256)
    sh.ids[j] = p.tables[it.table_off + it.page_begin + j] * p.kv_heads + it.kv_head;
  if ((int)threadIdx.x < it.rows) {
    const int r = it.row0 + threadIdx.x, query = r / p.group;
    sh.out_at[threadIdx.x] = (long)(it.q_row + query) * p.out_stride +
                             (long)(it.kv_head * p.group + r - query * p.group) * p.dims;
  }
  __syncthreads();

  char* const ring = sh.ring + ks * NB * TP * C::BLOCK;
  // Tile `turn * KS + ks` of the item into its slot; pages past the range
  // repeat the last one (no row sees their positions).
  auto fetch = [&](int turn) __attribute__((always_inline)) {
    char* const slot = ring + (turn % NB) * TP * C::BLOCK + wr * MINE * C::BLOCK;
    const int j0 = (turn * KS + ks) * TP + wr * MINE;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int n = __builtin_amdgcn_readfirstlane(sh.ids[min(j0 + i, npages - 1)]);
      if (it.once)
        fetch_block<W, kPageLoadPolicy>(slot + i * C::BLOCK, p.blocks, n, lane);
      else
        fetch_block<W, kPageReusePolicy>(slot + i * C::BLOCK, p.blocks, n, lane);
    }
  };
#pragma unroll
  for (int k = 0; k < NB - 1; ++k)
    if (k < turns) fetch(k);
  for (int j = threadIdx.x; j < npages; j += 256) sh.scales[j] = p.scales[sh.ids[j]];

  E4m3Rows<W> x;
  {
    const int r = wr * 32 + c;
    const bool live = r < it.rows;
    const int g = it.row0 + (live ? r : 0), query = g / p.group;
    const int end = it.page_end * 16 - 1;
    x.lim = live ? min(it.ctx + query, end) : -1;
    const int last = min(wr * 32 + 31, it.rows - 1);
    x.first_lim = wr * 32 < it.rows ? min(it.ctx + (it.row0 + wr * 32) / p.group, end) : -1;
    x.last_lim = wr * 32 < it.rows ? min(it.ctx + (it.row0 + last) / p.group, end) : -1;
    const long at = (long)(it.q_row + query) * p.q_stride + (long)(it.kv_head * p.group + g - query * p.group) * p.dims;
#pragma unroll
    for (int u = 0; u < E4m3Rows<W>::KS; ++u) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = 32 * u + 16 * h + 8 * e;
        x.q[u][e] = live && d < p.dims ? load_q8(p.q, at + d, p.row_type, p.scale_log2) : half8_t{};
      }
    }
    x.base = 0.0f;
    x.thr = -INFINITY;
    x.sum = 0.0f;
#pragma unroll
    for (int i = 0; i < E4m3Rows<W>::NT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) x.o[i][e] = 0.0f;
  }
  __syncthreads();  // scales are in LDS

  for (int turn = 0; turn < turns; ++turn) {
    if constexpr (RW == 1) {
      if (turn + NB - 1 < turns) {
        fetch(turn + NB - 1);
        wait_vmcnt<(NB - 1) * LOADS>();
      } else {
        wait_vmcnt<0>();
      }
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
    } else {
      wait_vmcnt_pages<NB - 2, LOADS>(min(NB - 2, turns - 1 - turn));
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (turn + NB - 1 < turns) fetch(turn + NB - 1);
    }
    const char* const slot = ring + (turn % NB) * TP * C::BLOCK;
    const int j0 = (turn * KS + ks) * TP;
#pragma unroll
    for (int b = 0; b < TP; b += 2) {
      const int page = it.page_begin + j0 + b;
      if (j0 + b < npages && page * 16 <= x.last_lim) {
        const uint32_t sa = __builtin_amdgcn_readfirstlane(sh.scales[j0 + b]);
        const uint32_t sb = __builtin_amdgcn_readfirstlane(sh.scales[min(j0 + b + 1, npages - 1)]);
        x.pair(slot + b * C::BLOCK, sa, sb, page, lane);
      }
    }
    if constexpr (RW == 1) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }

  // ---- the groups' states become one: common bases, sums, accumulators
  x.sum += __shfl_xor(x.sum, 32);
  // (a row of NaN scores never moves its base: its sum tells it from a row
  // that saw nothing)
  const bool none = x.thr == -INFINITY && x.sum == x.sum;
  if (h == 0) {
    sh.ml[0][wave][c] = none ? -INFINITY : x.base;
    sh.ml[1][wave][c] = x.sum;
  }
  __syncthreads();  // (also: every wave has left the ring)
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < KS; ++k) top = fmaxf(top, sh.ml[0][k * RW + wr][c]);
  const float f = none ? 0.0f : pow2i(x.base - top);
  if (ks == 0 && h == 0) {
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const float m = sh.ml[0][k * RW + wr][c];
      if (m != -INFINITY) sum += sh.ml[1][k * RW + wr][c] * pow2i(m - top);
    }
    sh.base[wr * 32 + c] = top;
    sh.sum[wr * 32 + c] = sum;
  }
  char* const stage = sh.ring + wave * 32 * W * 4;
#pragma unroll
  for (int i = 0; i < E4m3Rows<W>::NT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<float4_t*>(stage + staged<W>(c, 8 * i + 2 * e + h)) =
          float4_t{x.o[i][4 * e], x.o[i][4 * e + 1], x.o[i][4 * e + 2], x.o[i][4 * e + 3]} * f;
  __syncthreads();
  const auto rs_o = make_rsrc(p.part_o, 0x7fffffff);
  const auto rs_ml = make_rsrc(p.part_ml, 0x7fffffff);
  for (int idx = threadIdx.x; idx < it.rows * (W / 4); idx += 256) {
    const int r = idx / (W / 4), d4 = idx % (W / 4);
    float4_t acc = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < KS; ++k)
      acc += *reinterpret_cast<const float4_t*>(sh.ring + (k * RW + (r >> 5)) * 32 * W * 4 + staged<W>(r & 31, d4));
    if (it.part < 0) {
      const float sum = sh.sum[r];
      if (4 * d4 < p.dims)
        store_out4(p.out, sh.out_at[r] + 4 * d4, p.row_type, sum > 0.0f || sum != sum ? div4(acc, sum) : float4_t{0, 0, 0, 0});
    } else {
      coh_store4(rs_o, (uint32_t)((((size_t)it.part * kE4m3Rows + r) * W + 4 * d4) * 4), acc);
      if (d4 == 0) coh_store2(rs_ml, (uint32_t)(((size_t)it.part * kE4m3Rows + r) * 8), sh.base[r], sh.sum[r]);
    }
  }
  if (it.part >= 0) {
    // The last piece of the tile to arrive merges them all, in their order.
    const E4m3Merge m = p.merges[it.merge];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    wait_vmcnt<0>();
    __syncthreads();
    if (threadIdx.x == 0)
      sh.flag = __hip_atomic_fetch_add(p.counters + it.merge, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                m.n_parts - 1;
    __syncthreads();
    if (sh.flag) {
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
      if ((int)threadIdx.x < m.rows) {
        float mm = -INFINITY, sum = 0.0f;
        for (int k = 0; k < m.n_parts; ++k) {
          const float2 v = coh_load2(rs_ml, (uint32_t)(((size_t)(m.first_part + k) * kE4m3Rows + threadIdx.x) * 8));
          if (v.x == -INFINITY) continue;
          const float t = fmaxf(mm, v.x);
          sum = (mm == -INFINITY ? 0.0f : sum * pow2i(mm - t)) + v.y * pow2i(v.x - t);
          mm = t;
        }
        sh.base[threadIdx.x] = mm;
        sh.sum[threadIdx.x] = sum;
      }
      __syncthreads();
      for (int idx = threadIdx.x; idx < m.rows * (W / 4); idx += 256) {
        const int r = idx / (W / 4), d4 = idx % (W / 4);
        const float mm = sh.base[r], sum = sh.sum[r];
        float4_t acc = {0, 0, 0, 0};
        for (int k = 0; k < m.n_parts; ++k) {
          const size_t at = (size_t)(m.first_part + k) * kE4m3Rows + r;
          const float2 v = coh_load2(rs_ml, (uint32_t)(at * 8));
          const float4_t o = coh_load4(rs_o, (uint32_t)((at * W + 4 * d4) * 4));
          if (v.x != -INFINITY) acc += o * pow2i(v.x - mm);
        }
        if (4 * d4 < p.dims)
          store_out4(p.out, sh.out_at[r] + 4 * d4, p.row_type, sum > 0.0f || sum != sum ? div4(acc, sum) : float4_t{0, 0, 0, 0});
      }
      if (threadIdx.x == 0) __hip_atomic_store(p.counters + it.merge, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();  // the shared state is free for the next item
}

template <int W>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(E4m3Cfg<W>::PER_CU, E4m3Cfg<W>::PER_CU)))
void attention_e4m3_kernel(E4m3Attn p) {
  __shared__ E4m3Shared<W> sh;
  const int first = p.wg_first[blockIdx.x], last = p.wg_first[blockIdx.x + 1];
  for (int i = first; i < last; ++i) {
    const E4m3Item it = load_item(p.items, i);
    if (it.rw == 1)
      run_item<W, 1>(p, sh, it);
    else if (it.rw == 2)
      run_item<W, 2>(p, sh, it);
    else
      run_item<W, 4>(p, sh, it);
  }
}

}  // namespace

int e4m3_groups_per_cu(int width) {
  return width > 128 ? E4m3Cfg<256>::PER_CU : width > 64 ? E4m3Cfg<128>::PER_CU : E4m3Cfg<64>::PER_CU;
}

hipError_t launch_e4m3_attention(int width, int groups, const E4m3Attn& p, hipStream_t stream) {
  if (width == 64)
    attention_e4m3_kernel<64><<<groups, 256, 0, stream>>>(p);
  else if (width == 128)
    attention_e4m3_kernel<128><<<groups, 256, 0, stream>>>(p);
  else
    attention_e4m3_kernel<256><<<groups, 256, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace tge
