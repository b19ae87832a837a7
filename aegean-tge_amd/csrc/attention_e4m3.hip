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
// No accumulator and no weight crosses lanes until a tile ends.
//
// Every row sees its own position, so its weights sum to more than 0 unless all
// its scores are -infinity (an infinite q against K of the other sign): 0 / 0
// makes that row NaN, as the formula does.
//
// Roundings: rows of fp32 and bf16 are scaled and rounded to f16 once (a score
// moves by 2^-11 of the sum of its products' magnitudes, and by 2^-25 of the sum
// of |k| where scaled values lie below f16's normal range), rows of f16 enter as
// they are and their scores are scaled; weights are rounded to f16; sums, bases
// and accumulators are fp32, out is rounded once.
//
// What bounds it, MI355X, 28/4 heads of 128 dims unless said:
//   decode   the block reads (a probe that only reads blocks of this size 6.6
//            TB/s). 128 sessions of 8192 tokens 164-168 us, 6.4-6.6 TB/s; 64
//            ragged ones of 1k to 32k tokens, four drafted tokens each (613 MB),
//            118-121 us, 5.1-5.2 TB/s, no matter how the shares are cut, the
//            rest being starts and merges of 1.4 pieces a workgroup; 32 sessions
//            of 16/8 heads of 256 dims (1234 MB) 219-225 us, 5.5-5.6 TB/s. With
//            33 to 64 rows a KV head the conversions and products count too: 64
//            such sessions of 64/8 heads, eight drafted tokens each (1236 MB),
//            253 us, 4.9 TB/s.
//   prompts  issue: with the matrix cores 40 % and the vector units 50 % of the
//            time busy, converting the codes and the exponentials stand
//            between the products. 8192 tokens 460-487 us, 990-1046 TFLOP/s; 2048
//            behind 8000 of 64/8 heads 562-596 us, 1015-1078; 1333 behind 14003
//            300-316 us, 887-935 (a large f16 product of a library reaches 1105
//            here). Shorter ones lack work to even out causal tiles of unlike
//            lengths: 2048 tokens 49 us, 608 TFLOP/s; so do those of 256 dims,
//            one workgroup a unit: 2048 of 16/8 heads 70 us, 489.
//   few rows the chain of loads: item, block numbers, scales and blocks, then
//            the waves' turns, and a merge where the context is cut. One new
//            token at 1056 of 14/2 heads of 64 dims (uncut) 9.0-9.6 us.
// Rows of a tile, us at RW 1 / 2 / 4: 512 behind 1536 tokens 24 / 31 / 42, 2048
// tokens 56 / 49 / 50, 8192 tokens 567 / 508 / 470.
#include <type_traits>

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
  static constexpr int PER_CU = W > 128 ? 1 : W > 64 ? 2 : 3;  // workgroups a unit that their LDS leaves room for
  // At 256 dims a tile's codes do not fit beside the accumulators: they are
  // read where they are used, and a wave's own slots refilled by halves (K, V).
  static constexpr bool LAZY = W > 128;
  static constexpr int TP(int rw) { return rw == 4 ? 4 : 2; }  // pages of a tile
  static constexpr int NB(int rw) { return rw == 1 ? 2 : 4; }  // ring slots of a group
  static constexpr int RING = 16 * BLOCK;                      // (4 / rw) * NB * TP blocks
  static_assert(4 * NB(1) * TP(1) == 16 && 2 * NB(2) * TP(2) == 16 && NB(4) * TP(4) == 16, "ring size");
};

constexpr int kE4m3Window = 1024;  // pages whose block numbers are in LDS at a time

template <int W>
struct E4m3Shared {
  alignas(16) char ring[E4m3Cfg<W>::RING];  // at a tile's end: the waves' accumulators
  int ids[kE4m3Window];                  // of the item's pages: block numbers
  alignas(8) uint32_t scales[kE4m3Window];  // and their scale pairs
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

// A lane's q operands: of the row that starts at element `at` the dims 32u +
// 16h + 8e .., times c, as f16; zero where the lane has no row and past the
// head's dims. Every load is issued before any is used.
template <int KS>
__device__ __forceinline__ void load_q(half8_t (&r)[KS][2], const void* q, long at, int h, int dims, bool live, int type,
                                       float c) {
  auto place = [&](int u, int e) __attribute__((always_inline)) {
    const int d = 32 * u + 16 * h + 8 * e;
    return at + (d < dims ? d : 0);
  };
  if (type == TGE_ROWS_F32) {
    float4_t x[KS][2][2];
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float4_t* p = reinterpret_cast<const float4_t*>(static_cast<const float*>(q) + place(u, e));
        x[u][e][0] = p[0];
        x[u][e][1] = p[1];
      }
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 8; ++i) r[u][e][i] = (_Float16)(x[u][e][i >> 2][i & 3] * c);
  } else {
    u32x4_t w[KS][2];
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        w[u][e] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(q) + place(u, e));
#pragma unroll
    for (int u = 0; u < KS; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (type == TGE_ROWS_F16) {  // (c is 1)
          r[u][e] = bitcast<half8_t>(w[u][e]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            r[u][e][2 * i] = (_Float16)(__uint_as_float(w[u][e][i] << 16) * c);
            r[u][e][2 * i + 1] = (_Float16)(__uint_as_float(w[u][e][i] & 0xffff0000u) * c);
          }
        }
      }
  }
#pragma unroll
  for (int u = 0; u < KS; ++u)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (!live || 32 * u + 16 * h + 8 * e >= dims) r[u][e] = half8_t{};
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

// Copy the page block `n` to LDS at `slot`: KiB [FROM, TO) of it.
template <int W, int POLICY, int FROM, int TO>
__device__ __forceinline__ void fetch_block(char* slot, const char* blocks, int n, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BLOCK = E4m3Cfg<W>::BLOCK;
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(blocks + (size_t)n * BLOCK, BLOCK);
#pragma unroll
  for (int i = FROM; i < TO; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(slot + i * 1024), 16, i * 1024 + lane * 16, 0, 0,
                                             POLICY);
#endif
}

// The codes of 32 tokens (two blocks) in a lane's operand order, and the
// blocks' scale pairs.
template <int W>
struct E4m3Codes {
  static constexpr int KS = W / 32;  // K pieces of 16 dims (two operands each)
  static constexpr int NT = W / 32;  // 32-dim output tiles
  u32x4_t k[KS];
  uint32_t v[2][2][NT];  // [block][tokens 4h.. | 8 + 4h..][dims 32i + c]
  uint32_t sa, sb;

  __device__ __forceinline__ void read_scales(const uint32_t* scales) {
    const u32x2_t s = *reinterpret_cast<const u32x2_t*>(scales);
    sa = s[0];
    sb = s[1];
  }
  __device__ __forceinline__ void read_k(const char* slot, int lane) {
    const int c = lane & 31, h = lane >> 5;
    const char* kp = slot + (c >> 4) * E4m3Cfg<W>::BLOCK + h * 256 + (c & 15) * 16;
#pragma unroll
    for (int u = 0; u < KS; ++u) k[u] = *reinterpret_cast<const u32x4_t*>(kp + u * 512);
  }
  __device__ __forceinline__ void read_v(const char* slot, int lane) {
    const int c = lane & 31, h = lane >> 5;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const char* vp = slot + b * E4m3Cfg<W>::BLOCK + 16 * W + (h * 16 + (c & 15)) * 16;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (W == 64) {
          const u32x2_t x = *reinterpret_cast<const u32x2_t*>(vp + (c >> 4) * 8 + t * 512);
          v[b][t][0] = x[0];
          v[b][t][1] = x[1];
        } else {
#pragma unroll
          for (int i = 0; i < NT; i += 4) {
            const u32x4_t x = *reinterpret_cast<const u32x4_t*>(vp + (c >> 4) * (8 * W) + i * 256 + t * 512);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[b][t][i + e] = x[e];
          }
        }
      }
    }
  }
};

// A wave's rows against pages.
template <int W>
struct E4m3Rows {
  static constexpr int KS = E4m3Codes<W>::KS, NT = E4m3Codes<W>::NT;
  half8_t q[KS][2];    // row c, dims 32u + 16h + 8x ..
  f32x16_t o[NT];
  f32x16_t start;      // -base, sixteen times: the scores' start (0 when they are scaled afterwards; not at 256 dims)
  float base, thr, sum;  // of the row; `sum` over the lane's own tokens
  float after;         // factor of the scores once q has entered unscaled, or 0
  int lim;             // the row's last visible position within the item
  int first_lim, last_lim;  // over the wave's rows (wave-uniform)

  __device__ __forceinline__ f32x16_t fresh_start() const {
    f32x16_t s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = after != 0.0f ? 0.0f : -base;
    return s;
  }
  __device__ __forceinline__ void set_start() {
    if constexpr (!E4m3Cfg<W>::LAZY) start = fresh_start();
  }

  // Tokens [16 * page, 16 * page + 32): the weights of the lane's tokens to p.
  __device__ __forceinline__ void scores(const E4m3Codes<W>& x, int page, int lane, half8_t (&p)[2]) {
    const int c = lane & 31, h = lane >> 5;
    const float ks = __uint_as_float((c & 16 ? x.sb : x.sa) << 16);
    f32x16_t s;
    if constexpr (E4m3Cfg<W>::LAZY)
      s = fresh_start();
    else
      s = start;
#pragma unroll
    for (int u = 0; u < KS; ++u) {
      s = MFMA32x32x16(e4m3x8(x.k[u][0], x.k[u][1], ks), q[u][0], s);
      s = MFMA32x32x16(e4m3x8(x.k[u][2], x.k[u][3], ks), q[u][1], s);
    }
    if (after != 0.0f) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], after, -base);
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
      set_start();
    }
    const half2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const f32x2_t e = {__builtin_amdgcn_exp2f(s[r]), __builtin_amdgcn_exp2f(s[r + 1])};
      const half2_t w = __builtin_convertvector(e, half2_t);
      sum = __builtin_amdgcn_fdot2(w, ones, sum, false);
      p[r >> 3][r & 7] = w[0];
      p[r >> 3][(r & 7) + 1] = w[1];
    }
  }

  __device__ __forceinline__ void pair(const E4m3Codes<W>& x, int page, int lane) {
    half8_t p[2];
    scores(x, page, lane, p);
    values(x, p);
  }

  // The same tokens' values with those weights.
  __device__ __forceinline__ void values(const E4m3Codes<W>& x, const half8_t (&p)[2]) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float vs = __uint_as_float((b ? x.sb : x.sa) & 0xffff0000u);
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] = MFMA32x32x16(e4m3x8(x.v[b][0][i], x.v[b][1][i], vs), p[b], o[i]);
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
  t.next = w[12];
  return t;
}

// Chunk c (4 dims) of row r in the staged accumulators: 16-byte chunks are
// permuted within a row so that 32 rows fall on different banks.
template <int W>
__device__ __forceinline__ int staged(int r, int c) {
  return r * W * 4 + ((c ^ (r & (W / 4 - 1))) << 4);
}

// threadIdx.x, computed anew wherever this is called: without it the compiler
// moves every address of the item's end in front of the item loop and spills.
__device__ __forceinline__ int thread_here() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// The states of a split tile's pieces become its output. Every thread adds J
// chunks of 4 dims, K pieces in flight, weighted by the pieces' bases, which
// all threads take from LDS; the sums are in the pieces' order.
template <int W, int J, int K>
__device__ __forceinline__ void merge_parts(const E4m3Attn& p, E4m3Shared<W>& sh, const E4m3Item& it,
                                            const E4m3Merge& m) {
  const auto rs_o = make_rsrc(p.part_o, 0x7fffffff);
  const auto rs_ml = make_rsrc(p.part_ml, 0x7fffffff);
  const int t = thread_here(), rows = m.rows, n = m.n_parts, chunks = rows * (W / 4);
  float2* const ml = reinterpret_cast<float2*>(sh.ring);  // [n][rows]: (base, sum)
  const bool fits = (size_t)n * rows * sizeof(float2) <= sizeof(sh.ring);  // else they are read where they are used
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  auto state = [&](int k, int r) __attribute__((always_inline)) {
    return coh_load2(rs_ml, (uint32_t)(((size_t)(m.first_part + k) * p.part_rows + r) * 8));
  };
  float4_t o[J][K];
  auto load = [&](int i0, int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int idx = min(i0 + 256 * j, chunks - 1), r = idx / (W / 4), d4 = idx % (W / 4);
#pragma unroll
      for (int e = 0; e < K; ++e)
        o[j][e] = coh_load4(rs_o, (uint32_t)((((size_t)(m.first_part + min(k0 + e, n - 1)) * p.part_rows + r) * W + 4 * d4) * 4));
    }
  };
  if (fits) {
#pragma unroll 1
    for (int i = t; i < n * rows; i += 256) ml[i] = state(i / rows, i % rows);
  }
  load(t, 0);
  // (LDS alone is ordered: the accumulators stay in flight)
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll 1
  for (int i0 = t; i0 < chunks; i0 += 256 * J) {
    float4_t acc[J];
    float top[J], sum[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int r = min(i0 + 256 * j, chunks - 1) / (W / 4);
      acc[j] = float4_t{0, 0, 0, 0};
      top[j] = -INFINITY;
      sum[j] = 0.0f;
#pragma unroll 4
      for (int k = 0; k < n; ++k) top[j] = fmaxf(top[j], fits ? ml[k * rows + r].x : state(k, r).x);
    }
#pragma unroll 1
    for (int k0 = 0; k0 < n; k0 += K) {
      if (i0 != t || k0 != 0) load(i0, k0);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int r = min(i0 + 256 * j, chunks - 1) / (W / 4);
#pragma unroll
        for (int e = 0; e < K; ++e) {
          const int k = min(k0 + e, n - 1);
          const float2 v = fits ? ml[k * rows + r] : state(k, r);
          const float w = k0 + e >= n || v.x == -INFINITY ? 0.0f : pow2i(v.x - top[j]);
          sum[j] += w * v.y;
          acc[j] += o[j][e] * w;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int idx = i0 + 256 * j, r = idx / (W / 4), d4 = idx % (W / 4);
      if (idx < chunks && 4 * d4 < p.dims)
        store_out4(p.out, sh.out_at[r] + 4 * d4, p.row_type, div4(acc[j], sum[j]));
    }
  }
  if (t == 0) __hip_atomic_store(p.counters + it.merge, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
  // (the first pages' ids are on their way while the rows are set up)
  const int first_id = p.tables[it.table_off + min(it.page_begin + (int)threadIdx.x, it.page_end - 1)];
  // ---- the item's rows
  if ((int)threadIdx.x < it.rows) {
    const int r = it.row0 + threadIdx.x, query = r / p.group;
    sh.out_at[threadIdx.x] = (long)(it.q_row + query) * p.out_stride +
                             (long)(it.kv_head * p.group + r - query * p.group) * p.dims;
  }
  E4m3Rows<W> x;
  {
    // f16 rows enter the products as they are and the scores are scaled
    // afterwards; scaled first, their second rounding doubles the error of an
    // f16 output. (fp32 and bf16 rows are scaled and rounded to f16 once.)
    x.after = p.row_type == TGE_ROWS_F16 ? p.scale_log2 : 0.0f;
    const float factor = p.row_type == TGE_ROWS_F16 ? 1.0f : p.scale_log2;
    const int r = wr * 32 + c;
    const bool live = r < it.rows;
    const int g = it.row0 + (live ? r : 0), query = g / p.group;
    const int end = it.page_end * 16 - 1;
    x.lim = live ? min(it.ctx + query, end) : -1;
    const int last = min(wr * 32 + 31, it.rows - 1);
    x.first_lim = wr * 32 < it.rows ? min(it.ctx + (it.row0 + wr * 32) / p.group, end) : -1;
    x.last_lim = wr * 32 < it.rows ? min(it.ctx + (it.row0 + last) / p.group, end) : -1;
    const long at = (long)(it.q_row + query) * p.q_stride + (long)(it.kv_head * p.group + g - query * p.group) * p.dims;
    load_q(x.q, p.q, at, h, p.dims, live, p.row_type, factor);
    x.base = 0.0f;
    x.thr = -INFINITY;
    x.sum = 0.0f;
    x.set_start();
#pragma unroll
    for (int i = 0; i < E4m3Rows<W>::NT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) x.o[i][e] = 0.0f;
  }

  char* const ring = sh.ring + ks * NB * TP * C::BLOCK;
  for (int begin = it.page_begin; begin < it.page_end; begin += kE4m3Window) {
    const int npages = min(it.page_end - begin, kE4m3Window);
    const int ntiles = (npages + TP - 1) / TP;
    const int turns = (ntiles + KS - 1) / KS;
    // The pages' block numbers, to a whole number of tiles: pages past the
    // range repeat the last one, whose positions there no row sees.
    const int padded = (npages + 7) & ~7;
    for (int j = threadIdx.x; j < padded; j += 256) {
      const bool have = begin == it.page_begin && j < 256;
      const int id = have ? first_id : p.tables[it.table_off + begin + min(j, npages - 1)];
      sh.ids[j] = id * p.kv_heads + it.kv_head;
    }
    __syncthreads();

    // The blocks of the pages that this wave copies of tile `turn * KS + ks` (a
    // group past the item's last tile copies that one again), and their copies
    // into the tile's slot.
    struct Blocks {
      int n[MINE];
    };
    auto blocks_of = [&](int turn) __attribute__((always_inline)) {
      const int j0 = min(turn * KS + ks, ntiles - 1) * TP + wr * MINE;
      Blocks b;
#pragma unroll
      for (int i = 0; i < MINE; ++i) b.n[i] = sh.ids[j0 + i];
      return b;
    };
    auto fetch = [&](int turn, const Blocks& b, auto from, auto to) __attribute__((always_inline)) {
      char* const slot = ring + (turn % NB) * TP * C::BLOCK + wr * MINE * C::BLOCK;
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int block = __builtin_amdgcn_readfirstlane(b.n[i]);
        if (it.once)
          fetch_block<W, kPageLoadPolicy, from.value, to.value>(slot + i * C::BLOCK, p.blocks, block, lane);
        else
          fetch_block<W, kPageReusePolicy, from.value, to.value>(slot + i * C::BLOCK, p.blocks, block, lane);
      }
    };
    using First = std::integral_constant<int, 0>;  // (KiB of a block)
    using Middle = std::integral_constant<int, C::BLOCK / 2048>;
    using End = std::integral_constant<int, C::BLOCK / 1024>;
    constexpr int AHEAD = RW == 1 ? NB : NB - 1;  // tiles copied before the first is used
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (k < turns) fetch(k, blocks_of(k), First{}, End{});
    for (int j = threadIdx.x; j < padded; j += 256) sh.scales[j] = p.scales[sh.ids[j]];
    __syncthreads();  // scales are in LDS

    for (int turn = 0; turn < turns; ++turn) {
      char* const slot = ring + (turn % NB) * TP * C::BLOCK;
      const int j0 = (turn * KS + ks) * TP;
      const int page = begin + j0;
      if constexpr (RW == 1) {
        // The wave's own ring: once a tile's codes are in registers its slot
        // takes the tile NB turns on, so NB tiles are in flight while one is
        // worked on.
        if (turn + 1 < turns)
          wait_vmcnt<(NB - 1) * LOADS>();
        else
          wait_vmcnt<0>();
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        const int j = min(j0, padded - TP);
        const bool seen = j0 < npages && page * 16 <= x.last_lim;
        E4m3Codes<W> codes;
        half8_t weights[2];
        codes.read_scales(sh.scales + j);
        const Blocks next = blocks_of(turn + NB);
        if constexpr (C::LAZY) {
          codes.read_k(slot, lane);
          if (seen) x.scores(codes, page, lane, weights);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (turn + NB < turns) fetch(turn + NB, next, First{}, Middle{});
          codes.read_v(slot, lane);
          if (seen) x.values(codes, weights);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (turn + NB < turns) fetch(turn + NB, next, Middle{}, End{});
        } else {
          codes.read_k(slot, lane);
          codes.read_v(slot, lane);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (turn + NB < turns) fetch(turn + NB, next, First{}, End{});
          if (seen) x.pair(codes, page, lane);
        }
      } else {
        const Blocks next = blocks_of(turn + NB - 1);
        wait_vmcnt_pages<NB - 2, LOADS>(min(NB - 2, turns - 1 - turn));
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (turn + NB - 1 < turns) fetch(turn + NB - 1, next, First{}, End{});
#pragma unroll
        for (int b = 0; b < TP; b += 2) {
          if (j0 + b < npages && (page + b) * 16 <= x.last_lim) {
            E4m3Codes<W> codes;
            codes.read_scales(sh.scales + j0 + b);
            codes.read_k(slot + b * C::BLOCK, lane);
            if constexpr (C::LAZY) {
              half8_t weights[2];
              x.scores(codes, page + b, lane, weights);
              codes.read_v(slot + b * C::BLOCK, lane);
              x.values(codes, weights);
            } else {
              codes.read_v(slot + b * C::BLOCK, lane);
              x.pair(codes, page + b, lane);
            }
          }
        }
      }
    }
    if (begin + kE4m3Window < it.page_end) __syncthreads();  // every wave has left the window's tables
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
  const int t = thread_here();
  char* const stage = sh.ring + (t >> 6) * 32 * W * 4;
#pragma unroll
  for (int i = 0; i < E4m3Rows<W>::NT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<float4_t*>(stage + staged<W>(t & 31, 8 * i + 2 * e + ((t >> 5) & 1))) =
          float4_t{x.o[i][4 * e], x.o[i][4 * e + 1], x.o[i][4 * e + 2], x.o[i][4 * e + 3]} * f;
}

// The staged accumulators of the item's waves become output rows or, for a
// piece of a split tile, a partial state; the last piece of a tile to arrive
// merges them all.
template <int W>
__device__ __forceinline__ void finish_item(const E4m3Attn& p, E4m3Shared<W>& sh, const E4m3Item& it) {
  __syncthreads();
  const int rw = it.rw, copies = 4 / rw;
  const auto rs_o = make_rsrc(p.part_o, 0x7fffffff);
  const auto rs_ml = make_rsrc(p.part_ml, 0x7fffffff);
#pragma unroll 2
  for (int idx = thread_here(); idx < it.rows * (W / 4); idx += 256) {
    const int r = idx / (W / 4), d4 = idx % (W / 4);
    const char* from = sh.ring + (r >> 5) * 32 * W * 4 + staged<W>(r & 31, d4);
    float4_t acc = *reinterpret_cast<const float4_t*>(from);
    for (int k = 1; k < copies; ++k) acc += *reinterpret_cast<const float4_t*>(from + k * rw * 32 * W * 4);
    if (it.part < 0) {
      if (4 * d4 < p.dims) store_out4(p.out, sh.out_at[r] + 4 * d4, p.row_type, div4(acc, sh.sum[r]));
    } else {
      coh_store4(rs_o, (uint32_t)((((size_t)it.part * p.part_rows + r) * W + 4 * d4) * 4), acc);
      if (d4 == 0) coh_store2(rs_ml, (uint32_t)(((size_t)it.part * p.part_rows + r) * 8), sh.base[r], sh.sum[r]);
    }
  }
  if (it.part >= 0) {
    const E4m3Merge m = p.merges[it.merge];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    wait_vmcnt<0>();
    __syncthreads();
    if (threadIdx.x == 0)
      sh.flag = __hip_atomic_fetch_add(p.counters + it.merge, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                m.n_parts - 1;
    __syncthreads();
    if (sh.flag) {
      if (m.rows * (W / 4) <= 256)
        merge_parts<W, 1, W == 64 ? 12 : 16>(p, sh, it, m);
      else
        merge_parts<W, W == 64 ? 2 : 4, W == 64 ? 6 : 4>(p, sh, it, m);
    }
  }
  __syncthreads();  // the shared state is free for the next item
}

template <int W>
__device__ __forceinline__ void run_items(const E4m3Attn& p, E4m3Shared<W>& sh) {
  for (int i = blockIdx.x; i >= 0;) {
    const E4m3Item it = load_item(p.items, i);
    i = it.next;
    if (it.rw == 1)
      run_item<W, 1>(p, sh, it);
    else if (it.rw == 2)
      run_item<W, 2>(p, sh, it);
    else
      run_item<W, 4>(p, sh, it);
    finish_item<W>(p, sh, it);
  }
}

// (the attributes take numbers only: waves per SIMD)
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3, 3))) void attention_e4m3_64(E4m3Attn p) {
  __shared__ E4m3Shared<64> sh;
  run_items<64>(p, sh);
}
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_e4m3_128(E4m3Attn p) {
  __shared__ E4m3Shared<128> sh;
  run_items<128>(p, sh);
}
// One workgroup fills a compute unit's LDS, so a wave could have 512 registers;
// but the compiler then keeps the accumulators in the second register file and
// moves all of them around every pair of pages. With the LDS sized at launch
// it plans for two waves a SIMD and the 256 registers of the first file.
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_e4m3_256(E4m3Attn p) {
  extern __shared__ __align__(16) char at_launch[];
  run_items<256>(p, *reinterpret_cast<E4m3Shared<256>*>(at_launch));
}

}  // namespace

int e4m3_groups_per_cu(int width) {
  return width > 128 ? E4m3Cfg<256>::PER_CU : width > 64 ? E4m3Cfg<128>::PER_CU : E4m3Cfg<64>::PER_CU;
}

hipError_t launch_e4m3_attention(int width, int groups, const E4m3Attn& p, hipStream_t stream) {
  if (width == 64)
    attention_e4m3_64<<<groups, 256, 0, stream>>>(p);
  else if (width == 128)
    attention_e4m3_128<<<groups, 256, 0, stream>>>(p);
  else {
    constexpr size_t lds = sizeof(E4m3Shared<256>);
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(attention_e4m3_256),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
    attention_e4m3_256<<<groups, 256, lds, stream>>>(p);
  }
  return hipGetLastError();
}

}  // namespace tge
