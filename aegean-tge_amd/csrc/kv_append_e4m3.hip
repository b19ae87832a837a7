// Append into the e4m3 cache: bias and rotation of q, k and v, the block
// scales, the codes; and the page -> flat-row gather.
//
// A wave owns one part (K or V) of one page block: it reads the block's new
// rows, rotates them, takes the maximum, sets the exponent e (never below the
// block's own while the block holds older rows), encodes x * 2^-e to the
// nearest e4m3 code and writes the part, the slots behind the last new row
// cleared. Since scales are powers of two, older codes change only where e
// grows, and then only those that become subnormal are rounded again.
//
// The maximum of a block needs all its rows before the first code is written,
// so a wave holds a whole part in registers (16 tokens x W dims, 4 W / 16 of
// them a lane), rows are read once and codes leave in whole KiB. Bound by HBM
// for many rows: 20,000 bf16 rows of 4 x 128 dims (61 MB) 14.9 us, 4.1 TB/s, a
// large copy 4.8; 2048 f16 rows of 16/8 x 256 dims with rotation of q and k (62
// MB) 16.6 us, 3.7 TB/s. Few rows cost the launch and the chain tile -> rows ->
// maximum -> codes: one token 4.5 us, 64 sessions with four each 5.6 us.
// Rotated heads as wide as their block keep a dim and its partner in one lane:
// each is loaded once, tables and biases in 16-byte loads (2048 rows 29.1 ->
// 16.6 us).
// This file is built with -ffp-contract=off in addition to the explicit _rn
// intrinsics.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "e4m3_kernels.h"
#include "tge_kv.h"

namespace tge {
namespace {

typedef float float2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float from_bf16(uint32_t bits) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ float from_half(uint32_t bits) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// Eight values of a row (element index `at`, a multiple of 8).
template <int TYPE>
__device__ __forceinline__ void load_row8(float (&x)[8], const void* row, long at) {
  if constexpr (TYPE == TGE_ROWS_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(row) + at);
    const float4 a = p[0], b = p[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const u32x4_t w = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(row) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = TYPE == TGE_ROWS_BF16 ? from_bf16(w[i] & 0xffffu) : from_half(w[i] & 0xffffu);
      x[2 * i + 1] = TYPE == TGE_ROWS_BF16 ? from_bf16(w[i] >> 16) : from_half(w[i] >> 16);
    }
  }
}

// Rounded to nearest even (16-bit types).
template <int TYPE>
__device__ __forceinline__ void store_row8(const float (&x)[8], void* row, long at) {
  if constexpr (TYPE == TGE_ROWS_F32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(row) + at);
    p[0] = make_float4(x[0], x[1], x[2], x[3]);
    p[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t lo, hi;
      if constexpr (TYPE == TGE_ROWS_BF16) {
        lo = __builtin_bit_cast(uint16_t, (__bf16)x[2 * i]);
        hi = __builtin_bit_cast(uint16_t, (__bf16)x[2 * i + 1]);
      } else {
        lo = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i]);
        hi = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]);
      }
      w[i] = lo | hi << 16;
    }
    *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(row) + at) = w;
  }
}

// Eight floats of a table or bias from index `at` (a multiple of 8).
__device__ __forceinline__ void load_f8(float (&x)[8], const float* p, long at) { load_row8<TGE_ROWS_F32>(x, p, at); }

__device__ __forceinline__ void add8(float (&x)[8], const float* bias, int at) {
  if (!bias) return;
  float b[8];
  load_f8(b, bias, at);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __fadd_rn(x[i], b[i]);
}

// One output of the rotation, l*c - h*s or l*s + h*c, with the second product
// rounded, and one rounding of the sum (fma) or of the first product too.
__device__ __forceinline__ float rot(float a, float ca, float b, float cb, bool fma) {
  const float t = __fmul_rn(b, cb);
  return fma ? __fmaf_rn(a, ca, t) : __fadd_rn(__fmul_rn(a, ca), t);
}

// Four codes (bytes in order) of four values scaled by `inv` = 2^-e; a NaN
// is stored as zero, values out of range at the largest code.
__device__ __forceinline__ uint32_t encode4(const float* x, float inv) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float s = __fmul_rn(x[i], inv);
    y[i] = s == s ? fminf(fmaxf(s, -kE4m3Max), kE4m3Max) : 0.0f;
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}

// Four codes times 2^-k as codes (k > 0).
__device__ __forceinline__ uint32_t shrink4(uint32_t w, float factor) {
  const float2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const float2_t b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(__fmul_rn(a[0], factor), __fmul_rn(a[1], factor), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(__fmul_rn(b[0], factor), __fmul_rn(b[1], factor), r, true);
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Eight dims from d0 of a rotated K row: the row's own run and its partner
// half a head away, turned by the position's table row.
template <int TYPE>
__device__ __forceinline__ void rotated_run(float (&x)[8], const E4m3Append& p, const void* rows, long base,
                                            const float* bias, int head_at, int d0, int pos) {
  const int half = p.dims >> 1;
  const bool low = d0 < half;
  const int other = low ? d0 + half : d0 - half, f = low ? d0 : d0 - half;
  float y[8];
  load_row8<TYPE>(x, rows, base + d0);
  load_row8<TYPE>(y, rows, base + other);
  add8(x, bias, head_at + d0);
  add8(y, bias, head_at + other);
  float c[8], s[8];
  load_f8(c, p.rope_cos, (long)pos * half + f);
  load_f8(s, p.rope_sin, (long)pos * half + f);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x[i] = low ? rot(x[i], c[i], y[i], -s[i], p.rope_fma != 0) : rot(y[i], s[i], x[i], c[i], p.rope_fma != 0);
}

// A run of 8 low dims (from f) and its partners, turned together.
template <int TYPE>
__device__ __forceinline__ void rotated_pair(float (&l)[8], float (&h)[8], const E4m3Append& p, const void* rows,
                                             long base, const float* bias, int head_at, int f, int pos) {
  const int half = p.dims >> 1;
  float c[8], s[8];
  load_row8<TYPE>(l, rows, base + f);
  load_row8<TYPE>(h, rows, base + f + half);
  load_f8(c, p.rope_cos, (long)pos * half + f);
  load_f8(s, p.rope_sin, (long)pos * half + f);
  add8(l, bias, head_at + f);
  add8(h, bias, head_at + f + half);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = rot(l[i], c[i], h[i], -s[i], p.rope_fma != 0);
    h[i] = rot(l[i], s[i], h[i], c[i], p.rope_fma != 0);
    l[i] = a;
  }
}

template <int TYPE, int W, bool ROPE>
__device__ __forceinline__ void append_part(const E4m3Append& p, char* stage, const E4m3Tile& t, int h, int part,
                                            int lane) {
  constexpr int U = W / 64;  // KiB of a part
  const size_t n = (size_t)t.page * p.kv_heads + h;
  char* const dst = p.blocks + n * e4m3_block_bytes(W) + part * 16 * W;
  uint16_t* const scale = reinterpret_cast<uint16_t*>(p.scales + n) + part;
  const bool begun = t.slot > 0;
  const int had = begun ? (int)((*scale >> 7) & 0xffu) - 127 : kE4m3MinExp;

  // lane -> token slot and 16 dims of each run of 64
  const int slot = lane & 15, m = lane >> 4;
  const bool live = slot >= t.slot && slot < t.slot + t.count;
  const int row = t.row + (live ? slot - t.slot : 0);
  const void* const rows = part ? p.v : p.k;
  const long base = (long)row * (part ? p.v_stride : p.k_stride) + (long)h * p.dims;
  const float* const bias = part ? p.v_bias : p.k_bias;
  u32x4_t was[U];
  if (begun) {
#pragma unroll
    for (int u = 0; u < U; ++u) was[u] = *reinterpret_cast<const u32x4_t*>(dst + u * 1024 + lane * 16);
  }
  float x[U][2][8];
  // (heads as wide as their blocks of 128 or 256 dims hold a dim's partner in
  // the same lane: one load each)
  const bool paired = ROPE && U > 1 && part == 0 && p.dims == W;
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int d0 = 64 * u + 16 * m + 8 * r;
      if (paired) {
        if (u >= U / 2) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[u][r][i] = x[(u + U / 2) % U][r][i] = 0.0f;
        if (live)
          rotated_pair<TYPE>(x[u][r], x[(u + U / 2) % U][r], p, rows, base, bias, h * p.dims, d0,
                             t.pos + slot - t.slot);
        continue;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[u][r][i] = 0.0f;
      if (live && d0 < p.dims) {
        if (ROPE && part == 0) {
          rotated_run<TYPE>(x[u][r], p, rows, base, bias, h * p.dims, d0, t.pos + slot - t.slot);
        } else {
          load_row8<TYPE>(x[u][r], rows, base + d0);
          if (ROPE) add8(x[u][r], bias, h * p.dims + d0);
        }
      }
    }
  }
  float most = 0.0f;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[u][r][i]));  // (a NaN does not count)
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) most = fmaxf(most, __shfl_xor(most, off));
  const int need = e4m3_exponent(__float_as_uint(most));
  const int e = need > had ? need : had;
  const float inv = pow2f(-e);

  u32x4_t now[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int q = 0; q < 4; ++q) now[u][q] = encode4(&x[u][q >> 1][4 * (q & 1)], inv);
  }
  if (part == 1) {
    // token-major codes into the V order through the wave's LDS
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d = 64 * u + 16 * m + 4 * q;
#pragma unroll
        for (int b = 0; b < 4; ++b) stage[e4m3_v_index(slot, d + b, W)] = (char)(now[u][q] >> (8 * b));
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = *reinterpret_cast<const u32x4_t*>(stage + u * 1024 + lane * 16);
  }
  if (begun) {
    const float factor = pow2f(had - e < -126 ? -126 : had - e);
    // bytes of older rows: K, the lane's token; V, the first tokens of the
    // four that each dword holds
    uint32_t keep;
    if (part == 0) {
      keep = slot < t.slot ? 0xffffffffu : 0u;
    } else {
      const int k = t.slot - 4 * m;  // (m = lane >> 4: the lane's group of four tokens)
      keep = k <= 0 ? 0u : k >= 4 ? 0xffffffffu : (1u << (8 * k)) - 1u;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t o = e > had ? shrink4(was[u][q], factor) : was[u][q];
        now[u][q] = (o & keep) | (now[u][q] & ~keep);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) *reinterpret_cast<u32x4_t*>(dst + u * 1024 + lane * 16) = now[u];
  if (lane == 0) *scale = (uint16_t)((e + 127) << 7);
}

// Workgroups [0, kv_groups): four waves, one (tile, KV head, part) each; the
// rest rotate q, a lane for 8 low dims of a head and their partners.
template <int TYPE, int W, bool ROPE>
__global__ __launch_bounds__(256) void kv_append_e4m3_kernel(E4m3Append p, int kv_groups) {
  __shared__ __align__(16) char stage[4][16 * W];
  if (ROPE && (int)blockIdx.x >= kv_groups) {
    const uint32_t per_head = (uint32_t)p.dims >> 4;
    const uint32_t id = (blockIdx.x - kv_groups) * 256u + threadIdx.x;
    if (id >= (uint32_t)p.n_rows * p.q_heads * per_head) return;
    const int f = (int)(id % per_head) * 8;
    const uint32_t rest = id / per_head;
    const int head = (int)(rest % p.q_heads), row = (int)(rest / p.q_heads);
    float l[8], h[8];
    rotated_pair<TYPE>(l, h, p, p.q, (long)row * p.q_stride + (long)head * p.dims, p.q_bias, head * p.dims, f,
                       p.rows[row].pos);
    const long to = (long)row * p.q_out_stride + (long)head * p.dims + f;
    store_row8<TYPE>(l, p.q_out, to);
    store_row8<TYPE>(h, p.q_out, to + (p.dims >> 1));
    return;
  }
  const int wave = threadIdx.x >> 6;
  const uint32_t unit = blockIdx.x * 4u + wave;
  if (unit >= (uint32_t)p.n_tiles * p.kv_heads * 2u) return;  // whole waves
  const int part = (int)(unit & 1);
  const uint32_t rest = unit >> 1;
  append_part<TYPE, W, ROPE>(p, stage[wave], p.tiles[rest / p.kv_heads], (int)(rest % p.kv_heads), part,
                             threadIdx.x & 63);
}

// One lane for each code; the first lanes of a block take its scales.
__global__ __launch_bounds__(256) void kv_gather_e4m3_kernel(E4m3Gather p) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  const long kvd = (long)p.kv_heads * p.dims;
  if (id >= (long)p.count * kvd) return;
  const int pos = (int)(id / kvd), col = (int)(id % kvd), h = col / p.dims, d = col % p.dims;
  const size_t n = (size_t)p.table[pos >> 4] * p.kv_heads + h;
  const char* blk = p.blocks + n * e4m3_block_bytes(p.width);
  p.k_rows[id] = (uint8_t)blk[e4m3_k_index(pos & 15, d)];
  p.v_rows[id] = (uint8_t)blk[16 * p.width + e4m3_v_index(pos & 15, d, p.width)];
  if ((pos & 15) == 0 && d == 0) {
    const uint32_t s = p.scales[n];
    p.k_scales[(long)(pos >> 4) * p.kv_heads + h] = (uint16_t)s;
    p.v_scales[(long)(pos >> 4) * p.kv_heads + h] = (uint16_t)(s >> 16);
  }
}

template <int TYPE, bool ROPE>
hipError_t launch_append_type(const E4m3Append& p, hipStream_t stream) {
  const long waves = (long)p.n_tiles * p.kv_heads * 2;
  const long kv_groups = (waves + 3) / 4;
  const long q_lanes = ROPE && p.q ? (long)p.n_rows * p.q_heads * (p.dims >> 4) : 0;
  const long groups = kv_groups + (q_lanes + 255) / 256;
  if (groups > 0x7fffffff || waves > 0x7fffffff || q_lanes > 0x7fffffff) return hipErrorInvalidValue;
  const dim3 grid((unsigned)groups);
  if (p.width == 64)
    kv_append_e4m3_kernel<TYPE, 64, ROPE><<<grid, 256, 0, stream>>>(p, (int)kv_groups);
  else if (p.width == 128)
    kv_append_e4m3_kernel<TYPE, 128, ROPE><<<grid, 256, 0, stream>>>(p, (int)kv_groups);
  else
    kv_append_e4m3_kernel<TYPE, 256, ROPE><<<grid, 256, 0, stream>>>(p, (int)kv_groups);
  return hipGetLastError();
}

template <int TYPE>
hipError_t launch_append(const E4m3Append& p, hipStream_t stream) {
  return p.rope_cos ? launch_append_type<TYPE, true>(p, stream) : launch_append_type<TYPE, false>(p, stream);
}

}  // namespace

hipError_t launch_e4m3_append(const E4m3Append& p, hipStream_t stream) {
  if (p.row_type == TGE_ROWS_BF16) return launch_append<TGE_ROWS_BF16>(p, stream);
  if (p.row_type == TGE_ROWS_F16) return launch_append<TGE_ROWS_F16>(p, stream);
  return launch_append<TGE_ROWS_F32>(p, stream);
}

hipError_t launch_e4m3_gather(const E4m3Gather& p, hipStream_t stream) {
  const long n = (long)p.count * p.kv_heads * p.dims;
  if (n == 0) return hipSuccess;
  if ((n + 255) / 256 > 0x7fffffff) return hipErrorInvalidValue;
  kv_gather_e4m3_kernel<<<dim3((unsigned)((n + 255) / 256)), 256, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace tge
