// A wave's 16-token tile of K and V, as the decode kernels read and multiply
// it (decode.hip explains the layout).
#pragma once

#include "tc_common.hpp"

#ifndef TC_DECODE_AUX
#define TC_DECODE_AUX 2     // cache-policy bits of the K/V buffer loads (2: non-temporal stream)
#endif

namespace tc {
namespace {

constexpr int kHeadDim = 128;
constexpr int kWaveIter = 16;                        // tokens per wave iteration
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Reductions over the four 16-lane rows of a wave (every lane gets the result).
// v_permlane16_swap(x, x) leaves rows (x0, x0, x2, x2) and (x1, x1, x3, x3) in its two
// results, so their sum is x0 + x1 (x2 + x3) in every lane; permlane32 pairs the halves.
__device__ __forceinline__ float pair16_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float pair32_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float pair16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float rows_sum(float x) { return pair32_sum(pair16_sum(x)); }
__device__ __forceinline__ float rows_max(float x) { return pair32_max(pair16_max(x)); }

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// A wave-uniform read of memory that no kernel writes while this one runs:
// through the constant address space it becomes a scalar load.
__device__ __forceinline__ int32_t const_load(const int32_t* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}

// Buffer resource over `bytes` bytes at p; loads past the end return zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, int32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}

__device__ __forceinline__ uint4 bload16(__amdgpu_buffer_rsrc_t r, int32_t off) {
  const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, TC_DECODE_AUX);
  return make_uint4(v.x, v.y, v.z, v.w);
}

// K/V of one 16-token tile of a wave (lane l = 16 g + n): k[i] = token n,
// dims 32 i + 8 g .. +8 (the A operand of QK block i); v[j] = token 4 g + j,
// dims 8 n .. +8. Rows at or past `end` read as zero (their scores are
// masked), so no index clamping is needed.
struct Tile {
  uint4 k[4];
  uint4 v[4];
  int32_t rows;  // paged cache: the tile's key rows (the rest read as zero)
};

__device__ __forceinline__ void load_tile(Tile& t, const char* kslab, const char* vslab, int32_t row_k,
                                          int32_t row_v, int32_t t0, int32_t end, const int32_t* koff,
                                          const int32_t* voff) {
  // The clamp is wave-uniform, but i32 min/max select v_med3 (a VGPR);
  // readfirstlane keeps the buffer resource in SGPRs (no waterfall loop).
  const int32_t rows = __builtin_amdgcn_readfirstlane(min(max(end - t0, 0), 16));
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(kslab + static_cast<int64_t>(t0) * row_k, rows * row_k);
  const __amdgpu_buffer_rsrc_t rv = make_rsrc(vslab + static_cast<int64_t>(t0) * row_v, rows * row_v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    t.k[j] = bload16(rk, koff[j]);
    t.v[j] = bload16(rv, voff[j]);
  }
}

// Paged cache: rows (<= 16) key rows from slot `slot` of page `page`. The
// buffer range spans exactly those rows, so the rest of the tile reads as
// zero; an entry outside the pool or past the page's end loads nothing.
__device__ __forceinline__ void load_paged_tile(Tile& t, const char* kpool, const char* vpool, int32_t row_k,
                                                int32_t row_v, int64_t page_k, int64_t page_v, int32_t pages,
                                                int32_t page_tokens, int32_t page, int32_t slot, int32_t rows,
                                                const int32_t* koff, const int32_t* voff) {
  if (page < 0 || page >= pages || slot < 0 || rows < 0 || rows > 16 || slot > page_tokens - rows) {
    page = 0; slot = 0; rows = 0;
  }
  t.rows = rows;
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(kpool + page * page_k + static_cast<int64_t>(slot) * row_k, rows * row_k);
  const __amdgpu_buffer_rsrc_t rv = make_rsrc(vpool + page * page_v + static_cast<int64_t>(slot) * row_v, rows * row_v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    t.k[j] = bload16(rk, koff[j]);
    t.v[j] = bload16(rv, voff[j]);
  }
}

typedef _Float16 mfma_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 mfma_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 mfma_b8 __attribute__((ext_vector_type(8)));
typedef short mfma_s4 __attribute__((ext_vector_type(4)));
typedef float mfma_f4 __attribute__((ext_vector_type(4)));

template <int DT> struct DecodeMma;
template <> struct DecodeMma<TC_DTYPE_F16> {
  static __device__ __forceinline__ mfma_f4 qk(const uint4& a, const uint4& b, const mfma_f4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(mfma_h8, a), __builtin_bit_cast(mfma_h8, b), c,
                                                  0, 0, 0);
  }
  static __device__ __forceinline__ mfma_f4 pv(const uint2& a, const uint2& b, const mfma_f4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(mfma_h4, a), __builtin_bit_cast(mfma_h4, b), c,
                                                 0, 0, 0);
  }
  // Two fp32 values rounded to nearest even into one word (first in the low half).
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 v = {static_cast<_Float16>(x), static_cast<_Float16>(y)};
    return __builtin_bit_cast(uint32_t, v);
  }
};
template <> struct DecodeMma<TC_DTYPE_BF16> {
  static __device__ __forceinline__ mfma_f4 qk(const uint4& a, const uint4& b, const mfma_f4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mfma_b8, a), __builtin_bit_cast(mfma_b8, b), c,
                                                   0, 0, 0);
  }
  static __device__ __forceinline__ mfma_f4 pv(const uint2& a, const uint2& b, const mfma_f4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(mfma_s4, a), __builtin_bit_cast(mfma_s4, b),
                                                     c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 v = {static_cast<__bf16>(x), static_cast<__bf16>(y)};
    return __builtin_bit_cast(uint32_t, v);
  }
};

// Row-major V tile in a wave's LDS region: 16 token rows of 256 bytes, each
// padded to 288 so that the transposing reads (4 rows x 32 bytes per 16-lane
// group, 16 rows per instruction) and the 16-byte row stores fall on distinct
// banks.
constexpr int kVRowBytes = 2 * kHeadDim + 32;
constexpr int kVTileWords = 16 * kVRowBytes / 4;
typedef short lds_s4 __attribute__((ext_vector_type(4)));
constexpr float kLazyMax = 8.f;               // log2 units the running maximum may lag

}  // namespace
}  // namespace tc
