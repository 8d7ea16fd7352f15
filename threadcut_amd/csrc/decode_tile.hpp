// The decode partial pass as device code: a wave's 16-token tiles of K and V
// (decode.hip explains the layout), the arguments of a call and the work of one
// (split, KV head, sequence), for decode.hip's kernel and shared.hip's.
#pragma once

#include "tc_common.hpp"

#ifndef TC_DECODE_AUX
#define TC_DECODE_AUX 2     // cache-policy bits of the K/V buffer loads (2: non-temporal stream)
#endif

#ifndef TC_DECODE_STAMPS
#define TC_DECODE_STAMPS 0  // 1: the measurement build; every partial wave records a timeline
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

struct PartialArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  float* o_part;       // [B, H, S, G, D]
  float* lse_part;     // [B, H, S, G]
  const int32_t* lens; // [B] or null
  int64_t n;
  int64_t sq_b, sq_h, sq_g;
  int64_t sk_b, sk_h, sk_t;
  int64_t sv_b, sv_h, sv_t;
  int heads, group, splits, split_tokens;
  int interleave;      // 0: split s owns tokens [s*T, (s+1)*T); 1: 16-token tiles dealt round-robin
  int longest_first;   // per-sequence lengths, batch <= 64: work-group row z serves the z-th longest sequence
  float scale_log2;    // softmax scale * log2(e)
  // Append (k_new != null): the cache holds n - 1 tokens and the new token's
  // K/V rows [B, H, D] are attended from k_new/v_new and written to row n - 1
  // of the cache (k_w/v_w) by wave 0 of split 0; no other wave reads that row.
  const uint16_t* k_new;
  const uint16_t* v_new;
  int64_t skn_b, skn_h, svn_b, svn_h;
  uint16_t* k_w;
  uint16_t* v_w;
  // Paged cache (decode_partial_kernel<DT, true, ...>): k and v are page pools
  // [pages, H, P, D] with element strides (sk_b, sk_h, sk_t) = (page, head,
  // token). Sequence b's keys are the tiles tile_tab[b * max_tiles + i],
  // i < tiles[b], each {page, first slot, rows, 0}: rows (<= 16) consecutive
  // slots of one page. Entries outside the pool or the page count as empty.
  const int32_t* tile_tab;
  const int32_t* tiles;
  int64_t max_tiles;
  int32_t pages, page_tokens;
  // Paged append with device lengths (tok_off != null): sequence b holds
  // lens[b] tokens before this step; tile entries carry their first logical
  // position in the 4th word, and a tile's rows are those below lens[b]
  // (tiles reserved ahead read nothing). The new token goes to logical
  // position lens[b], whose row sits tok_off[b * tok_pitch + lens[b]] bytes
  // into the head slab of the pools.
  const int32_t* tok_off;
  int64_t tok_pitch;
  // One split: the result itself, rounded to the element type as the combine
  // rounds it (null: the partial goes to o_part, lse_part).
  uint16_t* out;
  int64_t so_b, so_h, so_g;
  // Window (decode_partial_kernel<..., true>): sequence b's query sees its last
  // `window` tokens, an appended one among them, and the first `sinks` ones.
  int32_t window, sinks;
  // Beside another part's splits (decode_partial<..., true>): a (sequence,
  // head) has part_splits of them in o_part and lse_part, which point at this
  // call's first.
  int part_splits;
#if TC_DECODE_STAMPS
  // Per wave ((b * heads + h) * splits + split) * waves + wave, 8 words:
  // realtime-clock stamps (100 MHz) at the kernel's start, after the first
  // tile's step, at the loop's end, after the merge barrier and after the
  // partial stores are issued, then HW_REG_HW_ID and HW_REG_XCC_ID.
  unsigned long long* stamps;
#endif
};

namespace {

// APPEND: the kernel attends (and writes) the new token of an append call
// (a.k_new != null); DIRECT: it writes the result (a.out != null), of one
// split. WINDOW (contiguous caches, tiles dealt round-robin): only the first
// a.sinks tokens and the last a.window are read: the tokens between the two
// are left out of the index space that the tiles are dealt from, in which the
// window follows the sinks' last, perhaps partial, tile. Nothing else of the
// cache is read, and the split plan goes by that space: 16 sequences of 1k to
// 32k tokens, a window of 4096 and 16 sinks (bf16, 259 MB): 46 us with the
// combine, 5.6 TB/s; one of 10240, window 1024: 4.4 us and 2.7 for the combine,
// two launches' time. The other instantiations carry none of that code.
// The work of W waves, which may be a work-group of its own or a part of one (tid is the thread's index in it): head h's
// split `split` of the z-th of `sequences` sequences. s_vt: the waves' V tiles; s_acc, s_m and s_l: the merge's rows,
// padded by 16 words, so the float4 stores of the g heads (one head per 16 lanes) fall on distinct banks.
template <int DT, bool PAGED, bool APPEND, bool DIRECT, int W, bool WINDOW, bool BESIDE>
__device__ __forceinline__ void decode_partial(const PartialArgs& a, const int h, const int split, const int z,
                                               const int sequences, const int tid, uint32_t (*s_vt)[kVTileWords],
                                               float (*s_acc)[8][kHeadDim + 16], float (*s_m)[W], float (*s_l)[W]) {
  using M = DecodeMma<DT>;
  using E = Elem<DT>;
#if TC_DECODE_STAMPS
  const unsigned long long st_start = __builtin_amdgcn_s_memrealtime();
  unsigned long long st_first = 0, st_loop = 0, st_merge = 0;
#endif
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15;   // head column (also the token row of the K operand)
  const int g = lane >> 4;   // lane group
  // With per-sequence lengths the work-groups of the z-th longest sequence
  // take grid row z, so the longest sequences are dispatched first (ties by
  // index): lane j ranks sequence j by length, and the ballot finds the lane
  // of rank z.
  int b = z;
  int32_t len_b = 0;  // longest-first: sequence b's length, read with the others
  if (!PAGED && a.longest_first) {
    const int B = sequences;
    const int32_t mine = lane < B ? a.lens[lane] : 0;
    int rank = 0;
    for (int i = 0; i < B; ++i) {
      const int32_t other = __builtin_amdgcn_readlane(mine, i);
      rank += (other > mine || (other == mine && i < lane)) ? 1 : 0;
    }
    const uint64_t hit = __builtin_amdgcn_ballot_w64(lane < B && rank == z);
    b = hit ? __builtin_ctzll(hit) : b;
    len_b = __builtin_amdgcn_readlane(mine, b);
  }

  // Paged: the pools' head slabs, pages added per tile; otherwise sequence b's slabs.
  const char* kslab = reinterpret_cast<const char*>(a.k + (PAGED ? 0 : b * a.sk_b) + h * a.sk_h);
  const char* vslab = reinterpret_cast<const char*>(a.v + (PAGED ? 0 : b * a.sv_b) + h * a.sv_h);
  const int32_t row_k = static_cast<int32_t>(a.sk_t) * 2, row_v = static_cast<int32_t>(a.sv_t) * 2;
  __asm__ volatile("" ::"s"(kslab), "s"(vslab));
  const int32_t nt = static_cast<int32_t>(a.n);
  const int32_t len_cap = APPEND ? nt - 1 : nt;
  // The wave's first tile and the distance between its tiles.
  int32_t tok, tok_step, wave_tokens = 0;
  if (a.interleave) {
    tok = (split * W + wave) * kWaveIter;
    tok_step = a.splits * W * kWaveIter;
  } else {
    wave_tokens = a.split_tokens / W;
    tok = split * a.split_tokens + wave * wave_tokens;
    tok_step = kWaveIter;
  }
  const int32_t* tab = PAGED ? a.tile_tab + static_cast<int64_t>(b) * a.max_tiles * 4 : nullptr;
  // Paged: lane i holds the table entry of the wave's i-th tile (tiles past
  // the 64th read theirs from memory). The entries are requested before the
  // tile count is known, bounded by the table's row, so the two reads are in
  // flight together.
  int32_t e_page = 0, e_slot = 0, e_cnt = 0, e_pos = 0;
  const int32_t ti = tok + lane * tok_step;
  if constexpr (PAGED) {
    if ((ti >> 4) < a.max_tiles) {
      const int4 e = *reinterpret_cast<const int4*>(tab + 4 * (ti >> 4));
      e_page = e.x; e_slot = e.y; e_cnt = e.z; e_pos = e.w;
    }
  }
  int32_t len = len_cap;
  int32_t last_tile = -1;  // paged append: the tile whose last row is the new token's slot
  int32_t plen = -1;  // paged append with device lengths: tokens cached before this step
  if constexpr (PAGED) {
    // Token index space of 16 per tile; a tile's own row count masks the rest.
    // The tile count and lengths are read with scalar loads (constant for the
    // kernel's lifetime).
    const int32_t ntiles = min(max(const_load(a.tiles + b), 0), static_cast<int32_t>(a.max_tiles));
    len = 16 * ntiles;
    if (a.tok_off) plen = max(const_load(a.lens + b), 0);
    else if (APPEND)
      last_tile = ntiles - 1;
  } else if (a.lens) {
    len = min(max(a.longest_first ? len_b : a.lens[b], 0), len_cap);
  }
  // The window's first token, and where it stands in the index space of the
  // tiles (0: the sequence is read whole).
  int32_t win0 = 0, win_at = 0;
  const int32_t last = len;  // tokens in the cache
  if constexpr (WINDOW) {
    win0 = __builtin_amdgcn_readfirstlane(max(len + (APPEND ? 1 : 0) - a.window, 0));
    if (win0 > a.sinks) {
      win_at = (a.sinks + kWaveIter - 1) / kWaveIter * kWaveIter;
      len = win_at + last - win0;
    } else {
      win0 = 0;
    }
  }
  const int32_t end = a.interleave ? len : min(tok + wave_tokens, len);

  // K: token n of the tile, bytes [64 i + 16 g, +16) for block i.
  // V: tokens 4g + j, dims 8n .. 8n + 7.
  int32_t koff[4], voff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    koff[i] = n * row_k + 64 * i + 16 * g;
    voff[i] = (4 * g + i) * row_v + 16 * n;
  }
  // Rows each preloaded tile contributes: none past the wave's tiles; the
  // append's last tile less the new token's row (attended from k_new); with
  // device lengths, the rows below lens[b].
  int32_t e_rows = 0;
  if constexpr (PAGED) {
    if (ti < end) {
      e_rows = (ti >> 4) == last_tile ? e_cnt - 1 : e_cnt;
      if (plen >= 0) e_rows = min(e_cnt, max(plen - e_pos, 0));
    }
  }
  int32_t li = 0;  // the wave's tiles loaded so far
  auto load = [&](Tile& tl, int32_t t0) {
    if constexpr (PAGED) {
      int32_t page = 0, slot = 0, rows = 0;
      if (li < 64) {
        page = __builtin_amdgcn_readlane(e_page, li);
        slot = __builtin_amdgcn_readlane(e_slot, li);
        rows = __builtin_amdgcn_readlane(e_rows, li);
      } else if (t0 < end) {
        const int4 e = *reinterpret_cast<const int4*>(tab + 4 * (t0 >> 4));
        page = __builtin_amdgcn_readfirstlane(e.x);
        slot = __builtin_amdgcn_readfirstlane(e.y);
        int32_t r = (t0 >> 4) == last_tile ? e.z - 1 : e.z;
        if (plen >= 0) r = min(e.z, max(plen - e.w, 0));
        rows = __builtin_amdgcn_readfirstlane(r);
      }
      ++li;
      load_paged_tile(tl, kslab, vslab, row_k, row_v, a.sk_b * 2, a.sv_b * 2, a.pages, a.page_tokens, page, slot,
                      rows, koff, voff);
    } else if constexpr (WINDOW) {
      const bool sink = t0 < win_at;
      const int32_t at = sink || t0 >= end ? t0 : t0 - win_at + win0;
      load_tile(tl, kslab, vslab, row_k, row_v, t0 < end ? at : 0, t0 >= end ? 0 : sink ? a.sinks : last, koff, voff);
    } else {
      load_tile(tl, kslab, vslab, row_k, row_v, t0, end, koff, voff);
    }
  };
  // The index at which the keys of the tile at t0 end.
  auto limit = [&](const Tile& tl, int32_t t0) -> int32_t {
    if constexpr (PAGED) return t0 + tl.rows;
    if constexpr (WINDOW) return t0 < win_at ? a.sinks : end;
    return end;
  };
  Tile t[2];
  load(t[0], tok);

  // Q as the B operand: head n, dims 32 i + 8 g .. +8 (zero for n >= G).
  uint4 qb[4];
  {
    const uint16_t* qrow = a.q + b * a.sq_b + h * a.sq_h + n * a.sq_g + 8 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      qb[i] = make_uint4(0u, 0u, 0u, 0u);
      if (n < a.group) qb[i] = *reinterpret_cast<const uint4*>(qrow + 32 * i);
    }
  }

  mfma_f4 acc[8];
#pragma unroll
  for (int bm = 0; bm < 8; ++bm) acc[bm] = mfma_f4{0.f, 0.f, 0.f, 0.f};
  float m = neg_inf(), l = 0.f;

  // One 16-token tile whose first token is t0 (tokens >= lim are masked).
  auto step = [&](const Tile& tl, int32_t t0, int32_t lim) {
    // S^T block: two independent chains of two MFMAs each.
    mfma_f4 s0 = M::qk(tl.k[0], qb[0], mfma_f4{0.f, 0.f, 0.f, 0.f});
    mfma_f4 s1 = M::qk(tl.k[1], qb[1], mfma_f4{0.f, 0.f, 0.f, 0.f});
    s0 = M::qk(tl.k[2], qb[2], s0);
    s1 = M::qk(tl.k[3], qb[3], s1);
    // V into LDS, row-major, while the matrix core works: lane (g, n)
    // stores tokens 4g + j, dims 8n .. 8n + 7.
    char* vrow = reinterpret_cast<char*>(s_vt[wave]);
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(vrow + (4 * g + j) * kVRowBytes + 16 * n) = tl.v[j];
    float x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      x[r] = (t0 + 4 * g + r < lim) ? (s0[r] + s1[r]) * a.scale_log2 : neg_inf();
    const float tmax = rows_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    // Lazy running maximum: moves only when the tile's exceeds it by kLazyMax.
    const float mn = (tmax > m + kLazyMax || m == neg_inf()) ? tmax : m;
    const float ms = (mn == neg_inf()) ? 0.f : mn;
    // Rescale what was accumulated (nothing while m is still -inf: acc and l are zero).
    if (__any(mn != m && m != neg_inf())) {
      const float alpha = __builtin_amdgcn_exp2f(m - ms);  // 0 while nothing was seen
#pragma unroll
      for (int bm = 0; bm < 8; ++bm) acc[bm] *= alpha;
      l *= alpha;
    }
    m = mn;
    float p[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(x[r] - ms);
    l += (p[0] + p[1]) + (p[2] + p[3]);
    const uint32_t h01 = M::pack(p[0], p[1]), h23 = M::pack(p[2], p[3]);
    const uint32_t r01 = M::pack(p[0] - E::lo(h01), p[1] - E::hi(h01));
    const uint32_t r23 = M::pack(p[2] - E::lo(h23), p[3] - E::hi(h23));
    const uint2 phi = make_uint2(h01, h23), plo = make_uint2(r01, r23);
#pragma unroll
    for (int bm = 0; bm < 8; ++bm) {
      // A operand V^T[16 bm + n][4g .. 4g + 3]: ds_read_b64_tr_b16 hands lane n
      // of a 16-lane group element (n % 4) of what lane 4 j + n / 4 addressed,
      // for j = 0..3; lane (g, n) addresses row 4g + n / 4, dims 16 bm + 4 (n % 4).
      const lds_s4 t4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) lds_s4*)(vrow + (4 * g + (n >> 2)) * kVRowBytes + 32 * bm + 8 * (n & 3)));
      const uint2 av = __builtin_bit_cast(uint2, t4);
      acc[bm] = M::pv(av, phi, acc[bm]);
      acc[bm] = M::pv(av, plo, acc[bm]);
    }
  };

  // Two tiles in flight: the next tile's loads are issued before the current
  // tile is consumed, and no load is issued past the wave's last tile.
  if (tok < end) {
    for (;;) {
      const int32_t tok1 = tok + tok_step, tok2 = tok1 + tok_step;
      load(t[1], tok1);
      step(t[0], tok, limit(t[0], tok));
#if TC_DECODE_STAMPS
      if (st_first == 0) st_first = __builtin_amdgcn_s_memrealtime();
#endif
      load(t[0], tok2);
      if (tok1 < end) step(t[1], tok1, limit(t[1], tok1));
      tok = tok2;
      if (tok >= end) break;
    }
  }

  if (APPEND && split == 0 && wave == 0) {
    // The appended token as a tile whose only row is token 0 (the buffer
    // range is one row, so the other rows read zero and are masked). Before
    // the wave's own tiles it holds them up: 11.9 against 11.5 us at 10240
    // tokens, 8.4 against 7.9 at 4000.
    const char* kn = reinterpret_cast<const char*>(a.k_new + b * a.skn_b + h * a.skn_h);
    const char* vn = reinterpret_cast<const char*>(a.v_new + b * a.svn_b + h * a.svn_h);
    const __amdgpu_buffer_rsrc_t rk = make_rsrc(kn, kHeadDim * 2);
    const __amdgpu_buffer_rsrc_t rv = make_rsrc(vn, kHeadDim * 2);
    Tile tn;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      tn.k[j] = bload16(rk, 64 * j + 16 * g + n * kHeadDim * 2);
      tn.v[j] = bload16(rv, (4 * g + j) * kHeadDim * 2 + 16 * n);
    }
    step(tn, 0, 1);
    if (lane < 32) {
      const bool is_v = lane >= 16;
      const int chunk = 8 * (lane & 15);
      const uint16_t* src = is_v ? a.v_new + b * a.svn_b + h * a.svn_h : a.k_new + b * a.skn_b + h * a.skn_h;
      uint16_t* dst = nullptr;
      if constexpr (PAGED) {
        // The new token's slot: with device lengths, the offset table's row of
        // position lens[b] (a position past the table's rows, or an offset
        // outside the pool, writes nothing); otherwise the last row of the
        // sequence's last tile (an invalid entry, or no tile, writes nothing).
        if (plen >= 0) {
          const int32_t off = plen < a.tok_pitch ? a.tok_off[static_cast<int64_t>(b) * a.tok_pitch + plen] : -1;
          const int64_t room = static_cast<int64_t>(a.pages) * a.sk_b * 2 - h * a.sk_h * 2 - kHeadDim * 2;
          if (off >= 0 && off <= room) {
            char* base = reinterpret_cast<char*>(is_v ? a.v_w + h * a.sv_h : a.k_w + h * a.sk_h);
            dst = reinterpret_cast<uint16_t*>(base + off);
          }
        } else if (last_tile >= 0) {
          const int4 e = *reinterpret_cast<const int4*>(tab + 4 * last_tile);
          if (!(e.x < 0 || e.x >= a.pages || e.y < 0 || e.z < 1 || e.z > 16 || e.y > a.page_tokens - e.z)) {
            const int64_t slot = e.y + e.z - 1;
            dst = is_v ? a.v_w + e.x * a.sv_b + h * a.sv_h + slot * a.sv_t
                       : a.k_w + e.x * a.sk_b + h * a.sk_h + slot * a.sk_t;
          }
        }
      } else {
        dst = is_v ? a.v_w + b * a.sv_b + h * a.sv_h + last * a.sv_t : a.k_w + b * a.sk_b + h * a.sk_h + last * a.sk_t;
      }
      if (dst) *reinterpret_cast<uint4*>(dst + chunk) = *reinterpret_cast<const uint4*>(src + chunk);
    }
  }

#if TC_DECODE_STAMPS
  st_loop = __builtin_amdgcn_s_memrealtime();
  auto record = [&]() {
    if (a.stamps && lane == 0) {
      unsigned long long* o =
          a.stamps + (((static_cast<int64_t>(b) * a.heads + h) * a.splits + split) * W + wave) * 8;
      o[0] = st_start; o[1] = st_first; o[2] = st_loop; o[3] = st_merge;
      o[4] = __builtin_amdgcn_s_memrealtime();
      o[5] = __builtin_amdgcn_s_getreg((31 << 11) | (0 << 6) | 4);   // HW_REG_HW_ID
      o[6] = __builtin_amdgcn_s_getreg((15 << 11) | (0 << 6) | 20);  // HW_REG_XCC_ID
    }
  };
#endif
  // The head's sum over the four lane groups; m is already common to them.
  l = rows_sum(l);
  const int64_t part = (static_cast<int64_t>(b) * a.heads + h) * (BESIDE ? a.part_splits : a.splits) + split;
  static_assert(W > 1, "the waves of a work-group are merged below");
  if (n < a.group) {
#pragma unroll
    for (int bm = 0; bm < 8; ++bm)
      *reinterpret_cast<float4*>(&s_acc[wave][n][16 * bm + 4 * g]) =
          make_float4(acc[bm][0], acc[bm][1], acc[bm][2], acc[bm][3]);
    if (g == 0) { s_m[n][wave] = m; s_l[n][wave] = l; }
  }
  // The split's output rows, addressed before the barrier (the address
  // arithmetic is then off the path from the barrier to the stores).
  float* const o_out = a.o_part + part * a.group * kHeadDim;
  float* const l_out = a.lse_part + part * a.group;
  __asm__ volatile("" ::"s"(o_out), "s"(l_out));
  __syncthreads();
#if TC_DECODE_STAMPS
  st_merge = __builtin_amdgcn_s_memrealtime();
#endif

  // Each thread merges two adjacent dims of one head (one pass for G <= 4).
  for (int idx = tid; idx < a.group * (kHeadDim / 2); idx += 64 * W) {
    const int hh = idx / (kHeadDim / 2);
    const int d = 2 * (idx % (kHeadDim / 2));
    float mw[W], lw[W];
    float2 ow[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      mw[w] = s_m[hh][w];
      lw[w] = s_l[hh][w];
      ow[w] = *reinterpret_cast<const float2*>(&s_acc[w][hh][d]);
    }
    float Mx = neg_inf();
#pragma unroll
    for (int w = 0; w < W; ++w) Mx = fmaxf(Mx, mw[w]);
    const float Ms = (Mx == neg_inf()) ? 0.f : Mx;
    float L = 0.f, O0 = 0.f, O1 = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(mw[w] - Ms);
      L += lw[w] * f;
      O0 += ow[w].x * f;
      O1 += ow[w].y * f;
    }
    // L >= 1 whenever a token was seen (the maximum contributes exp2(0)).
    const float inv = L == 0.f ? 0.f : __builtin_amdgcn_rcpf(L);
    float2 y = make_float2(O0 * inv, O1 * inv);
    if constexpr (DIRECT) {
      // Rounded to fp32 and then to the element type, as the combine reads and
      // writes it (the compiler would take both steps in one v_fma_mix).
      __asm__("" : "+v"(y.x), "+v"(y.y));
      uint16_t* dst = a.out + b * a.so_b + h * a.so_h + hh * a.so_g + d;
      *reinterpret_cast<uint32_t*>(dst) = E::bits(y.x) | (E::bits(y.y) << 16);
      continue;
    }
    *reinterpret_cast<float2*>(o_out + hh * kHeadDim + d) = y;
    if (d == 0) l_out[hh] = (L == 0.f) ? neg_inf() : (Mx + __builtin_amdgcn_logf(L)) * kLn2;
  }
#if TC_DECODE_STAMPS
  record();
#endif
}

}  // namespace
}  // namespace tc
