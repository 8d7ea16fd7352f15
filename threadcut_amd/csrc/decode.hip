// Split-KV GQA flash-decode for gfx950: a partial online-softmax kernel over
// (split, kv head, sequence) work-groups on the matrix cores, and a separate
// log-sum-exp combine.
//
// Reference semantics: threadcut/flash_decode.py:21-54 (`_partial`: fp32
// softmax, scale applied after q.k, -inf guards, out = acc / l,
// lse = m + log l) and :57-69 (decode_attention: splits = cdiv(n, split),
// merge with softmax(lse) weights, cast to q.dtype).
//
// Per wave and 16-token tile, with n = lane % 16 (query head: a column of
// every 16x16 MFMA block; columns n >= G hold zeros) and g = lane / 16:
//   S^T[token][head] = K[token][:] . Q[head][:]   four v_mfma_f32_16x16x32
//     (k = 32 dims each). A = K rows: lane l loads token l % 16, bytes
//     [64 i + 16 g, +16) of its row for block i, so each load instruction
//     reads 16 rows x 64 contiguous bytes; B = Q with the same dims, held in
//     registers for the whole kernel. Lane l receives S^T[4g + r][n], r < 4.
//   softmax per head in fp32, log2 domain, the tile maximum across the four
//     lane groups by two permlane swaps; the running maximum moves only when
//     a tile's exceeds it by 2^8 (p is then at most 2^8), so the accumulators
//     are rescaled rarely.
//   O^T[dim][head] += V^T[dim][token] . P^T[token][head]   eight
//     v_mfma_f32_16x16x16 (k = 16 tokens), each twice: with P rounded to the
//     element type and with the rounding residue, so the weights carry about
//     16 (bf16) or 22 (fp16) significant bits. P^T leaves the S^T registers as
//     the B operand without moving between lanes (lane l holds tokens
//     4g..4g+3 of head n in both layouts). V is loaded as 4 tokens x 8 dims
//     per lane and stored row-major to the wave's own LDS region (16-byte
//     stores, rows padded to 288 bytes); the A operand V^T comes back through
//     the transposing ds_read_b64_tr_b16, so V is never transposed in
//     registers.
// The matrix core sums over a wave's tokens, so a wave's accumulator is
// complete; the four waves of a work-group are merged through LDS and the
// work-group writes one (o, lse) partial per query head.

#include <math.h>

#include <algorithm>
#include <mutex>

#include "decode_tile.hpp"
#include "shared.hpp"

namespace tc {
namespace {

// Tuning knobs (measured on MI355X; override with -D for sweeps).
#ifndef TC_DECODE_WAVES
#define TC_DECODE_WAVES 4   // waves per partial work-group
#endif
#ifndef TC_DECODE_INTERLEAVE
#define TC_DECODE_INTERLEAVE 1  // tc_decode_attention deals tiles round-robin over the splits
#endif
#ifndef TC_DECODE_RAGGED_WGS_PER_CU
#define TC_DECODE_RAGGED_WGS_PER_CU 8  // at most, with per-sequence lengths: finer splits balance them
#endif
#ifndef TC_DECODE_WGS_PER_CU
#define TC_DECODE_WGS_PER_CU 1  // partial work-groups per compute unit the split heuristic aims at
#endif
#ifndef TC_DECODE_WPE
#define TC_DECODE_WPE 1  // amdgpu_waves_per_eu floor of the partial kernel (2 caps a wave at 256 registers)
#endif
#ifndef TC_DECODE_WPE_PAGED
#define TC_DECODE_WPE_PAGED 2  // the same for the paged instantiations
#endif

constexpr int64_t kMaxTokens = int64_t(1) << 29;  // token positions stay 32-bit in the kernel
constexpr int kWaves = TC_DECODE_WAVES;
// Short caches (at most TC_DECODE_SHORT_TOKENS tokens, one length for the
// batch): partial work-groups of two waves over the same splits. A wave then
// has two tiles where it had one, and the merge of two waves costs less than
// that of four (36 layers, Qwen3-4B heads, call us: 512 tokens 5.76 against
// 5.87, 1024 5.89 against 6.02, 1536 6.05 against 6.25, 2048 6.50 against
// 6.84; at 3072 and 4096 tokens two waves are slower).
constexpr int kShortWaves = 2;
constexpr int kSplitGranule = kWaves * kWaveIter > 64 ? kWaves * kWaveIter : 64;  // split length granule
static_assert(kSplitGranule % (kShortWaves * kWaveIter) == 0, "short plans split at the same granule");

struct CombineArgs {
  const float* o_part;
  const float* lse_part;
  uint16_t* out;
  int64_t so_b, so_h, so_g;
  int heads, group, splits;
};

// Grid (heads, splits, batch), the KV head fastest: consecutive work-groups go
// to consecutive XCDs, so with 8 KV heads every split of head h runs on XCD h
// and its partials stay in that XCD's L2 for the combine. W waves per
// work-group: kWaves, or kShortWaves for short caches.
template <int DT, bool PAGED, bool APPEND, bool DIRECT, int W, bool WINDOW = false>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(PAGED ? TC_DECODE_WPE_PAGED : TC_DECODE_WPE))) void decode_partial_kernel(const PartialArgs a) {
  __shared__ uint32_t s_vt[W][kVTileWords];
  __shared__ float s_acc[W][8][kHeadDim + 16];
  __shared__ float s_m[8][W];
  __shared__ float s_l[8][W];
  decode_partial<DT, PAGED, APPEND, DIRECT, W, WINDOW, false>(a, blockIdx.x, blockIdx.y, blockIdx.z, gridDim.z, threadIdx.x, s_vt,
                                                       s_acc, s_m, s_l);
}

// x of the lane pair (l, l ^ 16) or (l, l ^ 32): the lower row's value in lo,
// the upper row's in hi, in both lanes.
template <bool ROW32>
__device__ __forceinline__ void swap_pair(float x, float& lo, float& hi) {
  const uint32_t u = __float_as_uint(x);
  const auto r = ROW32 ? __builtin_amdgcn_permlane32_swap(u, u, false, false)
                       : __builtin_amdgcn_permlane16_swap(u, u, false, false);
  lo = __uint_as_float(r[0]);
  hi = __uint_as_float(r[1]);
}

// x of lanes l and l ^ K (K = 8: DPP row rotate by 8; 16, 32: permlane swaps),
// the lower lane's value in lo, the upper lane's in hi, in both lanes.
template <int K>
__device__ __forceinline__ void lane_pair(float x, int lane, float& lo, float& hi) {
  if constexpr (K == 8) {
    const float o = __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x128, 0xf, 0xf, false));  // row_ror:8
    const bool upper = (lane & 8) != 0;
    lo = upper ? o : x;
    hi = upper ? x : o;
  } else {
    swap_pair<K == 32>(x, lo, hi);
  }
}
// One merge step of the (max, sum, weighted o) states of lanes l and l ^ K,
// lower lane first, so both lanes hold the same bits afterwards.
template <int K>
__device__ __forceinline__ void combine_merge(float& M, float& L, float4& O, int lane) {
  float m0, m1, x0, x1;
  lane_pair<K>(M, lane, m0, m1);
  const float Mx = fmaxf(m0, m1);
  const float Ms = (Mx == neg_inf()) ? 0.f : Mx;
  const float f0 = __builtin_amdgcn_exp2f((m0 - Ms) * kLog2e);
  const float f1 = __builtin_amdgcn_exp2f((m1 - Ms) * kLog2e);
  lane_pair<K>(L, lane, x0, x1); L = x0 * f0 + x1 * f1;
  lane_pair<K>(O.x, lane, x0, x1); O.x = x0 * f0 + x1 * f1;
  lane_pair<K>(O.y, lane, x0, x1); O.y = x0 * f0 + x1 * f1;
  lane_pair<K>(O.z, lane, x0, x1); O.z = x0 * f0 + x1 * f1;
  lane_pair<K>(O.w, lane, x0, x1); O.w = x0 * f0 + x1 * f1;
  M = Mx;
}

// Combine: one wave per (sequence, KV head, query head, quarter of the dims),
// grid (heads, batch, group * 4), the KV head fastest, so with 8 heads head
// h's waves run on XCD h, where the partial kernel wrote its partials. Lane
// (sg, chunk) takes dims 32 q + 4 chunk .. + 3 of splits sg, sg + 8, sg + 16,
// ...: four splits a lane per round of 32, every load of a round issued before
// the first is consumed (one memory round trip per round). Each round folds
// its splits into a running (max, sum, weighted o) with one exponential per
// split; the eight split groups are then merged across lanes (a DPP row
// rotate, permlane16 and permlane32 swaps). Spreading a head's dims over four
// waves keeps each wave's loads to 8 a round (the one-wave-per-head form
// issued 32).
template <int DT>
__global__ __launch_bounds__(64) void decode_combine_kernel(const CombineArgs a) {
  using E = Elem<DT>;
  constexpr int kPer = 4;  // splits a lane loads per round
  const int lane = threadIdx.x;
  const int chunk = lane & 7;
  const int sg = lane >> 3;
  const int h = blockIdx.x;
  const int b = blockIdx.y;
  const int g = blockIdx.z >> 2;
  const int qtr = blockIdx.z & 3;
  const int G = a.group;
  const int S = a.splits;
  const int64_t bh = static_cast<int64_t>(b) * a.heads + h;
  // Buffer ranges over this (sequence, head)'s partials: loads past them read zero.
  const __amdgpu_buffer_rsrc_t ro = make_rsrc(a.o_part + bh * S * G * kHeadDim, S * G * kHeadDim * 4);
  const __amdgpu_buffer_rsrc_t rl = make_rsrc(a.lse_part + bh * S * G, S * G * 4);
  // Per-lane byte offsets (split sg of a round); the round's split r0 + 8 j
  // adds a wave-uniform offset.
  const int32_t o_split = G * kHeadDim * 4;  // bytes between splits
  const int32_t o_lane = sg * o_split + (g * kHeadDim + 32 * qtr + 4 * chunk) * 4;
  const int32_t l_lane = (sg * G + g) * 4;

  float M = neg_inf(), L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int r0 = 0; r0 < S; r0 += 8 * kPer) {
    u32x4 ov[kPer];
    float ls[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int32_t s0 = r0 + 8 * j;
      // The buffer range check covers the scalar offset too (measured on
      // gfx950), so splits past S read zero.
      ov[j] = __builtin_amdgcn_raw_buffer_load_b128(ro, o_lane, s0 * o_split, 0);
      ls[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rl, l_lane, s0 * G * 4, 0));
    }
    // Every load of the round is in flight before the first is consumed.
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (r0 + 8 * j + sg >= S) ls[j] = neg_inf();  // past the last split (the load read zero)
    float mr = ls[0];
#pragma unroll
    for (int j = 1; j < kPer; ++j) mr = fmaxf(mr, ls[j]);
    const float Mn = fmaxf(M, mr);
    const float Ms = (Mn == neg_inf()) ? 0.f : Mn;
    const float f = __builtin_amdgcn_exp2f((M - Ms) * kLog2e);  // 0 while nothing was seen
    L *= f;
    O.x *= f; O.y *= f; O.z *= f; O.w *= f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const float w = __builtin_amdgcn_exp2f((ls[j] - Ms) * kLog2e);
      L += w;
      O.x += w * __uint_as_float(ov[j].x);
      O.y += w * __uint_as_float(ov[j].y);
      O.z += w * __uint_as_float(ov[j].z);
      O.w += w * __uint_as_float(ov[j].w);
    }
    M = Mn;
  }
  // Merge the split groups: lanes l ^ 8, l ^ 16 and l ^ 32.
  combine_merge<8>(M, L, O, lane);
  combine_merge<16>(M, L, O, lane);
  combine_merge<32>(M, L, O, lane);
  if (sg == 0) {
    // An empty cache (no splits, or every split empty) gives zeros.
    const float inv = (M == neg_inf()) ? 0.f : 1.f / L;
    const uint32_t w0 = E::bits(O.x * inv) | (E::bits(O.y * inv) << 16);
    const uint32_t w1 = E::bits(O.z * inv) | (E::bits(O.w * inv) << 16);
    uint16_t* dst = a.out + b * a.so_b + h * a.so_h + g * a.so_g + 32 * qtr + 4 * chunk;
    *reinterpret_cast<uint2*>(dst) = make_uint2(w0, w1);
  }
}

// ---------------------------------------------------------------------------
// Host-side validation and launch.
// ---------------------------------------------------------------------------

#if TC_DECODE_STAMPS
unsigned long long* g_stamps = nullptr;  // the stamp buffer partial launches record into (null: none)
#endif

int check_strides(const char* what, const int64_t* st, int n) {
  if (!st) return fail(TC_ERR_INVALID_ARGUMENT, "%s strides are null", what);
  for (int i = 0; i < n; ++i) {
    if (st[i] < 0) return fail(TC_ERR_INVALID_ARGUMENT, "%s stride %d is negative (%lld)", what, i, (long long)st[i]);
    if (st[i] % 8 != 0)
      return fail(TC_ERR_ALIGNMENT, "%s stride %d (%lld elements) is not a multiple of 8", what, i, (long long)st[i]);
  }
  return TC_OK;
}

int check_common(int batch, int kv_heads, int group, int head_dim, int dtype) {
  if (batch < 1 || batch > 65535) return fail(TC_ERR_INVALID_ARGUMENT, "batch %d outside [1, 65535]", batch);
  if (kv_heads < 1 || kv_heads > 65535) return fail(TC_ERR_INVALID_ARGUMENT, "kv_heads %d outside [1, 65535]", kv_heads);
  if (group < 1 || group > 8) return fail(TC_ERR_UNSUPPORTED, "group (query heads per KV head) %d outside [1, 8]", group);
  if (head_dim != kHeadDim) return fail(TC_ERR_UNSUPPORTED, "head_dim %d unsupported (kernels are built for 128)", head_dim);
  if (dtype != TC_DTYPE_F16 && dtype != TC_DTYPE_BF16) return fail(TC_ERR_UNSUPPORTED, "dtype %d unsupported", dtype);
  return TC_OK;
}

inline dim3 partial_grid(const PartialArgs& a, int batch) { return dim3(a.heads, a.splits, batch); }

template <int DT, bool PAGED, bool APPEND, int W, bool WINDOW = false>
void launch_partial_waves(const PartialArgs& a, int batch, hipStream_t stream) {
  if (a.out)
    hipLaunchKernelGGL((decode_partial_kernel<DT, PAGED, APPEND, true, W, WINDOW>), partial_grid(a, batch),
                       dim3(64 * W), 0, stream, a);
  else
    hipLaunchKernelGGL((decode_partial_kernel<DT, PAGED, APPEND, false, W, WINDOW>), partial_grid(a, batch),
                       dim3(64 * W), 0, stream, a);
}

template <int DT, bool PAGED>
void launch_partial_paged(const PartialArgs& a, int batch, int waves, hipStream_t stream) {
  if constexpr (!PAGED) {
    if (a.window && a.k_new) return launch_partial_waves<DT, false, true, kWaves, true>(a, batch, stream);
    if (a.window) return launch_partial_waves<DT, false, false, kWaves, true>(a, batch, stream);
  }
  if (a.k_new) return launch_partial_waves<DT, PAGED, true, kWaves>(a, batch, stream);
  if constexpr (!PAGED)
    if (waves == kShortWaves) return launch_partial_waves<DT, false, false, kShortWaves>(a, batch, stream);
  launch_partial_waves<DT, PAGED, false, kWaves>(a, batch, stream);
}

template <int DT>
hipError_t launch_partial_dt(const PartialArgs& a, int batch, int waves, hipStream_t stream) {
  if (a.tile_tab)
    launch_partial_paged<DT, true>(a, batch, waves, stream);
  else
    launch_partial_paged<DT, false>(a, batch, waves, stream);
  return hipGetLastError();
}

// Waves per partial work-group: two for a short cache with one length for the
// batch, read by the plain call with its tiles dealt round-robin; else four.
// A whole call (few_tiles) also asks for at most 8 tiles a split: with more,
// in a batch, four waves are faster (16 sequences of 1000 tokens, 32 tiles a
// split: 16.8 against 17.7 us; 4 of 1000, 8 tiles: the same).
inline int partial_waves(int64_t n_tokens, bool lens, bool paged, bool append, int interleave, bool few_tiles) {
  return (few_tiles && interleave && !lens && !paged && !append && n_tokens <= TC_DECODE_SHORT_TOKENS) ? kShortWaves : kWaves;
}

// Split plan of a call: S splits of T tokens each (S * T >= n, T a multiple of
// the granule). With split_tokens > 0 the caller fixes T. Otherwise S is
// chosen so that B * Hkv * S work-groups are TC_DECODE_WGS_PER_CU per compute
// unit (every work-group then streams the same share of the cache when its
// tiles are dealt round-robin), but never more splits than a head has
// wave-tiles and never more than TC_MAX_SPLITS. Ragged batches (per-sequence
// lengths) aim at 8, 4 or 2 work-groups per unit where a wave of the longest
// sequence then still has 4.5 tiles, else at 1: short sequences leave their
// work-groups light, and many small work-groups let the dispatcher balance the
// rest, but a work-group costs its first round trip, its merge and its partial
// whatever it reads. At 8 always, four sequences of 2500-5000 tokens took 21.8
// us (1.2 tiles a wave) against 13.8 at 2; 16 of 2000-4000 35.2 against 30.5 at
// 4; 8 of 750-1500 17.6 against 11.3 at 1; 2 of 1500-3000 11.6 against 8.6 at
// 1; 16 of 1k-32k tokens stay at 8 (150 us against 160 at 4, 156 at 16).
// The plan does not depend on the work-group shape: a short
// cache read by two-wave work-groups keeps the four-wave plan's splits (its
// waves then take two tiles each where four-wave ones took one).
int split_plan(int batch, int kv_heads, int64_t max_tokens, int split_tokens, int ragged, int* S_out, int* T_out) {
  if (batch < 1 || kv_heads < 1 || max_tokens < 0)
    return fail(TC_ERR_INVALID_ARGUMENT, "split query with batch %d, kv_heads %d, max_tokens %lld", batch, kv_heads,
                (long long)max_tokens);
  // Shortest split that keeps the split count within TC_MAX_SPLITS.
  const int64_t floor_t = ceil_div(ceil_div(max_tokens, TC_MAX_SPLITS), kSplitGranule) * kSplitGranule;
  int64_t t, S;
  if (split_tokens > 0) {
    t = max(ceil_div(split_tokens, kSplitGranule) * kSplitGranule, floor_t);
    S = ceil_div(max_tokens, t);
  } else {
    int cus = 0;
    const int rc = current_device_cus(&cus);
    if (rc != TC_OK) return rc;
    const int64_t per_head = static_cast<int64_t>(batch) * kv_heads;
    int64_t per_cu = TC_DECODE_WGS_PER_CU;
    if (ragged) {
      const int64_t tiles = ceil_div(max_tokens, kWaveIter), splits1 = std::max<int64_t>(1, cus / per_head);
      per_cu = TC_DECODE_RAGGED_WGS_PER_CU;
      while (per_cu > 1 && 2 * tiles < 9 * kWaves * splits1 * per_cu) per_cu /= 2;
    }
    const int64_t target = per_cu * cus;
    const int64_t max_s = std::max<int64_t>(1, std::min<int64_t>(ceil_div(ceil_div(max_tokens, kWaveIter), kWaves),
                                                        TC_MAX_SPLITS));
    S = std::max<int64_t>(1, std::min<int64_t>((target + per_head / 2) / per_head, max_s));
    t = max(ceil_div(ceil_div(max_tokens, S), kSplitGranule) * kSplitGranule, floor_t);
    if (max_tokens == 0) S = 0;
  }
  t = max(t, static_cast<int64_t>(kSplitGranule));
  if (t > (1 << 30)) return fail(TC_ERR_INVALID_ARGUMENT, "split length %lld too large", (long long)t);
  *S_out = static_cast<int>(S);
  *T_out = static_cast<int>(t);
  return TC_OK;
}

}  // namespace
}  // namespace tc

using namespace tc;

extern "C" {

int tc_decode_split_tokens(int batch, int kv_heads, int64_t max_tokens, int split_tokens, int ragged) {
  clear_error();
  int S = 0, t = 0;
  const int rc = split_plan(batch, kv_heads, max_tokens, split_tokens, ragged, &S, &t);
  return rc == TC_OK ? t : -rc;
}

int tc_decode_num_splits(int batch, int kv_heads, int64_t max_tokens, int split_tokens, int ragged) {
  clear_error();
  int S = 0, t = 0;
  const int rc = split_plan(batch, kv_heads, max_tokens, split_tokens, ragged, &S, &t);
  return rc == TC_OK ? S : -rc;
}

size_t tc_decode_workspace_bytes(int batch, int kv_heads, int group, int head_dim, int num_splits) {
  if (batch < 1 || kv_heads < 1 || group < 1 || head_dim < 1 || num_splits < 0) return 0;
  const size_t parts = static_cast<size_t>(batch) * kv_heads * num_splits * group;
  return parts * head_dim * sizeof(float) + parts * sizeof(float);
}

}  // extern "C"

namespace tc {
namespace {

// The new token of an append-and-attend call: K/V rows [B, H, D] and the
// writable cache they go to.
struct Append {
  const void* k_new;
  const int64_t* kn_strides;  // (batch, head)
  const void* v_new;
  const int64_t* vn_strides;
  void* k_cache;
  void* v_cache;
};

// A paged cache: the tile table of every sequence and the pool's shape.
struct Paged {
  const int32_t* tile_tab;  // [B, max_tiles, 4]
  const int32_t* tiles;     // [B]
  int64_t max_tiles;
  int pages, page_tokens;
  const int32_t* tok_off = nullptr;  // device-length append: [B, tok_pitch] row byte offsets
  int64_t tok_pitch = 0;
};

// The visible tokens of a windowed call: the last `window` and the first `sinks`.
struct Window {
  int64_t window, sinks;
};

// Index space that the tiles of the longest sequence of n_tokens span (PartialArgs::window).
int64_t window_span(const Window& w, int64_t n_tokens) {
  if (n_tokens - w.window <= w.sinks) return n_tokens;
  return ceil_div(w.sinks, kWaveIter) * kWaveIter + w.window;
}

// *whole: the window hides nothing, so that the call is the plain one.
int check_window(int64_t window, int64_t sinks, int64_t n_tokens, Window* w, bool* whole) {
  if (n_tokens < 0 || window < 1 || sinks < 0)
    return fail(TC_ERR_INVALID_ARGUMENT, "window %lld, %lld sink tokens of %lld", (long long)window, (long long)sinks,
                (long long)n_tokens);
  *w = Window{std::min(window, n_tokens), std::min(sinks, n_tokens)};
  *whole = n_tokens - w->window <= w->sinks;
  return TC_OK;
}

int partial_impl(const void* q_dev, const int64_t q_strides[3], const void* k_dev, const int64_t k_strides[3],
                 const void* v_dev, const int64_t v_strides[3], const int32_t* lens_dev, int64_t n_tokens, int batch,
                 int kv_heads, int group, int head_dim, int dtype, float scale, int split_tokens, int num_splits,
                 float* o_part_dev, float* lse_part_dev, int interleave, const Append* app, void* stream,
                 const Paged* paged = nullptr, bool whole_call = false, void* out_dev = nullptr,
                 const int64_t* out_strides = nullptr, const Window* window = nullptr,
                 PartialArgs* only = nullptr) {
  int rc = check_common(batch, kv_heads, group, head_dim, dtype);
  if (rc != TC_OK) return rc;
  if (n_tokens == 0 && num_splits == 0) return TC_OK;  // empty caches: nothing to read
  if (!q_dev || !k_dev || !v_dev || !o_part_dev || !lse_part_dev)
    return fail(TC_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned16(q_dev) || !aligned16(k_dev) || !aligned16(v_dev) || !aligned16(o_part_dev))
    return fail(TC_ERR_ALIGNMENT, "q/k/v/o_part base pointers must be 16-byte aligned");
  if ((rc = check_strides("q", q_strides, 3)) != TC_OK) return rc;
  if ((rc = check_strides("k", k_strides, 3)) != TC_OK) return rc;
  if ((rc = check_strides("v", v_strides, 3)) != TC_OK) return rc;
  if (n_tokens < 0) return fail(TC_ERR_INVALID_ARGUMENT, "n_tokens %lld is negative", (long long)n_tokens);
  if (n_tokens > kMaxTokens)
    return fail(TC_ERR_INVALID_ARGUMENT, "n_tokens %lld above %lld", (long long)n_tokens, (long long)kMaxTokens);
  if (split_tokens <= 0 || split_tokens % kSplitGranule != 0)
    return fail(TC_ERR_INVALID_ARGUMENT, "split_tokens %d must be a positive multiple of %d", split_tokens,
                kSplitGranule);
  if (num_splits < 0 || num_splits > TC_MAX_SPLITS)
    return fail(TC_ERR_INVALID_ARGUMENT, "num_splits %d outside [0, %d]", num_splits, TC_MAX_SPLITS);
  if (static_cast<int64_t>(num_splits) * split_tokens < (window ? window_span(*window, n_tokens) : n_tokens))
    return fail(TC_ERR_INVALID_ARGUMENT, "%d splits of %d tokens do not cover %lld tokens", num_splits, split_tokens,
                (long long)n_tokens);
  if (static_cast<int64_t>(num_splits) * split_tokens > 2 * kMaxTokens)
    return fail(TC_ERR_INVALID_ARGUMENT, "%d splits of %d tokens span more than %lld tokens", num_splits,
                split_tokens, (long long)(2 * kMaxTokens));
  if (num_splits == 0) return TC_OK;
  if (!isfinite(scale)) return fail(TC_ERR_INVALID_ARGUMENT, "scale is not finite");
  // Per-lane buffer offsets span 16 token rows in 32 bits.
  constexpr int64_t kMaxTokenStride = int64_t(1) << 26;
  if (k_strides[2] < head_dim || v_strides[2] < head_dim || k_strides[2] >= kMaxTokenStride ||
      v_strides[2] >= kMaxTokenStride)
    return fail(TC_ERR_INVALID_ARGUMENT, "k/v token strides (%lld, %lld) outside [%d, 2^26)",
                (long long)k_strides[2], (long long)v_strides[2], head_dim);

  PartialArgs a;
  a.q = static_cast<const uint16_t*>(q_dev);
  a.k = static_cast<const uint16_t*>(k_dev);
  a.v = static_cast<const uint16_t*>(v_dev);
  a.o_part = o_part_dev;
  a.lse_part = lse_part_dev;
  a.lens = lens_dev;
  a.n = n_tokens;
  a.sq_b = q_strides[0]; a.sq_h = q_strides[1]; a.sq_g = q_strides[2];
  a.sk_b = k_strides[0]; a.sk_h = k_strides[1]; a.sk_t = k_strides[2];
  a.sv_b = v_strides[0]; a.sv_h = v_strides[1]; a.sv_t = v_strides[2];
  a.heads = kv_heads;
  a.group = group;
  a.splits = num_splits;
  a.split_tokens = split_tokens;
  a.part_splits = num_splits;
  a.interleave = interleave;
  // Longest sequences first: only for per-sequence lengths of a contiguous
  // cache, and up to 64 sequences (one lane each).
  a.longest_first = (lens_dev && !paged && batch > 1 && batch <= 64) ? 1 : 0;
  a.k_new = app ? static_cast<const uint16_t*>(app->k_new) : nullptr;
  a.v_new = app ? static_cast<const uint16_t*>(app->v_new) : nullptr;
  a.skn_b = app ? app->kn_strides[0] : 0;
  a.skn_h = app ? app->kn_strides[1] : 0;
  a.svn_b = app ? app->vn_strides[0] : 0;
  a.svn_h = app ? app->vn_strides[1] : 0;
  a.k_w = app ? static_cast<uint16_t*>(app->k_cache) : nullptr;
  a.v_w = app ? static_cast<uint16_t*>(app->v_cache) : nullptr;
  a.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  a.tile_tab = paged ? paged->tile_tab : nullptr;
  a.tiles = paged ? paged->tiles : nullptr;
  a.max_tiles = paged ? paged->max_tiles : 0;
  a.pages = paged ? paged->pages : 0;
  a.page_tokens = paged ? paged->page_tokens : 0;
  a.tok_off = paged ? paged->tok_off : nullptr;
  a.tok_pitch = paged ? paged->tok_pitch : 0;
  a.window = window ? static_cast<int32_t>(window->window) : 0;
  a.sinks = window ? static_cast<int32_t>(window->sinks) : 0;
  a.out = static_cast<uint16_t*>(out_dev);
  a.so_b = out_dev ? out_strides[0] : 0;
  a.so_h = out_dev ? out_strides[1] : 0;
  a.so_g = out_dev ? out_strides[2] : 0;
#if TC_DECODE_STAMPS
  a.stamps = g_stamps;
#endif

  if (only) {  // the caller launches
    *only = a;
    return TC_OK;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int waves = partial_waves(n_tokens, lens_dev != nullptr, paged != nullptr, app != nullptr, interleave,
                                  !whole_call || n_tokens <= int64_t(8) * kWaveIter * num_splits);
  const hipError_t e = dtype == TC_DTYPE_F16 ? launch_partial_dt<TC_DTYPE_F16>(a, batch, waves, s)
                                             : launch_partial_dt<TC_DTYPE_BF16>(a, batch, waves, s);
  return hip_status(e, "decode_partial launch");
}

}  // namespace
}  // namespace tc

extern "C" {

int tc_decode_partial(const void* q_dev, const int64_t q_strides[3], const void* k_dev, const int64_t k_strides[3],
                      const void* v_dev, const int64_t v_strides[3], const int32_t* lens_dev, int64_t n_tokens,
                      int batch, int kv_heads, int group, int head_dim, int dtype, float scale, int split_tokens,
                      int num_splits, float* o_part_dev, float* lse_part_dev, void* stream) {
  clear_error();
  return partial_impl(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, lens_dev, n_tokens, batch, kv_heads, group,
                      head_dim, dtype, scale, split_tokens, num_splits, o_part_dev, lse_part_dev, 0, nullptr,
                      stream);
}

int tc_decode_partial_interleaved(const void* q_dev, const int64_t q_strides[3], const void* k_dev,
                                  const int64_t k_strides[3], const void* v_dev, const int64_t v_strides[3],
                                  const int32_t* lens_dev, int64_t n_tokens, int batch, int kv_heads, int group,
                                  int head_dim, int dtype, float scale, int split_tokens, int num_splits,
                                  float* o_part_dev, float* lse_part_dev, void* stream) {
  clear_error();
  return partial_impl(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, lens_dev, n_tokens, batch, kv_heads, group,
                      head_dim, dtype, scale, split_tokens, num_splits, o_part_dev, lse_part_dev, 1, nullptr,
                      stream);
}

int tc_decode_combine(const float* o_part_dev, const float* lse_part_dev, int batch, int kv_heads, int group,
                      int head_dim, int num_splits, void* out_dev, const int64_t out_strides[3], int dtype,
                      void* stream) {
  clear_error();
  int rc = check_common(batch, kv_heads, group, head_dim, dtype);
  if (rc != TC_OK) return rc;
  if (!out_dev || (num_splits > 0 && (!o_part_dev || !lse_part_dev)))
    return fail(TC_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned16(out_dev) || (num_splits > 0 && !aligned16(o_part_dev)))
    return fail(TC_ERR_ALIGNMENT, "out/o_part base pointers must be 16-byte aligned");
  if ((rc = check_strides("out", out_strides, 3)) != TC_OK) return rc;
  if (num_splits < 0 || num_splits > TC_MAX_SPLITS)
    return fail(TC_ERR_INVALID_ARGUMENT, "num_splits %d outside [0, %d]", num_splits, TC_MAX_SPLITS);

  CombineArgs a;
  a.o_part = o_part_dev;
  a.lse_part = lse_part_dev;
  a.out = static_cast<uint16_t*>(out_dev);
  a.so_b = out_strides[0]; a.so_h = out_strides[1]; a.so_g = out_strides[2];
  a.heads = kv_heads;
  a.group = group;
  a.splits = num_splits;
  hipStream_t s = static_cast<hipStream_t>(stream);
  // One wave per (KV head, sequence, query head, quarter of the dims), the KV
  // head fastest.
  const dim3 grid(kv_heads, batch, group * 4), block(64);
  if (dtype == TC_DTYPE_F16)
    hipLaunchKernelGGL((decode_combine_kernel<TC_DTYPE_F16>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((decode_combine_kernel<TC_DTYPE_BF16>), grid, block, 0, s, a);
  return hip_status(hipGetLastError(), "decode_combine launch");
}

}  // extern "C"

namespace tc {
namespace {

int attention_impl(const void* q_dev, const int64_t q_strides[3], const void* k_dev, const int64_t k_strides[3],
                   const void* v_dev, const int64_t v_strides[3], const int32_t* lens_dev, int64_t n_tokens,
                   int batch, int kv_heads, int group, int head_dim, int dtype, float scale, int split_tokens,
                   void* workspace_dev, size_t workspace_bytes, void* out_dev, const int64_t out_strides[3],
                   const Append* app, int ragged_plan, void* stream, const Paged* paged = nullptr,
                   const Window* window = nullptr) {
  int rc = check_common(batch, kv_heads, group, head_dim, dtype);
  if (rc != TC_OK) return rc;
  if (n_tokens < 0) return fail(TC_ERR_INVALID_ARGUMENT, "n_tokens %lld is negative", (long long)n_tokens);
  int S = 0, t = 0;
  const int64_t span = window ? window_span(*window, n_tokens) : n_tokens;
  if ((rc = split_plan(batch, kv_heads, span, split_tokens, ragged_plan, &S, &t)) != TC_OK) return rc;
  const size_t need = tc_decode_workspace_bytes(batch, kv_heads, group, head_dim, S);
  if (S > 0 && (!workspace_dev || workspace_bytes < need))
    return fail(TC_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed for %d splits", workspace_bytes, need, S);
  float* o_part = static_cast<float*>(workspace_dev);
  float* lse_part = S > 0 ? o_part + static_cast<size_t>(batch) * kv_heads * S * group * head_dim : nullptr;
  // One split (many sequences, or at most 64 tokens) needs no combine: the
  // partial kernel writes the result, bit for bit what the combine would make
  // of it. 32 sequences of 300 tokens 13.9 -> 10.4 us.
  const bool direct = S == 1;
  if (direct) {
    if (!out_dev) return fail(TC_ERR_INVALID_ARGUMENT, "null tensor pointer");
    if (!aligned16(out_dev)) return fail(TC_ERR_ALIGNMENT, "out base pointer must be 16-byte aligned");
    if ((rc = check_strides("out", out_strides, 3)) != TC_OK) return rc;
  }
  if (S > 0) {
    // Splits here are internal, so their tiles are dealt round-robin (the merged result is the same).
    rc = partial_impl(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, lens_dev, n_tokens, batch, kv_heads, group,
                      head_dim, dtype, scale, t, S, o_part, lse_part, TC_DECODE_INTERLEAVE, app, stream, paged,
                      true, direct ? out_dev : nullptr, out_strides, window);
    if (rc != TC_OK || direct) return rc;
  }
  return tc_decode_combine(o_part, lse_part, batch, kv_heads, group, head_dim, S, out_dev, out_strides, dtype, stream);
}

}  // namespace
}  // namespace tc

extern "C" {

int tc_decode_attention(const void* q_dev, const int64_t q_strides[3], const void* k_dev, const int64_t k_strides[3],
                        const void* v_dev, const int64_t v_strides[3], const int32_t* lens_dev, int64_t n_tokens,
                        int batch, int kv_heads, int group, int head_dim, int dtype, float scale, int split_tokens,
                        void* workspace_dev, size_t workspace_bytes, void* out_dev, const int64_t out_strides[3],
                        void* stream) {
  clear_error();
  return attention_impl(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, lens_dev, n_tokens, batch, kv_heads,
                        group, head_dim, dtype, scale, split_tokens, workspace_dev, workspace_bytes, out_dev,
                        out_strides, nullptr, lens_dev != nullptr, stream);
}

}  // extern "C"

extern "C" {

int64_t tc_decode_window_tokens(int64_t n_tokens, int64_t window, int64_t sink_tokens) {
  clear_error();
  Window w;
  bool whole;
  const int rc = check_window(window, sink_tokens, n_tokens, &w, &whole);
  return rc == TC_OK ? window_span(w, n_tokens) : -rc;
}

int tc_decode_window_attention(const void* q_dev, const int64_t q_strides[3], const void* k_dev,
                               const int64_t k_strides[3], const void* v_dev, const int64_t v_strides[3],
                               const int32_t* lens_dev, int64_t n_tokens, int64_t window, int64_t sink_tokens,
                               int batch, int kv_heads, int group, int head_dim, int dtype, float scale,
                               int split_tokens, void* workspace_dev, size_t workspace_bytes, void* out_dev,
                               const int64_t out_strides[3], void* stream) {
  clear_error();
  Window w;
  bool whole;
  const int rc = check_window(window, sink_tokens, n_tokens, &w, &whole);
  if (rc != TC_OK) return rc;
  return attention_impl(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, lens_dev, n_tokens, batch, kv_heads,
                        group, head_dim, dtype, scale, split_tokens, workspace_dev, workspace_bytes, out_dev,
                        out_strides, nullptr, lens_dev != nullptr, stream, nullptr, whole ? nullptr : &w);
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Allocation-free decode: the split partials of tc_decode_attention_noalloc
// live in `scratch`, a static array that every GPU the library runs on holds
// until the process ends. Its device address differs per GPU and is taken
// once per device with hipGetSymbolAddress; host code never passes the
// array's own name to a kernel.
// ---------------------------------------------------------------------------

static __device__ __align__(256) unsigned char scratch[TC_DECODE_SCRATCH_BYTES];

namespace tc {
namespace {

constexpr int kScratchDevices = 64;
std::mutex g_scratch_mutex;
void* g_scratch_dev[kScratchDevices] = {};

// Device address of `scratch` on the current device (looked up on first use).
int scratch_on_current_device(void** out) {
  int dev = 0;
  int rc = hip_status(hipGetDevice(&dev), "hipGetDevice");
  if (rc != TC_OK) return rc;
  if (dev < 0 || dev >= kScratchDevices) return fail(TC_ERR_HIP, "device id %d out of range", dev);
  std::lock_guard<std::mutex> lock(g_scratch_mutex);
  if (!g_scratch_dev[dev]) {
    void* p = nullptr;
    rc = hip_status(hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)), "hipGetSymbolAddress(scratch)");
    if (rc != TC_OK) return rc;
    if (!p || !aligned16(p)) return fail(TC_ERR_HIP, "scratch symbol address %p unusable", p);
    g_scratch_dev[dev] = p;
  }
  *out = g_scratch_dev[dev];
  return TC_OK;
}

}  // namespace
}  // namespace tc

extern "C" {

int tc_decode_attention_noalloc(const void* q_dev, const int64_t q_strides[3], const void* k_dev,
                                const int64_t k_strides[3], const void* v_dev, const int64_t v_strides[3],
                                const int32_t* lens_dev, int64_t n_tokens, int batch, int kv_heads, int group,
                                int head_dim, int dtype, float scale, int split_tokens, void* out_dev,
                                const int64_t out_strides[3], void* stream) {
  clear_error();
  int rc = check_common(batch, kv_heads, group, head_dim, dtype);
  if (rc != TC_OK) return rc;
  if (n_tokens < 0) return fail(TC_ERR_INVALID_ARGUMENT, "n_tokens %lld is negative", (long long)n_tokens);
  int S = 0, t = 0;
  if ((rc = split_plan(batch, kv_heads, n_tokens, split_tokens, lens_dev != nullptr, &S, &t)) != TC_OK) return rc;
  const size_t need = tc_decode_workspace_bytes(batch, kv_heads, group, head_dim, S);
  if (need > TC_DECODE_SCRATCH_BYTES)
    return fail(TC_ERR_WORKSPACE,
                "%d splits of batch %d x %d kv heads x %d query heads need %zu bytes of partials; the static scratch "
                "holds %zu (pass a workspace to tc_decode_attention instead)",
                S, batch, kv_heads, group, need, (size_t)TC_DECODE_SCRATCH_BYTES);
  void* ws = nullptr;
  if (S > 0 && (rc = scratch_on_current_device(&ws)) != TC_OK) return rc;
  return attention_impl(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, lens_dev, n_tokens, batch, kv_heads,
                        group, head_dim, dtype, scale, split_tokens, ws, TC_DECODE_SCRATCH_BYTES, out_dev,
                        out_strides, nullptr, lens_dev != nullptr, stream);
}

static int append_impl(const void* q_dev, const int64_t q_strides[3], void* k_cache_dev, const int64_t k_strides[3],
                       void* v_cache_dev, const int64_t v_strides[3], const void* k_new_dev,
                       const int64_t k_new_strides[2], const void* v_new_dev, const int64_t v_new_strides[2],
                       const int32_t* pos_dev, int64_t n_tokens, int batch, int kv_heads, int group, int head_dim,
                       int dtype, float scale, int split_tokens, void* workspace_dev, size_t workspace_bytes,
                       void* out_dev, const int64_t out_strides[3], void* stream, const Window* window = nullptr) {
  if (n_tokens < 1) return fail(TC_ERR_INVALID_ARGUMENT, "append needs n_tokens >= 1 (got %lld)", (long long)n_tokens);
  if (!k_new_dev || !v_new_dev || !k_new_strides || !v_new_strides)
    return fail(TC_ERR_INVALID_ARGUMENT, "null new-token K/V");
  if (!aligned16(k_new_dev) || !aligned16(v_new_dev))
    return fail(TC_ERR_ALIGNMENT, "new-token K/V not 16-byte aligned");
  for (int i = 0; i < 2; ++i)
    if (k_new_strides[i] < 0 || v_new_strides[i] < 0 || k_new_strides[i] % 8 || v_new_strides[i] % 8)
      return fail(TC_ERR_ALIGNMENT, "new-token K/V strides must be non-negative multiples of 8");
  const Append app{k_new_dev, k_new_strides, v_new_dev, v_new_strides, k_cache_dev, v_cache_dev};
  return attention_impl(q_dev, q_strides, k_cache_dev, k_strides, v_cache_dev, v_strides, pos_dev, n_tokens, batch,
                        kv_heads, group, head_dim, dtype, scale, split_tokens, workspace_dev, workspace_bytes, out_dev,
                        out_strides, &app, 0, stream, nullptr, window);
}

int tc_decode_append_attention(const void* q_dev, const int64_t q_strides[3], void* k_cache_dev,
                               const int64_t k_strides[3], void* v_cache_dev, const int64_t v_strides[3],
                               const void* k_new_dev, const int64_t k_new_strides[2], const void* v_new_dev,
                               const int64_t v_new_strides[2], int64_t n_tokens, int batch, int kv_heads, int group,
                               int head_dim, int dtype, float scale, int split_tokens, void* workspace_dev,
                               size_t workspace_bytes, void* out_dev, const int64_t out_strides[3], void* stream) {
  clear_error();
  return append_impl(q_dev, q_strides, k_cache_dev, k_strides, v_cache_dev, v_strides, k_new_dev, k_new_strides,
                     v_new_dev, v_new_strides, nullptr, n_tokens, batch, kv_heads, group, head_dim, dtype, scale,
                     split_tokens, workspace_dev, workspace_bytes, out_dev, out_strides, stream);
}

int tc_decode_append_attention_at(const void* q_dev, const int64_t q_strides[3], void* k_cache_dev,
                                  const int64_t k_strides[3], void* v_cache_dev, const int64_t v_strides[3],
                                  const void* k_new_dev, const int64_t k_new_strides[2], const void* v_new_dev,
                                  const int64_t v_new_strides[2], const int32_t* pos_dev, int64_t capacity,
                                  int batch, int kv_heads, int group, int head_dim, int dtype, float scale,
                                  int split_tokens, void* workspace_dev, size_t workspace_bytes, void* out_dev,
                                  const int64_t out_strides[3], void* stream) {
  clear_error();
  if (!pos_dev) return fail(TC_ERR_INVALID_ARGUMENT, "null append positions");
  return append_impl(q_dev, q_strides, k_cache_dev, k_strides, v_cache_dev, v_strides, k_new_dev, k_new_strides,
                     v_new_dev, v_new_strides, pos_dev, capacity, batch, kv_heads, group, head_dim, dtype, scale,
                     split_tokens, workspace_dev, workspace_bytes, out_dev, out_strides, stream);
}

int tc_decode_append_window_attention(const void* q_dev, const int64_t q_strides[3], void* k_cache_dev,
                                      const int64_t k_strides[3], void* v_cache_dev, const int64_t v_strides[3],
                                      const void* k_new_dev, const int64_t k_new_strides[2], const void* v_new_dev,
                                      const int64_t v_new_strides[2], const int32_t* pos_dev, int64_t n_tokens,
                                      int64_t window, int64_t sink_tokens, int batch, int kv_heads, int group,
                                      int head_dim, int dtype, float scale, int split_tokens, void* workspace_dev,
                                      size_t workspace_bytes, void* out_dev, const int64_t out_strides[3],
                                      void* stream) {
  clear_error();
  Window w;
  bool whole;
  const int rc = check_window(window, sink_tokens, n_tokens, &w, &whole);
  if (rc != TC_OK) return rc;
  return append_impl(q_dev, q_strides, k_cache_dev, k_strides, v_cache_dev, v_strides, k_new_dev, k_new_strides,
                     v_new_dev, v_new_strides, pos_dev, n_tokens, batch, kv_heads, group, head_dim, dtype, scale,
                     split_tokens, workspace_dev, workspace_bytes, out_dev, out_strides, stream, whole ? nullptr : &w);
}

int tc_decode_paged_attention(const void* q_dev, const int64_t q_strides[3], const void* k_pool_dev,
                              const void* v_pool_dev, const int64_t pool_strides[3], int num_pages, int page_tokens,
                              const int32_t* tile_table_dev, const int32_t* tiles_dev, int64_t max_tiles, int batch,
                              int kv_heads, int group, int head_dim, int dtype, float scale, int split_tokens,
                              void* workspace_dev, size_t workspace_bytes, void* out_dev,
                              const int64_t out_strides[3], void* stream) {
  clear_error();
  if (num_pages < 1 || page_tokens < 1)
    return fail(TC_ERR_INVALID_ARGUMENT, "pool of %d pages of %d tokens", num_pages, page_tokens);
  if (max_tiles < 0 || max_tiles > kMaxTokens / 16)
    return fail(TC_ERR_INVALID_ARGUMENT, "max_tiles %lld outside [0, %lld]", (long long)max_tiles,
                (long long)(kMaxTokens / 16));
  if (max_tiles > 0 && (!tile_table_dev || !tiles_dev)) return fail(TC_ERR_INVALID_ARGUMENT, "null tile table");
  if (max_tiles > 0 && !aligned16(tile_table_dev))
    return fail(TC_ERR_ALIGNMENT, "tile table not 16-byte aligned");
  if (!pool_strides) return fail(TC_ERR_INVALID_ARGUMENT, "null pool strides");
  // An empty table plans zero splits, so the partial kernel (the only reader
  // of the table) is not launched.
  const Paged p{tile_table_dev, tiles_dev, max_tiles, num_pages, page_tokens};
  return attention_impl(q_dev, q_strides, k_pool_dev, pool_strides, v_pool_dev, pool_strides, nullptr,
                        16 * max_tiles, batch, kv_heads, group, head_dim, dtype, scale, split_tokens, workspace_dev,
                        workspace_bytes, out_dev, out_strides, nullptr, batch > 1, stream, &p);
}

int tc_decode_paged_append_attention(const void* q_dev, const int64_t q_strides[3], void* k_pool_dev,
                                     void* v_pool_dev, const int64_t pool_strides[3], int num_pages,
                                     int page_tokens, const int32_t* tile_table_dev, const int32_t* tiles_dev,
                                     int64_t max_tiles, const void* k_new_dev, const int64_t k_new_strides[2],
                                     const void* v_new_dev, const int64_t v_new_strides[2], int batch,
                                     int kv_heads, int group, int head_dim, int dtype, float scale,
                                     int split_tokens, void* workspace_dev, size_t workspace_bytes, void* out_dev,
                                     const int64_t out_strides[3], void* stream) {
  clear_error();
  if (num_pages < 1 || page_tokens < 1)
    return fail(TC_ERR_INVALID_ARGUMENT, "pool of %d pages of %d tokens", num_pages, page_tokens);
  if (max_tiles < 1 || max_tiles > kMaxTokens / 16)
    return fail(TC_ERR_INVALID_ARGUMENT, "append needs max_tiles in [1, %lld] (got %lld)",
                (long long)(kMaxTokens / 16), (long long)max_tiles);
  if (!tile_table_dev || !tiles_dev) return fail(TC_ERR_INVALID_ARGUMENT, "null tile table");
  if (!aligned16(tile_table_dev)) return fail(TC_ERR_ALIGNMENT, "tile table not 16-byte aligned");
  if (!pool_strides) return fail(TC_ERR_INVALID_ARGUMENT, "null pool strides");
  if (!k_new_dev || !v_new_dev || !k_new_strides || !v_new_strides)
    return fail(TC_ERR_INVALID_ARGUMENT, "null new-token K/V");
  if (!aligned16(k_new_dev) || !aligned16(v_new_dev))
    return fail(TC_ERR_ALIGNMENT, "new-token K/V not 16-byte aligned");
  for (int i = 0; i < 2; ++i)
    if (k_new_strides[i] < 0 || v_new_strides[i] < 0 || k_new_strides[i] % 8 || v_new_strides[i] % 8)
      return fail(TC_ERR_ALIGNMENT, "new-token K/V strides must be non-negative multiples of 8");
  const Append app{k_new_dev, k_new_strides, v_new_dev, v_new_strides, k_pool_dev, v_pool_dev};
  const Paged p{tile_table_dev, tiles_dev, max_tiles, num_pages, page_tokens};
  return attention_impl(q_dev, q_strides, k_pool_dev, pool_strides, v_pool_dev, pool_strides, nullptr,
                        16 * max_tiles, batch, kv_heads, group, head_dim, dtype, scale, split_tokens, workspace_dev,
                        workspace_bytes, out_dev, out_strides, &app, batch > 1, stream, &p);
}

int tc_decode_paged_append_attention_at(const void* q_dev, const int64_t q_strides[3], void* k_pool_dev,
                                        void* v_pool_dev, const int64_t pool_strides[3], int num_pages,
                                        int page_tokens, const int32_t* tile_table_dev, const int32_t* tiles_dev,
                                        int64_t max_tiles, const int32_t* tok_off_dev, int64_t tok_pitch,
                                        const int32_t* lens_dev, const void* k_new_dev,
                                        const int64_t k_new_strides[2], const void* v_new_dev,
                                        const int64_t v_new_strides[2], int batch, int kv_heads, int group,
                                        int head_dim, int dtype, float scale, int split_tokens, void* workspace_dev,
                                        size_t workspace_bytes, void* out_dev, const int64_t out_strides[3],
                                        void* stream) {
  clear_error();
  if (num_pages < 1 || page_tokens < 1)
    return fail(TC_ERR_INVALID_ARGUMENT, "pool of %d pages of %d tokens", num_pages, page_tokens);
  if (max_tiles < 1 || max_tiles > kMaxTokens / 16)
    return fail(TC_ERR_INVALID_ARGUMENT, "append needs max_tiles in [1, %lld] (got %lld)",
                (long long)(kMaxTokens / 16), (long long)max_tiles);
  if (!tile_table_dev || !tiles_dev || !tok_off_dev || !lens_dev)
    return fail(TC_ERR_INVALID_ARGUMENT, "null tile table, token offsets or lengths");
  if (!aligned16(tile_table_dev)) return fail(TC_ERR_ALIGNMENT, "tile table not 16-byte aligned");
  if (tok_pitch < 1 || tok_pitch > kMaxTokens)
    return fail(TC_ERR_INVALID_ARGUMENT, "token offset rows of %lld entries", (long long)tok_pitch);
  if (!pool_strides) return fail(TC_ERR_INVALID_ARGUMENT, "null pool strides");
  if (static_cast<int64_t>(num_pages) * pool_strides[0] * 2 >= (int64_t(1) << 31))
    return fail(TC_ERR_UNSUPPORTED, "pools of 2 GiB or more (token offsets are 32-bit)");
  if (!k_new_dev || !v_new_dev || !k_new_strides || !v_new_strides)
    return fail(TC_ERR_INVALID_ARGUMENT, "null new-token K/V");
  if (!aligned16(k_new_dev) || !aligned16(v_new_dev))
    return fail(TC_ERR_ALIGNMENT, "new-token K/V not 16-byte aligned");
  for (int i = 0; i < 2; ++i)
    if (k_new_strides[i] < 0 || v_new_strides[i] < 0 || k_new_strides[i] % 8 || v_new_strides[i] % 8)
      return fail(TC_ERR_ALIGNMENT, "new-token K/V strides must be non-negative multiples of 8");
  const Append app{k_new_dev, k_new_strides, v_new_dev, v_new_strides, k_pool_dev, v_pool_dev};
  const Paged p{tile_table_dev, tiles_dev, max_tiles, num_pages, page_tokens, tok_off_dev, tok_pitch};
  return attention_impl(q_dev, q_strides, k_pool_dev, pool_strides, v_pool_dev, pool_strides, lens_dev,
                        16 * max_tiles, batch, kv_heads, group, head_dim, dtype, scale, split_tokens, workspace_dev,
                        workspace_bytes, out_dev, out_strides, &app, batch > 1, stream, &p);
}

}  // extern "C"

namespace tc {
namespace {

// The prefix of a shared-prefix call: contiguous [H, tokens, D] of K and V with (head, token) strides, or tiles of the
// page pools that hold every sequence's own tokens too.
struct Prefix {
  const void* k;
  const int64_t* k_strides;
  const void* v;
  const int64_t* v_strides;
  int64_t tokens;
  const int32_t* tiles = nullptr;
};

// Many rows with few splits are joined by the kernel that gives a row to half a wave: the combine kernel's four waves a
// row, which read 32 splits at once, then cost their dispatch. Whole calls (us; the combine kernel's first): 4096 rows of
// 9 splits 84.5, 80.4; 4096 of 3 59.0, 52.9; 1024 of 9 34.8, 34.1; 768 of 14 the same; 512 of 15 13.2, 13.8; 1024 of 20
// 32.0, 32.6; 1280 of 25 29.5, 30.0; 128 of 29 18.3, 19.9.
constexpr int kJoinRows = 1024, kJoinSplits = 16;

// Splits of a shared-prefix call: the prefix's come first.
int shared_plan(int batch, int kv_heads, int group, int64_t prefix_tokens, int64_t max_tokens, int ragged, int* S_prefix,
                int* S_own, int* T_own) {
  int cus = 0, rc;
  if (batch < 1 || kv_heads < 1 || group < 1 || prefix_tokens < 0 || prefix_tokens > kMaxTokens || max_tokens < 0 ||
      max_tokens > kMaxTokens)
    return fail(TC_ERR_INVALID_ARGUMENT, "prefix of %lld and own %lld tokens, batch %d, kv_heads %d, group %d",
                (long long)prefix_tokens, (long long)max_tokens, batch, kv_heads, group);
  if (prefix_tokens == 0) {
    *S_prefix = 0;
    return split_plan(batch, kv_heads, max_tokens, 0, ragged, S_own, T_own);
  }
  if ((rc = current_device_cus(&cus)) != TC_OK) return rc;
  shared_splits(batch, kv_heads, group, ceil_div(prefix_tokens, kWaveIter), max_tokens, ragged != 0, cus, S_prefix, S_own);
  *T_own = static_cast<int>(std::max<int64_t>(1, ceil_div(ceil_div(max_tokens, std::max(*S_own, 1)), kSplitGranule)) * kSplitGranule);
  return TC_OK;
}

int shared_impl(const void* q_dev, const int64_t q_strides[3], const Prefix& x, const void* k_dev,
                const int64_t k_strides[3], const void* v_dev, const int64_t v_strides[3], const int32_t* lens_dev,
                int64_t n_tokens, int batch, int kv_heads, int group, int head_dim, int dtype, float scale,
                void* workspace_dev, size_t workspace_bytes, void* out_dev, const int64_t out_strides[3],
                const Append* app, int ragged, void* stream, const Paged* paged) {
  int rc = check_common(batch, kv_heads, group, head_dim, dtype);
  if (rc != TC_OK) return rc;
  if (n_tokens < 0) return fail(TC_ERR_INVALID_ARGUMENT, "n_tokens %lld is negative", (long long)n_tokens);
  if (x.tokens == 0)
    return attention_impl(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, lens_dev, n_tokens, batch, kv_heads,
                          group, head_dim, dtype, scale, 0, workspace_dev, workspace_bytes, out_dev, out_strides, app,
                          ragged, stream, paged);
  int Sp = 0, S = 0, t = 0;
  if ((rc = shared_plan(batch, kv_heads, group, x.tokens, n_tokens, ragged, &Sp, &S, &t)) != TC_OK) return rc;
  if (!q_dev || !x.k || !x.v || !out_dev) return fail(TC_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned16(q_dev) || !aligned16(x.k) || !aligned16(x.v) || !aligned16(out_dev) || !aligned16(workspace_dev))
    return fail(TC_ERR_ALIGNMENT, "q/k/v/out/workspace base pointers must be 16-byte aligned");
  if ((rc = check_strides("q", q_strides, 3)) != TC_OK) return rc;
  if ((rc = check_strides("out", out_strides, 3)) != TC_OK) return rc;
  if ((rc = check_strides("prefix k", x.k_strides, x.tiles ? 3 : 2)) != TC_OK) return rc;
  if ((rc = check_strides("prefix v", x.v_strides, x.tiles ? 3 : 2)) != TC_OK) return rc;
  const int64_t sk_t = x.k_strides[x.tiles ? 2 : 1], sv_t = x.v_strides[x.tiles ? 2 : 1];
  constexpr int64_t kMaxTokenStride = int64_t(1) << 26;  // a tile's 16 rows in 32-bit offsets
  if (sk_t < head_dim || sv_t < head_dim || sk_t >= kMaxTokenStride || sv_t >= kMaxTokenStride)
    return fail(TC_ERR_INVALID_ARGUMENT, "prefix token strides (%lld, %lld) outside [%d, 2^26)", (long long)sk_t,
                (long long)sv_t, head_dim);
  if (!isfinite(scale)) return fail(TC_ERR_INVALID_ARGUMENT, "scale is not finite");
  const size_t need = tc_decode_workspace_bytes(batch, kv_heads, group, head_dim, Sp + S);
  if (!workspace_dev || workspace_bytes < need)
    return fail(TC_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed for %d splits", workspace_bytes, need, Sp + S);
  float* o_part = static_cast<float*>(workspace_dev);
  float* lse_part = o_part + static_cast<size_t>(batch) * kv_heads * (Sp + S) * group * head_dim;
  PartialArgs own{};
  if (S > 0 && (rc = partial_impl(q_dev, q_strides, k_dev, k_strides, v_dev, v_strides, lens_dev, n_tokens, batch,
                                  kv_heads, group, head_dim, dtype, scale, t, S, o_part, lse_part, 1, app, stream,
                                  paged, true, nullptr, nullptr, nullptr, &own)) != TC_OK) return rc;
  if (S > 0) {  // their splits come after the prefix's
    own.o_part += static_cast<int64_t>(Sp) * group * head_dim;
    own.lse_part += static_cast<int64_t>(Sp) * group;
    own.part_splits = Sp + S;
  }
#if TC_DECODE_STAMPS
  own.stamps = nullptr;  // the timeline's buffer is laid out for the decode partial kernel's grid
#endif
  PrefixArgs a;
  a.q = static_cast<const uint16_t*>(q_dev);
  a.k = static_cast<const uint16_t*>(x.k);
  a.v = static_cast<const uint16_t*>(x.v);
  a.o_part = o_part;
  a.lse_part = lse_part;
  a.sq_b = q_strides[0]; a.sq_h = q_strides[1]; a.sq_g = q_strides[2];
  a.sk_p = x.tiles ? x.k_strides[0] : 0;
  a.sv_p = x.tiles ? x.v_strides[0] : 0;
  a.sk_h = x.k_strides[x.tiles ? 1 : 0];
  a.sv_h = x.v_strides[x.tiles ? 1 : 0];
  a.sk_t = sk_t;
  a.sv_t = sv_t;
  a.tile_tab = x.tiles;
  a.tiles = static_cast<int32_t>(ceil_div(x.tokens, kWaveIter));
  a.n = static_cast<int32_t>(x.tokens);
  a.pages = paged ? paged->pages : 0;
  a.page_tokens = paged ? paged->page_tokens : 0;
  a.heads = kv_heads;
  a.group = group;
  a.batch = batch;
  a.splits = Sp;
  a.part_splits = Sp + S;
  // (A scale of 0 as one so small that every weight is 1: a hidden key's -inf times it stays -inf.)
  a.c = std::max(static_cast<float>(fabs(static_cast<double>(scale)) * 1.4426950408889634), 1e-30f);
  a.sign = scale < 0.f ? 0x80008000u : 0u;
  const int64_t shares = int64_t(Sp) * ceil_div(int64_t(batch) * group, 256) + int64_t(S) * batch;
  if (shares * kv_heads > 0x7fffffff) return fail(TC_ERR_UNSUPPORTED, "grid too large");
  if ((rc = hip_status(launch_shared(a, own, dtype, static_cast<hipStream_t>(stream)), "shared-prefix launch")) != TC_OK) return rc;
  if (int64_t(batch) * kv_heads * group >= kJoinRows && Sp + S <= kJoinSplits) {
    const JoinArgs j{o_part, lse_part, static_cast<uint16_t*>(out_dev), out_strides[0], out_strides[1], out_strides[2],
                     kv_heads, group, batch, Sp + S};
    return hip_status(launch_join(j, dtype, static_cast<hipStream_t>(stream)), "shared-prefix join launch");
  }
  return tc_decode_combine(o_part, lse_part, batch, kv_heads, group, head_dim, Sp + S, out_dev, out_strides, dtype,
                           stream);
}

}  // namespace
}  // namespace tc

extern "C" {

int tc_decode_shared_num_splits(int batch, int kv_heads, int group, int64_t prefix_tokens, int64_t max_tokens,
                                int ragged) {
  clear_error();
  int Sp = 0, S = 0, t = 0;
  const int rc = shared_plan(batch, kv_heads, group, prefix_tokens, max_tokens, ragged, &Sp, &S, &t);
  return rc == TC_OK ? Sp + S : -rc;
}

int tc_decode_shared_attention(const void* q_dev, const int64_t q_strides[3], const void* k_prefix_dev,
                               const int64_t k_prefix_strides[2], const void* v_prefix_dev,
                               const int64_t v_prefix_strides[2], int64_t prefix_tokens, const void* k_dev,
                               const int64_t k_strides[3], const void* v_dev, const int64_t v_strides[3],
                               const int32_t* lens_dev, int64_t n_tokens, int batch, int kv_heads, int group,
                               int head_dim, int dtype, float scale, void* workspace_dev, size_t workspace_bytes,
                               void* out_dev, const int64_t out_strides[3], void* stream) {
  clear_error();
  const Prefix x{k_prefix_dev, k_prefix_strides, v_prefix_dev, v_prefix_strides, prefix_tokens};
  return shared_impl(q_dev, q_strides, x, k_dev, k_strides, v_dev, v_strides, lens_dev, n_tokens, batch, kv_heads,
                     group, head_dim, dtype, scale, workspace_dev, workspace_bytes, out_dev, out_strides, nullptr,
                     lens_dev != nullptr, stream, nullptr);
}

int tc_decode_paged_shared_attention(const void* q_dev, const int64_t q_strides[3], void* k_pool_dev, void* v_pool_dev,
                                     const int64_t pool_strides[3], int num_pages, int page_tokens,
                                     const int32_t* shared_table_dev, int64_t shared_tiles,
                                     const int32_t* tile_table_dev, const int32_t* tiles_dev, int64_t max_tiles,
                                     const void* k_new_dev, const int64_t k_new_strides[2], const void* v_new_dev,
                                     const int64_t v_new_strides[2], int batch, int kv_heads, int group, int head_dim,
                                     int dtype, float scale, void* workspace_dev, size_t workspace_bytes,
                                     void* out_dev, const int64_t out_strides[3], void* stream) {
  clear_error();
  if (num_pages < 1 || page_tokens < 1)
    return fail(TC_ERR_INVALID_ARGUMENT, "pool of %d pages of %d tokens", num_pages, page_tokens);
  if (max_tiles < 0 || max_tiles > kMaxTokens / 16 || shared_tiles < 0 || shared_tiles > kMaxTokens / 16)
    return fail(TC_ERR_INVALID_ARGUMENT, "tables of %lld and %lld tiles", (long long)shared_tiles, (long long)max_tiles);
  if ((max_tiles > 0 && (!tile_table_dev || !tiles_dev)) || (shared_tiles > 0 && !shared_table_dev))
    return fail(TC_ERR_INVALID_ARGUMENT, "null tile table");
  if (!aligned16(tile_table_dev) || !aligned16(shared_table_dev))
    return fail(TC_ERR_ALIGNMENT, "tile table not 16-byte aligned");
  if (!pool_strides) return fail(TC_ERR_INVALID_ARGUMENT, "null pool strides");
  const Append app{k_new_dev, k_new_strides, v_new_dev, v_new_strides, k_pool_dev, v_pool_dev};
  if (k_new_dev || v_new_dev) {
    if (max_tiles < 1) return fail(TC_ERR_INVALID_ARGUMENT, "append without tiles of the sequences' own");
    if (!k_new_dev || !v_new_dev || !k_new_strides || !v_new_strides)
      return fail(TC_ERR_INVALID_ARGUMENT, "null new-token K/V");
    if (!aligned16(k_new_dev) || !aligned16(v_new_dev))
      return fail(TC_ERR_ALIGNMENT, "new-token K/V not 16-byte aligned");
    for (int i = 0; i < 2; ++i)
      if (k_new_strides[i] < 0 || v_new_strides[i] < 0 || k_new_strides[i] % 8 || v_new_strides[i] % 8)
        return fail(TC_ERR_ALIGNMENT, "new-token K/V strides must be non-negative multiples of 8");
  }
  const Paged p{tile_table_dev, tiles_dev, max_tiles, num_pages, page_tokens};
  const Prefix x{k_pool_dev, pool_strides, v_pool_dev, pool_strides, 16 * shared_tiles,
                 shared_tiles ? shared_table_dev : nullptr};
  return shared_impl(q_dev, q_strides, x, k_pool_dev, pool_strides, v_pool_dev, pool_strides, nullptr, 16 * max_tiles,
                     batch, kv_heads, group, head_dim, dtype, scale, workspace_dev, workspace_bytes, out_dev,
                     out_strides, k_new_dev ? &app : nullptr, batch > 1, stream, &p);
}

}  // extern "C"

#if TC_DECODE_STAMPS
// Measurement build only (libthreadcut_stamps.so): the device buffer that the
// partial kernels launched from now on record their wave timelines into
// (8 words per wave, see PartialArgs::stamps), or null for none.
extern "C" void tc_decode_set_stamps(void* stamps_dev) { tc::g_stamps = static_cast<unsigned long long*>(stamps_dev); }
#endif
