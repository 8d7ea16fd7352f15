// Decode attention of a batch over a prefix that all of its sequences share:
// the prefix's keys and values are read once for the whole batch.
//
//   out_b = softmax([q_b Kp^T, q_b K_b^T] scale) [Vp; V_b]
//
// is the merge, by log-sum-exp, of the attention over the prefix and over each
// sequence's own tokens. The second is the work of the decode partial kernel;
// for the first, of one KV head, the B*G query rows of all sequences are the
// columns of the products that the decode kernel makes for the G rows of one
// sequence, so a K/V tile serves all of them. One launch does both: some
// work-groups take shares of the prefix, the others sequences' own tokens.
//
// Per wave and step of 32 tokens (two 16-token tiles t = 0, 1), with column
// n = lane % 16 of block r and lane group g = lane / 16:
//   S^T[token][column] = K . Q: per tile and block four v_mfma_f32_16x16x32,
//     Q in registers for the whole kernel; lane (g, n) gets tokens 4g .. 4g + 3
//     of each tile.
//   softmax per column in fp32, log2 domain, as in the decode kernel.
//   O^T[dim][column] += V^T . P^T: eight v_mfma_f32_16x16x32 a block whose 32
//     k indices are, for lane group g, the tokens 4g .. 4g + 3 of both tiles:
//     P^T leaves the S^T registers without moving between lanes, V^T comes from
//     the wave's LDS region by the transposing read, once for all blocks.
//
// Bound: HBM for few columns (16 over 10000 tokens of 8 heads, 200 to 500
// own tokens each: 15.5 us with the combine, 47 MB); for many the vector instructions of the softmax
// beside the products (512 columns over 16384 tokens of 8 heads: 81 us, of which
// reading once would take 52; its products alone 25).
#include <algorithm>

#include "decode_tile.hpp"
#include "shared.hpp"

namespace tc {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kRowBytes = 2 * kHeadDim;  // a K or V row in LDS
constexpr int kStep = 32;                // keys of a wave's step: two 16-key tiles
constexpr int kMergeRow = kHeadDim + 16; // floats of a column's row in the merge (padded: the stores spread over the banks)

// Work-groups of W waves: CG column groups of 16 R columns, W / CG key groups.
// Columns of all groups see every key of a work-group's tile; with one column
// group the waves split its keys and need no barrier.
template <int W_, int CG_, int R_>
struct Shape {
  static constexpr int W = W_, CG = CG_, R = R_, KG = W_ / CG_;
  static constexpr int kColumns = 16 * R * CG;
  static constexpr int kTiles = 8;                         // 16-key tiles of a work-group's tile
  static constexpr int kSteps = kTiles / (2 * KG);         // steps of a wave in it
  static constexpr int kBuf = 16 * kTiles * kRowBytes;     // bytes of its K (and V)
  static constexpr bool kResidue = CG == 1;                // weights as two numbers of the type
};

// Slot of 16-byte chunk x of row r of a 16-key tile. Half of a V read covers 8
// rows of two neighbouring chunks, a quarter of a K read rows 0-3 and 12-15 of
// one chunk and rows 4-11 of its neighbour (which the hardware takes together:
// with 2 (r % 8) + r / 8 every K read met two rows a bank); both fall on
// distinct banks.
__device__ __forceinline__ int slot_of(int x, int r) { return x ^ (2 * ((r & 7) ^ (r >> 3 << 2)) + (r >> 3)); }

// Split `split` of the prefix for head h and the columns of block `block`.
template <int DT, bool PAGED, class S>
__device__ __forceinline__ void prefix_partial(const PrefixArgs& a, const int h, const int split, const int block,
                                               char* const s_k0, char* const s_k1, char* const s_v0, char* const s_v1,
                                               float (*s_m)[16], float (*s_l)[16]) {
  using M = DecodeMma<DT>;
  using E = Elem<DT>;
  constexpr int R = S::R, CG = S::CG, KG = S::KG;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int cg = wave % CG, kg = wave / CG;
  const int c0 = block * S::kColumns + 16 * R * cg;
  const int columns = a.batch * a.group;
  const char* kslab = reinterpret_cast<const char*>(a.k + h * a.sk_h);
  const char* vslab = reinterpret_cast<const char*>(a.v + h * a.sv_h);
  const int32_t row_k = static_cast<int32_t>(a.sk_t) * 2, row_v = static_cast<int32_t>(a.sv_t) * 2;

  // The work-group's tiles: groups of kTiles 16-key tiles, every splits-th of them. A wave loads the K and V of a
  // share of the group (with one column group that of its own keys) and multiplies the two tiles of each of its steps.
  constexpr int kParts = 4 * S::kTiles / S::W;  // pieces of 4 rows of K, and of V, that a wave loads
  const int32_t groups = (a.tiles + S::kTiles - 1) / S::kTiles;

  // Paged: lane i holds the table entry of tile i % kTiles of the (i / kTiles)-th group from `held` on.
  int32_t e_page = 0, e_slot = 0, e_rows = 0, held = 0;
  constexpr int kHeld = 64 / S::kTiles;
  auto hold = [&](int32_t it) {
    held = it;
    const int32_t group = split + (it + lane / S::kTiles) * a.splits;
    const int64_t tile = static_cast<int64_t>(group) * S::kTiles + lane % S::kTiles;
    e_page = e_slot = e_rows = 0;
    if (tile < a.tiles) {
      const int4 e = *reinterpret_cast<const int4*>(a.tile_tab + 4 * tile);
      // An entry outside the pool or past the page's end counts as empty.
      if (!(e.x < 0 || e.x >= a.pages || e.y < 0 || e.z < 0 || e.z > 16 || e.y > a.page_tokens - e.z)) {
        e_page = e.x; e_slot = e.y; e_rows = e.z;
      }
    }
  };
  // Rows of tile t of the work-group's it-th group.
  auto rows_of = [&](int32_t it, int t) -> int32_t {
    if constexpr (PAGED) return __builtin_amdgcn_readlane(e_rows, (it - held) * S::kTiles + t);
    // (i32 min and max select a vector instruction: without readfirstlane the buffer ranges would not be scalar.)
    return __builtin_amdgcn_readfirstlane(min(max(a.n - 16 * ((split + it * a.splits) * S::kTiles + t), 0), 16));
  };
  // This wave's loads of group it, straight into LDS: 4 rows an instruction, lane l filling slot l % 16 of row l / 16.
  auto load = [&](char* dk, char* dv, int32_t it) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int part = wave * kParts + i, t = part >> 2;
      const int32_t rows = rows_of(it, t);
      const char *kp = kslab, *vp = vslab;
      if constexpr (PAGED) {
        const int at = (it - held) * S::kTiles + t;
        const int64_t page = __builtin_amdgcn_readlane(e_page, at), slot = __builtin_amdgcn_readlane(e_slot, at);
        kp += page * a.sk_p * 2 + slot * row_k;
        vp += page * a.sv_p * 2 + slot * row_v;
      } else {
        const int64_t tile = rows > 0 ? (split + it * a.splits) * S::kTiles + t : 0;
        kp += 16 * tile * row_k;
        vp += 16 * tile * row_v;
      }
      const __amdgpu_buffer_rsrc_t rk = make_rsrc(kp, rows * row_k), rv = make_rsrc(vp, rows * row_v);
      const int r = 4 * (part & 3) + g;
      const int x = 16 * slot_of(n, r);  // (the swizzle is its own inverse)
      __attribute__((address_space(3))) void* pk = (__attribute__((address_space(3))) void*)(dk + 4 * part * kRowBytes);
      __attribute__((address_space(3))) void* pv = (__attribute__((address_space(3))) void*)(dv + 4 * part * kRowBytes);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, pk, 16, r * row_k + x, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, pv, 16, r * row_v + x, 0, 0, 0);
    }
  };
  const int32_t its = split < groups ? (groups - split + a.splits - 1) / a.splits : 0;
  if constexpr (PAGED) hold(0);
  if (its > 0) load(s_k0, s_v0, 0);

  uint4 qb[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = c0 + 16 * r + n;
    const uint32_t b = static_cast<uint32_t>(c) / a.group, i = c - b * a.group;
    const uint16_t* q = a.q + b * a.sq_b + h * a.sq_h + i * a.sq_g + 8 * g;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      qb[r][j] = c < columns ? *reinterpret_cast<const uint4*>(q + 32 * j) : make_uint4(0, 0, 0, 0);
      qb[r][j].x ^= a.sign; qb[r][j].y ^= a.sign; qb[r][j].z ^= a.sign; qb[r][j].w ^= a.sign;
    }
  }

  // acc: O^T; l: the sum of the weights, in every register (a product with ones); m: the running maximum, in units of
  // a.c times a score, -inf at first, and ms what is subtracted (0 then).
  f32x4 acc[R][8], l[R];
  float m[R], ms[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = neg_inf();
    ms[r] = 0.f;
    l[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int bm = 0; bm < 8; ++bm) acc[r][bm] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Byte offsets, in a 16-row tile, of the lane's K reads (row n, chunk 4 i + g) and its transposing V reads (row
  // 4 g + n / 4, 8 bytes at dim 16 bm + 4 (n % 4)).
  int koff[4], voff[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) koff[i] = n * kRowBytes + 16 * slot_of(4 * i + g, n);
  {
    const int r = 4 * g + (n >> 2);
#pragma unroll
    for (int bm = 0; bm < 8; ++bm) voff[bm] = r * kRowBytes + 16 * slot_of(2 * bm + ((n & 3) >> 1), r) + 8 * (n & 1);
  }

  // One step: 32 keys from (lk, lv); rows0 and rows1 of them in the two tiles. Vector instructions are
  // what many columns are bound by (the exponentials alone take as long as half of the products), so the rest of the
  // softmax is kept short: the maximum is compared with the running one lane by lane, and reduced over the lanes only
  // where some lane's exceeds it; the weights are summed by the matrix core.
  uint4 kf[2][4];
  auto read_k = [&](const char* lk) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) kf[t][i] = *reinterpret_cast<const uint4*>(lk + 16 * kRowBytes * t + koff[i]);
  };
  // kf holds the step's K; `more`: the next step's is read from lk_next under the products with V.
  auto step = [&](const char* lk_next, const char* lv, bool more, int32_t rows0, int32_t rows1) {
    // Rows past a tile's end score -inf from the start (their keys read as zeros).
    f32x4 none[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      none[0][j] = 4 * g + j < rows0 ? 0.f : neg_inf();
      none[1][j] = 4 * g + j < rows1 ? 0.f : neg_inf();
    }
    f32x4 sc[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[r][t] = M::qk(kf[t][0], qb[r][0], none[t]);
#pragma unroll
        for (int i = 1; i < 4; ++i) sc[r][t] = M::qk(kf[t][i], qb[r][i], sc[r][t]);
      }
    }
    // V^T[16 bm + n][4g .. 4g + 3 of both tiles], once for all column blocks; read under the softmax.
    uint4 vf[8];
#pragma unroll
    for (int bm = 0; bm < 8; ++bm) {
      uint2 t2[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
        t2[t] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) lds_s4*)(lv + 16 * kRowBytes * t + voff[bm])));
      vf[bm] = make_uint4(t2[0].x, t2[0].y, t2[1].x, t2[1].y);
    }
    __builtin_amdgcn_sched_barrier(0);
    float mx[R];
    bool any = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const f32x4 &x = sc[r][0], &y = sc[r][1];
      mx[r] = a.c * fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
      any |= mx[r] > m[r] + kLazyMax;
    }
    // The running maximum moves only when the step's exceeds it by 2^8, for a column's lanes together.
    if (__any(any)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float tmax = rows_max(mx[r]);
        const bool move = tmax > m[r] + kLazyMax;
        const float alpha = move ? __builtin_amdgcn_exp2f(m[r] - tmax) : 1.f;  // 0 while nothing was seen
        m[r] = move ? tmax : m[r];
        ms[r] = m[r] == neg_inf() ? 0.f : m[r];
#pragma unroll
        for (int bm = 0; bm < 8; ++bm) acc[r][bm] *= alpha;
        l[r] *= alpha;
      }
    }
    uint4 ph[R], pl[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(sc[r][j >> 2][j & 3], a.c, -ms[r]));
      uint32_t w[4], e[4] = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = M::pack(p[2 * j], p[2 * j + 1]);
      if constexpr (S::kResidue) {
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = M::pack(p[2 * j] - E::lo(w[j]), p[2 * j + 1] - E::hi(w[j]));
      }
      ph[r] = make_uint4(w[0], w[1], w[2], w[3]);
      pl[r] = make_uint4(e[0], e[1], e[2], e[3]);
    }
    if (more) read_k(lk_next);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      constexpr uint32_t kOnes = DT == TC_DTYPE_F16 ? 0x3C003C00u : 0x3F803F80u;
      const uint4 ones = make_uint4(kOnes, kOnes, kOnes, kOnes);
      l[r] = M::qk(ones, ph[r], l[r]);
#pragma unroll
      for (int bm = 0; bm < 8; ++bm) acc[r][bm] = M::qk(vf[bm], ph[r], acc[r][bm]);
      if constexpr (S::kResidue) {
        // What rounding to the type left of the weights goes through the product too, as in the decode kernel (with
        // many columns, which are bound by the products, it does not, as in prefill).
        l[r] = M::qk(ones, pl[r], l[r]);
#pragma unroll
        for (int bm = 0; bm < 8; ++bm) acc[r][bm] = M::qk(vf[bm], pl[r], acc[r][bm]);
      }
    }
  };

  // A group from (lk, lv) while the next one loads into (dk, dv).
  auto body = [&](int32_t it, const char* lk, const char* lv, char* dk, char* dv) {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of group it have landed
    if constexpr (CG > 1) __syncthreads();               // and everyone's; (dk, dv) is read no more
    int32_t rows[2 * S::kSteps];
#pragma unroll
    for (int i = 0; i < 2 * S::kSteps; ++i) rows[i] = rows_of(it, 2 * S::kSteps * kg + i);
    if (it + 1 < its) {
      if constexpr (PAGED)
        if (it + 1 - held >= kHeld) hold(it + 1);
      load(dk, dv, it + 1);
    }
    const int at = S::kSteps * kg * kStep * kRowBytes;
    read_k(lk + at);
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i)
      step(lk + at + (i + 1) * kStep * kRowBytes, lv + at + i * kStep * kRowBytes, i + 1 < S::kSteps, rows[2 * i],
           rows[2 * i + 1]);
  };
  for (int32_t it = 0; it < its; it += 2) {
    body(it, s_k0, s_v0, s_k1, s_v1);
    if (it + 1 < its) body(it + 1, s_k1, s_v1, s_k0, s_v0);
  }

  // The key groups' results of a column are merged block by block through LDS and written by the first group. Lane
  // (g, n) holds dims 16 bm + 4 g .. + 3 of column n.
  constexpr int kHold = S::kBuf / (16 * kMergeRow * 4);  // waves' rows that a tile buffer holds
  static_assert((KG - 1) * CG <= 4 * kHold, "the other groups' rows fit the tile buffers");
  auto rows16 = [&](int w) {  // of wave w >= CG
    const int i = w - CG, buf = i / kHold;
    return reinterpret_cast<float*>(buf == 0 ? s_k0 : buf == 1 ? s_k1 : buf == 2 ? s_v0 : s_v1) + i % kHold * 16 * kMergeRow;
  };
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float L = l[r][0], mx = m[r];
    if constexpr (KG > 1) {
      __syncthreads();  // the tiles, or the block before, are done with
      if (kg > 0) {
#pragma unroll
        for (int bm = 0; bm < 8; ++bm)
          *reinterpret_cast<float4*>(rows16(wave) + n * kMergeRow + 16 * bm + 4 * g) =
              make_float4(acc[r][bm][0], acc[r][bm][1], acc[r][bm][2], acc[r][bm][3]);
      }
      if (g == 0) { s_m[wave][n] = mx; s_l[wave][n] = L; }
      __syncthreads();
      if (kg > 0) continue;
#pragma unroll
      for (int k = 1; k < KG; ++k) mx = fmaxf(mx, s_m[k * CG + cg][n]);
      const float ms = mx == neg_inf() ? 0.f : mx;
      const float mine = __builtin_amdgcn_exp2f(m[r] - ms);
      L *= mine;
#pragma unroll
      for (int bm = 0; bm < 8; ++bm) acc[r][bm] *= mine;
#pragma unroll
      for (int k = 1; k < KG; ++k) {
        const float f = __builtin_amdgcn_exp2f(s_m[k * CG + cg][n] - ms);
        L += s_l[k * CG + cg][n] * f;
#pragma unroll
        for (int bm = 0; bm < 8; ++bm) {
          const float4 o = *reinterpret_cast<const float4*>(rows16(k * CG + cg) + n * kMergeRow + 16 * bm + 4 * g);
          acc[r][bm][0] += o.x * f;
          acc[r][bm][1] += o.y * f;
          acc[r][bm][2] += o.z * f;
          acc[r][bm][3] += o.w * f;
        }
      }
    }
    const int c = c0 + 16 * r + n;
    if (c >= columns) continue;
    const float inv = L == 0.f ? 0.f : __builtin_amdgcn_rcpf(L);
    const uint32_t b = static_cast<uint32_t>(c) / a.group, i = c - b * a.group;
    const int64_t part = ((static_cast<int64_t>(b) * a.heads + h) * a.part_splits + split) * a.group + i;
    float* const o = a.o_part + part * kHeadDim + 4 * g;
#pragma unroll
    for (int bm = 0; bm < 8; ++bm)
      *reinterpret_cast<float4*>(o + 16 * bm) =
          make_float4(acc[r][bm][0] * inv, acc[r][bm][1] * inv, acc[r][bm][2] * inv, acc[r][bm][3] * inv);
    if (g == 0) a.lse_part[part] = L == 0.f ? neg_inf() : (mx + __builtin_amdgcn_logf(L)) * kLn2;
  }
}

// The grid: the KV head fastest (with 8 heads a head's work-groups share an
// XCD's L2); then the prefix's splits and column blocks, then the sequences'
// own tokens, which 4 waves take as in the decode partial kernel (so a
// work-group of 8 takes two shares).
template <int DT, bool PAGED, bool APPEND, class S>
__global__ __launch_bounds__(64 * S::W) __attribute__((amdgpu_waves_per_eu(S::W / 4))) void shared_partial_kernel(
    const PrefixArgs a, const PartialArgs o) {
  __shared__ __attribute__((aligned(1024))) char s_k0[S::kBuf], s_k1[S::kBuf], s_v0[S::kBuf], s_v1[S::kBuf];
  __shared__ float s_m[S::W][16], s_l[S::W][16];
  const uint32_t heads = a.heads, y = blockIdx.x / heads, h = blockIdx.x - y * heads;
  const uint32_t shares = a.splits * static_cast<uint32_t>(a.blocks);
  if (y < shares) {
    const uint32_t block = y / a.splits;
    prefix_partial<DT, PAGED, S>(a, h, y - block * a.splits, block, s_k0, s_k1, s_v0, s_v1, s_m, s_l);
    return;
  }
  constexpr int kOwn = 4, kUnits = S::W / kOwn;
  const int unit = kUnits > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * kOwn)) : 0;
  const uint32_t j = (y - shares) * kUnits + unit, z = j / o.splits;
  static_assert(kOwn * kVTileWords * 4 <= S::kBuf && kOwn * 8 * (kHeadDim + 16) * 4 <= S::kBuf, "a share's LDS");
  char* const vt = unit ? s_v0 : s_k0;
  char* const acc = unit ? s_v1 : s_k1;
  static_assert(2 * 8 * kOwn <= S::W / kUnits * 16, "a share's maxima and sums");
  float* const ml = unit ? s_l[0] : s_m[0];
  if (z < static_cast<uint32_t>(a.batch))
    decode_partial<DT, PAGED, APPEND, false, kOwn, false, true>(
        o, h, j - z * o.splits, z, a.batch, threadIdx.x - unit * 64 * kOwn, reinterpret_cast<uint32_t(*)[kVTileWords]>(vt),
        reinterpret_cast<float(*)[8][kHeadDim + 16]>(acc), reinterpret_cast<float(*)[kOwn]>(ml),
        reinterpret_cast<float(*)[kOwn]>(ml + 8 * kOwn));
  else
    __syncthreads();  // the one that the other half of the work-group meets in its merge
}

// A row (one query head of one sequence) takes 32 lanes, 4 dims each; a work-group 8 rows of one KV head. Its splits are
// read 8 at a time, all before the first is used.
template <int DT>
__global__ __launch_bounds__(256) void join_kernel(const JoinArgs a) {
  using E = Elem<DT>;
  constexpr int kPer = 8;
  const int row = blockIdx.y * 8 + threadIdx.x / 32, d = 4 * (threadIdx.x % 32), h = blockIdx.x;
  if (row >= a.batch * a.group) return;
  const int b = row / a.group, g = row - b * a.group, S = a.splits;
  const int64_t first = (static_cast<int64_t>(b) * a.heads + h) * S * a.group + g;
  const float* const o = a.o_part + first * kHeadDim + d;
  const float* const lse = a.lse_part + first;
  float m = neg_inf(), L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < S; s0 += kPer) {
    float4 v[kPer];
    float x[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int64_t at = static_cast<int64_t>(min(s0 + j, S - 1)) * a.group;
      v[j] = *reinterpret_cast<const float4*>(o + at * kHeadDim);
      x[j] = lse[at];
    }
    float mn = m;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (s0 + j >= S) x[j] = neg_inf();
      mn = fmaxf(mn, x[j]);
    }
    const float ms = mn == neg_inf() ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f((m - ms) * kLog2e);  // 0 while nothing was seen
    m = mn;
    L *= f;
    O.x *= f; O.y *= f; O.z *= f; O.w *= f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const float w = __builtin_amdgcn_exp2f((x[j] - ms) * kLog2e);
      L += w;
      O.x += w * v[j].x; O.y += w * v[j].y; O.z += w * v[j].z; O.w += w * v[j].w;
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;  // a row that saw nothing is zero
  *reinterpret_cast<uint2*>(a.out + b * a.so_b + h * a.so_h + g * a.so_g + d) =
      make_uint2(E::bits(O.x * inv) | (E::bits(O.y * inv) << 16), E::bits(O.z * inv) | (E::bits(O.w * inv) << 16));
}

// The shape of a call: all columns in one work-group up to 256, else in blocks of them, and no more column groups than
// they fill, so that the rest of the waves share the keys. Against the next larger shape (us, 8 heads of 4 rows, 200 own
// tokens, prefixes of 2048 and 16384): 16 columns 8.0 and 18.6, 9.3 and 20.5; 32: 10.8 and 21.8, 11.1 and 19.8 (but
// with the weights rounded once); 64: 13.1 and 22.1, 11.9 and 23.8; 128: 16.9 and 31.7, 16.5 and 34.6.
struct Plan {
  int cg, r;
  int64_t blocks;
};

Plan shape_plan(int batch, int group) {
  const int64_t c = static_cast<int64_t>(batch) * group;
  if (c <= 16) return Plan{1, 1, 1};
  if (c <= 32) return Plan{1, 2, 1};
  const int cg = c <= 64 ? 2 : c <= 128 ? 4 : 8;
  return Plan{cg, 2, ceil_div(c, 256)};
}

template <int DT, bool PAGED, bool APPEND, int W, int CG, int R>
void launch_shape(const PrefixArgs& a, const PartialArgs& o, hipStream_t s) {
  constexpr int kUnits = W / 4;
  const int64_t rows = static_cast<int64_t>(a.splits) * a.blocks + ceil_div(static_cast<int64_t>(o.splits) * a.batch, kUnits);
  hipLaunchKernelGGL((shared_partial_kernel<DT, PAGED, APPEND, Shape<W, CG, R>>), dim3(static_cast<unsigned>(a.heads * rows)),
                     dim3(64 * W), 0, s, a, o);
}

template <int DT, bool PAGED, bool APPEND>
void launch(const PrefixArgs& a, const PartialArgs& o, const Plan& p, hipStream_t s) {
  switch (p.cg) {
    case 1:
      if (p.r == 1) return launch_shape<DT, PAGED, APPEND, 4, 1, 1>(a, o, s);
      return launch_shape<DT, PAGED, APPEND, 4, 1, 2>(a, o, s);
    case 2: return launch_shape<DT, PAGED, APPEND, 8, 2, 2>(a, o, s);
    case 4: return launch_shape<DT, PAGED, APPEND, 8, 4, 2>(a, o, s);
    default: return launch_shape<DT, PAGED, APPEND, 8, 8, 2>(a, o, s);
  }
}

template <int DT>
void launch_dt(const PrefixArgs& a, const PartialArgs& o, const Plan& p, hipStream_t s) {
  if (!a.tile_tab) return launch<DT, false, false>(a, o, p, s);
  if (o.k_new) return launch<DT, true, true>(a, o, p, s);
  launch<DT, true, false>(a, o, p, s);
}

}  // namespace

// One work-group fits a compute unit, so the units are dealt to the prefix and to the own tokens by what each has to
// read, and each share is cut into as many splits as it has units. Eight column groups make the prefix bound by its
// products, so a tile weighs twice there: 64 sequences x 4 rows over 16384 tokens take 85.5 us, with a weight of 1,
// 1.5 and 3 118.8, 95.7 and 94.6. Ragged own tokens, whose longest is given here, weigh 0.6: with 1 those took 105.6
// us, 32 x 4 rows over 8000 tokens 46.9 instead of 34.8. A sequence's own share costs as much as 64 tokens before its
// first, and where there are few sequences they find units of their own; every split gets the same number of tile
// groups, as the longest one counts (both: 40 x 2 rows over 3000 tokens with 60 own 15.0 us instead of 18.5, 20 x 8
// over 12000 with 20 own 29.3 instead of 32.7, 2 x 4 over 16000 17.5 instead of 19.9, 24 x 4 forked 27.1 a layer
// instead of 28.3; nothing slower). Twice the splits for ragged own tokens helped the longest sequence of some batches
// (60 x 8 rows over 500: 50.2 us instead of 58.9) and cost others more in joining (12 x 8 forked: 19.5 instead of 16.1).
void shared_splits(int batch, int heads, int group, int64_t prefix_tiles, int64_t own_tokens, bool ragged, int cus,
                   int* prefix, int* own) {
  const Plan p = shape_plan(batch, group);
  const int64_t per_split = heads * p.blocks, most = ceil_div(prefix_tiles, 8), tiles = ceil_div(own_tokens, kWaveIter);
  const double wp = 16.0 * prefix_tiles * heads * p.blocks * (p.cg == 8 ? 2.0 : 1.0);
  const int64_t pairs = static_cast<int64_t>(batch) * heads;
  const double wo = pairs * (own_tokens * (ragged ? 0.6 : 1.0) + 64);
  const int64_t cap = cus - std::min<int64_t>(pairs, cus / 8);
  const int64_t mine = std::min(static_cast<int64_t>(cus * wp / (wp + wo)), cap);
  int64_t sp = std::max<int64_t>(1, std::min<int64_t>({(mine + per_split / 2) / per_split, most, 1024}));
  int64_t each = (2 * most + sp) / (2 * sp);  // groups of a split
  if (ceil_div(most, each) * per_split > std::max(cap, sp * per_split)) ++each;
  sp = ceil_div(most, each);
  const int64_t left = std::max<int64_t>(cus - sp * per_split, cus / 8) * (p.cg == 1 ? 1 : 2);
  *prefix = static_cast<int>(sp);
  *own = static_cast<int>(tiles ? std::max<int64_t>(1, std::min<int64_t>({(left + pairs / 2) / pairs, ceil_div(tiles, 4), 1024})) : 0);
}

hipError_t launch_join(const JoinArgs& a, int dtype, hipStream_t stream) {
  const dim3 grid(a.heads, static_cast<unsigned>(ceil_div(int64_t(a.batch) * a.group, 8)));
  if (dtype == TC_DTYPE_F16)
    hipLaunchKernelGGL((join_kernel<TC_DTYPE_F16>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((join_kernel<TC_DTYPE_BF16>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_shared(const PrefixArgs& a_in, const PartialArgs& o, int dtype, hipStream_t stream) {
  PrefixArgs a = a_in;
  const Plan p = shape_plan(a.batch, a.group);
  a.blocks = static_cast<int>(p.blocks);
  if (dtype == TC_DTYPE_F16)
    launch_dt<TC_DTYPE_F16>(a, o, p, stream);
  else
    launch_dt<TC_DTYPE_BF16>(a, o, p, stream);
  return hipGetLastError();
}

}  // namespace tc
