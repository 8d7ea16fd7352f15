// Decode attention of a batch over a prefix that all of its sequences share:
// the prefix's keys and values are read once for the whole batch.
//
//   out_b = softmax([q_b Kp^T, q_b K_b^T] scale) [Vp; V_b]
//
// is the merge, by log-sum-exp, of the attention over the prefix and over each
// sequence's own tokens. The second is the decode partial kernel; this file's
// kernel is the first: for one KV head, the B*G query rows of all sequences
// are the columns of the products that the decode kernel makes for the G rows
// of one sequence, so a K/V tile in registers serves all of them.
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
#include <algorithm>

#include "decode_tile.hpp"
#include "shared.hpp"

namespace tc {
namespace {

constexpr int kWaves = 4;
constexpr int kStepTiles = 2;  // 16-token tiles of a wave's step

typedef float f32x4 __attribute__((ext_vector_type(4)));

// One product of 32 tokens (or dims): A and B hold 8 elements a lane.
template <int DT>
__device__ __forceinline__ f32x4 mma32(const uint4& a, const uint4& b, const f32x4& c) {
  return DecodeMma<DT>::qk(a, b, c);
}

struct Step {
  uint4 k[kStepTiles][4], v[kStepTiles][4];
  int32_t rows[kStepTiles];
};

// R: blocks of 16 columns a work-group holds.
template <int DT, bool PAGED, int R>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(1))) void prefix_partial_kernel(
    const PrefixArgs a) {
  using M = DecodeMma<DT>;
  using E = Elem<DT>;
  __shared__ union {
    uint32_t v[kWaves][kStepTiles][kVTileWords];
    float acc[kWaves][16][kHeadDim + 16];
  } s;
  __shared__ float s_m[16][kWaves], s_l[16][kWaves];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  // Grid (heads, splits, column blocks), the KV head fastest: with 8 heads a head's work-groups share an XCD's L2.
  const int h = blockIdx.x, split = blockIdx.y;
  const int c0 = static_cast<int>(blockIdx.z) * 16 * R;
  const int columns = a.batch * a.group;
  const char* kslab = reinterpret_cast<const char*>(a.k + h * a.sk_h);
  const char* vslab = reinterpret_cast<const char*>(a.v + h * a.sv_h);
  const int32_t row_k = static_cast<int32_t>(a.sk_t) * 2, row_v = static_cast<int32_t>(a.sv_t) * 2;
  const int32_t steps = (a.tiles + kStepTiles - 1) / kStepTiles;
  const int32_t stride = a.splits * kWaves;
  int32_t st = split * kWaves + wave;

  int32_t koff[4], voff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    koff[i] = n * row_k + 64 * i + 16 * g;
    voff[i] = (4 * g + i) * row_v + 16 * n;
  }
  auto load = [&](Step& x, int32_t step) {
#pragma unroll
    for (int t = 0; t < kStepTiles; ++t) {
      const int32_t tile = kStepTiles * step + t;
      const char *kp = kslab, *vp = vslab;
      int32_t rows = 0;
      if constexpr (PAGED) {
        if (tile < a.tiles) {
          const int32_t* e = a.tile_tab + 4 * static_cast<int64_t>(tile);
          const int32_t page = const_load(e), slot = const_load(e + 1), cnt = const_load(e + 2);
          if (!(page < 0 || page >= a.pages || slot < 0 || cnt < 0 || cnt > 16 || slot > a.page_tokens - cnt)) {
            rows = cnt;
            kp += page * a.sk_p * 2 + static_cast<int64_t>(slot) * row_k;
            vp += page * a.sv_p * 2 + static_cast<int64_t>(slot) * row_v;
          }
        }
      } else {
        rows = min(max(a.n - kWaveIter * tile, 0), kWaveIter);
        if (rows > 0) {
          kp += static_cast<int64_t>(kWaveIter * tile) * row_k;
          vp += static_cast<int64_t>(kWaveIter * tile) * row_v;
        }
      }
      rows = __builtin_amdgcn_readfirstlane(rows);
      x.rows[t] = rows;
      const __amdgpu_buffer_rsrc_t rk = make_rsrc(kp, rows * row_k), rv = make_rsrc(vp, rows * row_v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x.k[t][j] = bload16(rk, koff[j]);
        x.v[t][j] = bload16(rv, voff[j]);
      }
    }
  };
  Step x[2];
  load(x[0], st);

  uint4 qb[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = c0 + 16 * r + n;
    const uint32_t b = static_cast<uint32_t>(c) / a.group, i = c - b * a.group;
    const uint16_t* q = a.q + b * a.sq_b + h * a.sq_h + i * a.sq_g + 8 * g;
#pragma unroll
    for (int j = 0; j < 4; ++j) qb[r][j] = c < columns ? *reinterpret_cast<const uint4*>(q + 32 * j) : make_uint4(0, 0, 0, 0);
  }

  f32x4 acc[R][8];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = neg_inf();
    l[r] = 0.f;
#pragma unroll
    for (int bm = 0; bm < 8; ++bm) acc[r][bm] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  char* const vl = reinterpret_cast<char*>(s.v[wave]);
  auto step = [&](const Step& y) {
    // V into LDS, row-major: lane (g, n) stores tokens 4g + j, dims 8n .. 8n + 7 of each tile.
#pragma unroll
    for (int t = 0; t < kStepTiles; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4*>(vl + (16 * t + 4 * g + j) * kVRowBytes + 16 * n) = y.v[t][j];
    uint4 ph[R], pl[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float sc[8];
#pragma unroll
      for (int t = 0; t < kStepTiles; ++t) {
        f32x4 s0 = mma32<DT>(y.k[t][0], qb[r][0], f32x4{0.f, 0.f, 0.f, 0.f});
        f32x4 s1 = mma32<DT>(y.k[t][1], qb[r][1], f32x4{0.f, 0.f, 0.f, 0.f});
        s0 = mma32<DT>(y.k[t][2], qb[r][2], s0);
        s1 = mma32<DT>(y.k[t][3], qb[r][3], s1);
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[4 * t + j] = 4 * g + j < y.rows[t] ? (s0[j] + s1[j]) * a.scale_log2 : neg_inf();
      }
      float mx = sc[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = fmaxf(mx, sc[j]);
      const float tmax = rows_max(mx);
      // The running maximum moves only when the step's exceeds it by 2^8.
      const float mn = (tmax > m[r] + kLazyMax || m[r] == neg_inf()) ? tmax : m[r];
      const float ms = mn == neg_inf() ? 0.f : mn;
      if (__any(mn != m[r] && m[r] != neg_inf())) {
        const float alpha = __builtin_amdgcn_exp2f(m[r] - ms);
#pragma unroll
        for (int bm = 0; bm < 8; ++bm) acc[r][bm] *= alpha;
        l[r] *= alpha;
      }
      m[r] = mn;
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(sc[j] - ms);
      l[r] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      // The weights as two numbers of the type (the second what rounding the first left), as in the decode kernel.
      uint32_t w[4], e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = M::pack(p[2 * j], p[2 * j + 1]);
        e[j] = M::pack(p[2 * j] - E::lo(w[j]), p[2 * j + 1] - E::hi(w[j]));
      }
      ph[r] = make_uint4(w[0], w[1], w[2], w[3]);
      pl[r] = make_uint4(e[0], e[1], e[2], e[3]);
    }
#pragma unroll
    for (int bm = 0; bm < 8; ++bm) {
      // V^T[16 bm + n][4g .. 4g + 3 of both tiles], by the transposing read (decode.hip).
      uint2 t2[kStepTiles];
#pragma unroll
      for (int t = 0; t < kStepTiles; ++t)
        t2[t] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) lds_s4*)(vl + (16 * t + 4 * g + (n >> 2)) * kVRowBytes + 32 * bm +
                                                        8 * (n & 3))));
      const uint4 av = make_uint4(t2[0].x, t2[0].y, t2[1].x, t2[1].y);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        acc[r][bm] = mma32<DT>(av, ph[r], acc[r][bm]);
        acc[r][bm] = mma32<DT>(av, pl[r], acc[r][bm]);
      }
    }
  };

  // Two steps in flight; no load past the wave's last.
  if (st < steps) {
    for (;;) {
      load(x[1], st + stride);
      step(x[0]);
      load(x[0], st + 2 * stride);
      if (st + stride < steps) step(x[1]);
      st += 2 * stride;
      if (st >= steps) break;
    }
  }

  // The four waves' results merged block by block through LDS.
#pragma unroll
  for (int r = 0; r < R; ++r) {
    __syncthreads();  // the V tiles, or the block before, are done with
#pragma unroll
    for (int bm = 0; bm < 8; ++bm)
      *reinterpret_cast<float4*>(&s.acc[wave][n][16 * bm + 4 * g]) =
          make_float4(acc[r][bm][0], acc[r][bm][1], acc[r][bm][2], acc[r][bm][3]);
    const float lr = rows_sum(l[r]);
    if (g == 0) { s_m[n][wave] = m[r]; s_l[n][wave] = lr; }
    __syncthreads();
    for (int idx = threadIdx.x; idx < 16 * (kHeadDim / 2); idx += 64 * kWaves) {
      const int col = idx / (kHeadDim / 2), d = 2 * (idx % (kHeadDim / 2));
      const int c = c0 + 16 * r + col;
      if (c >= columns) break;
      float mx = neg_inf();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, s_m[col][w]);
      const float ms = mx == neg_inf() ? 0.f : mx;
      float L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(s_m[col][w] - ms);
        const float2 o = *reinterpret_cast<const float2*>(&s.acc[w][col][d]);
        L += s_l[col][w] * f;
        o0 += o.x * f;
        o1 += o.y * f;
      }
      const float inv = L == 0.f ? 0.f : __builtin_amdgcn_rcpf(L);
      const uint32_t b = static_cast<uint32_t>(c) / a.group, i = c - b * a.group;
      const int64_t part = ((static_cast<int64_t>(b) * a.heads + h) * a.part_splits + split) * a.group + i;
      *reinterpret_cast<float2*>(a.o_part + part * kHeadDim + d) = make_float2(o0 * inv, o1 * inv);
      if (d == 0) a.lse_part[part] = L == 0.f ? neg_inf() : (mx + __builtin_amdgcn_logf(L)) * kLn2;
    }
  }
}

// Blocks of 16 columns a work-group holds: all, up to four.
int column_blocks(int batch, int group) {
  const int64_t c = static_cast<int64_t>(batch) * group;
  return c <= 16 ? 1 : c <= 32 ? 2 : 4;
}

template <int DT, bool PAGED>
void launch(const PrefixArgs& a, hipStream_t s) {
  const int r = column_blocks(a.batch, a.group);
  const dim3 grid(a.heads, a.splits, (a.batch * a.group + 16 * r - 1) / (16 * r)), block(64 * kWaves);
  if (r == 1)
    hipLaunchKernelGGL((prefix_partial_kernel<DT, PAGED, 1>), grid, block, 0, s, a);
  else if (r == 2)
    hipLaunchKernelGGL((prefix_partial_kernel<DT, PAGED, 2>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((prefix_partial_kernel<DT, PAGED, 4>), grid, block, 0, s, a);
}

}  // namespace

// As many work-groups as compute units, but a step for every wave.
int prefix_splits(int batch, int heads, int group, int64_t tiles, int cus) {
  const int64_t r = column_blocks(batch, group);
  const int64_t per_split = heads * ((static_cast<int64_t>(batch) * group + 16 * r - 1) / (16 * r));
  const int64_t most = ceil_div(ceil_div(tiles, kStepTiles), kWaves);
  return static_cast<int>(std::max<int64_t>(tiles > 0, std::min<int64_t>({(cus + per_split / 2) / per_split, most, 1024})));
}

hipError_t launch_prefix(const PrefixArgs& a, int dtype, hipStream_t stream) {
  if (dtype == TC_DTYPE_F16) {
    if (a.tile_tab) launch<TC_DTYPE_F16, true>(a, stream); else launch<TC_DTYPE_F16, false>(a, stream);
  } else {
    if (a.tile_tab) launch<TC_DTYPE_BF16, true>(a, stream); else launch<TC_DTYPE_BF16, false>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace tc
