// New tokens' K/V rows written into the page slots of a paged cache, with the
// position rotation applied on the way: the keys (and the queries of the same
// tokens, if given) arrive as the projections left them, are rotated to their
// positions as threadcut/kv.py:20-25 rotates (k*cos + rotate_half(k)*sin in
// fp32, rounded once), and the keys go straight to their slots; the values are
// copied. One launch for K, V and Q of one or more layers.
//
// Bound: HBM (each byte read and written once). A thread owns 16 dims of a
// token's rows, the 8 lower ones and the 8 that rotate_half pairs them with,
// so a rotation stays inside a thread; its 8 angles serve kHeads heads, whose
// loads are all in flight before the first store.
//
// An angle is position * inv_freq, of which only the part of a turn counts.
// At position 10^6 a product in 32 bits is off by up to 0.03 rad, so turns =
// position * (inv_freq / 2 pi) is taken in 64 bits, its whole part dropped
// there, and sin and cos of the rest (at most half a turn) in 32 bits.
#include "tc_common.hpp"

namespace tc {
namespace {

constexpr int kHeadDim = 128;
constexpr int kHalf = kHeadDim / 2;
constexpr int kThreads = 256;
constexpr int kChunks = kHalf / 8;                 // threads of a row
constexpr int kTileRows = kThreads / kChunks;      // tokens of a work-group
constexpr int kMaxLayers = 48;

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <int LAYERS>
struct RopeArgs {
  const uint16_t* k[LAYERS];
  const uint16_t* v[LAYERS];
  const uint16_t* q[LAYERS];
  uint16_t* k_pool[LAYERS];
  uint16_t* v_pool[LAYERS];
  uint16_t* q_out[LAYERS];
  int64_t sk[3], sv[3], sq[3];      // (batch, head, token) strides of the rows
  int64_t sp[3];                    // (page, head, slot) strides of the pools
  int64_t so[3];                    // (batch, head, token) strides of the rotated queries
  const int4* slots;                // [batch * rows] {page, slot, position, -}
  const float* freq_dev;            // inv_freq on the device, or null: freq
  float freq[kHalf];
  uint32_t total, rows;             // tokens of the call; of a sequence
  int kv_heads, q_heads;
  int pages, page_tokens;
};

// Grid (tiles of 32 tokens, groups of HEADS heads: K, then V, then Q, layers).
template <int DT, int LAYERS, int HEADS>
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(const RopeArgs<LAYERS> a) {
  const int u = threadIdx.x & (kChunks - 1);
  const uint32_t t = blockIdx.x * kTileRows + threadIdx.x / kChunks;
  if (t >= a.total) return;
  const int layer = LAYERS == 1 ? 0 : static_cast<int>(blockIdx.z);
  const int groups = (a.kv_heads + HEADS - 1) / HEADS;
  const int group = static_cast<int>(blockIdx.y);
  const int kind = group < groups ? 0 : group < 2 * groups ? 1 : 2;  // K, V, Q
  const int h0 = (group - kind * groups) * HEADS;
  const int heads = kind == 2 ? a.q_heads : a.kv_heads;
  const int4 slot = a.slots[t];
  const uint32_t b = t / a.rows, r = t - b * a.rows;
  const int64_t* st = kind == 0 ? a.sk : kind == 1 ? a.sv : a.sq;
  const int64_t s_h = st[1];
  const uint16_t* src = (kind == 0 ? a.k[layer] : kind == 1 ? a.v[layer] : a.q[layer]) + b * st[0] + r * st[2] +
                        h0 * s_h + 8 * u;
  u32x4 lo[HEADS], hi[HEADS];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const uint16_t* p = src + (h0 + i < heads ? i : 0) * s_h;
    lo[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    hi[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + kHalf));
  }
  uint16_t* dst;
  int64_t d_h;
  if (kind == 2) {
    d_h = a.so[1];
    dst = a.q_out[layer] + b * a.so[0] + r * a.so[2] + h0 * d_h + 8 * u;
  } else {
    // A slot outside the pool is skipped.
    if (slot.x < 0 || slot.x >= a.pages || slot.y < 0 || slot.y >= a.page_tokens) return;
    d_h = a.sp[1];
    dst = (kind == 0 ? a.k_pool[layer] : a.v_pool[layer]) + slot.x * a.sp[0] + slot.y * a.sp[2] + h0 * d_h + 8 * u;
  }
  if (kind != 1) {
    const float* f = a.freq_dev ? a.freq_dev : a.freq;
    float c[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      constexpr double kPerTurn = 0.15915494309189533577;  // 1 / 2 pi
      const double turns = static_cast<double>(slot.z) * (static_cast<double>(f[8 * u + j]) * kPerTurn);
      sincospif(2.f * static_cast<float>(turns - __builtin_rint(turns)), &s[j], &c[j]);
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      uint4 x = make_uint4(lo[i].x, lo[i].y, lo[i].z, lo[i].w), y = make_uint4(hi[i].x, hi[i].y, hi[i].z, hi[i].w);
      rotate_pair<DT>(x, y, c, s);
      lo[i] = u32x4{x.x, x.y, x.z, x.w};
      hi[i] = u32x4{y.x, y.y, y.z, y.w};
    }
  }
#pragma unroll
  for (int i = 0; i < HEADS; ++i)
    if (h0 + i < heads) {
      __builtin_nontemporal_store(lo[i], reinterpret_cast<u32x4*>(dst + i * d_h));
      __builtin_nontemporal_store(hi[i], reinterpret_cast<u32x4*>(dst + i * d_h + kHalf));
    }
}

int check_strides(const char* what, const int64_t* st) {
  if (!st) return fail(TC_ERR_INVALID_ARGUMENT, "%s strides are null", what);
  for (int i = 0; i < 3; ++i) {
    if (st[i] < 0) return fail(TC_ERR_INVALID_ARGUMENT, "%s stride %d is negative", what, i);
    if (st[i] % 8) return fail(TC_ERR_ALIGNMENT, "%s stride %d (%lld) not a multiple of 8", what, i, (long long)st[i]);
  }
  return TC_OK;
}

template <int LAYERS, int HEADS>
void launch_heads(const RopeArgs<LAYERS>& a, int dtype, int layers, hipStream_t s) {
  const dim3 grid((a.total + kTileRows - 1) / kTileRows,
                  2 * ((a.kv_heads + HEADS - 1) / HEADS) + (a.q_heads + HEADS - 1) / HEADS, layers);
  if (dtype == TC_DTYPE_F16)
    hipLaunchKernelGGL((rope_rows_kernel<TC_DTYPE_F16, LAYERS, HEADS>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((rope_rows_kernel<TC_DTYPE_BF16, LAYERS, HEADS>), grid, dim3(kThreads), 0, s, a);
}

// Heads a thread takes: with more, its angles serve more rows and more of its
// loads are in flight, with fewer there are more work-groups. By the rows of
// all heads and layers (us with 1, 2, 4 and 8 heads, 8 KV and 32 query heads):
// 48 (one token) 3.40, 3.67, 4.17, 4.94; 1584 3.39, 3.61, 4.20, 5.19; 28800
// 5.77, 5.18, 5.22, 6.29; 67200 9.50, 7.98, 7.71, 8.61; 98304 11.6, 10.4, 8.30,
// 10.2; 2.5 million (24 layers, no queries) 228, 223, 228, 229.
template <int LAYERS>
void launch(const RopeArgs<LAYERS>& a, int dtype, int layers, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.total) * (2 * a.kv_heads + a.q_heads) * layers;
  if (rows <= 6000)
    launch_heads<LAYERS, 1>(a, dtype, layers, s);
  else if (rows <= 50000)
    launch_heads<LAYERS, 2>(a, dtype, layers, s);
  else
    launch_heads<LAYERS, 4>(a, dtype, layers, s);
}

}  // namespace
}  // namespace tc

using namespace tc;

extern "C" int tc_paged_append_rope(const void* const* k_rows_host, const int64_t k_strides[3],
                                    const void* const* v_rows_host, const int64_t v_strides[3],
                                    void* const* k_pools_host, void* const* v_pools_host,
                                    const int64_t pool_strides[3], int num_pages, int page_tokens,
                                    const int32_t* slots_dev, const void* const* q_rows_host,
                                    const int64_t q_strides[3], void* const* q_out_host,
                                    const int64_t q_out_strides[3], int q_heads, const float* inv_freq_host,
                                    const float* inv_freq_dev, int num_layers, int batch, int kv_heads, int64_t rows,
                                    int head_dim, int dtype, void* stream) {
  clear_error();
  int rc;
  if (num_pages < 1 || page_tokens < 1)
    return fail(TC_ERR_INVALID_ARGUMENT, "pool of %d pages of %d tokens", num_pages, page_tokens);
  if (num_layers < 0) return fail(TC_ERR_INVALID_ARGUMENT, "num_layers %d is negative", num_layers);
  if (batch < 1 || kv_heads < 1 || q_heads < 0)
    return fail(TC_ERR_INVALID_ARGUMENT, "batch %d, kv_heads %d, q_heads %d", batch, kv_heads, q_heads);
  if (head_dim != kHeadDim) return fail(TC_ERR_UNSUPPORTED, "head_dim %d unsupported (kernels are built for 128)", head_dim);
  if (dtype != TC_DTYPE_F16 && dtype != TC_DTYPE_BF16) return fail(TC_ERR_UNSUPPORTED, "dtype %d unsupported", dtype);
  if (rows < 0) return fail(TC_ERR_INVALID_ARGUMENT, "rows %lld is negative", (long long)rows);
  if (rows == 0 || num_layers == 0) return TC_OK;
  if (rows > 0x7fffffff / batch) return fail(TC_ERR_UNSUPPORTED, "%lld rows of %d sequences", (long long)rows, batch);
  if (2 * static_cast<int64_t>(kv_heads) + q_heads > 65535)
    return fail(TC_ERR_UNSUPPORTED, "%d KV heads and %d query heads exceed the grid", kv_heads, q_heads);
  if (!slots_dev) return fail(TC_ERR_INVALID_ARGUMENT, "null slot list");
  if (!aligned16(slots_dev)) return fail(TC_ERR_ALIGNMENT, "slot list not 16-byte aligned");
  if (!inv_freq_host == !inv_freq_dev)
    return fail(TC_ERR_INVALID_ARGUMENT, "inverse frequencies: one of the host's and the device's");
  if (reinterpret_cast<uintptr_t>(inv_freq_dev) & 3u) return fail(TC_ERR_ALIGNMENT, "inverse frequencies not 4-byte aligned");
  if (!k_rows_host || !v_rows_host || !k_pools_host || !v_pools_host || (q_heads && (!q_rows_host || !q_out_host)))
    return fail(TC_ERR_INVALID_ARGUMENT, "null pointer array");
  if ((rc = check_strides("k rows", k_strides)) != TC_OK) return rc;
  if ((rc = check_strides("v rows", v_strides)) != TC_OK) return rc;
  if ((rc = check_strides("pool", pool_strides)) != TC_OK) return rc;
  if (q_heads && (rc = check_strides("q rows", q_strides)) != TC_OK) return rc;
  if (q_heads && (rc = check_strides("rotated q", q_out_strides)) != TC_OK) return rc;
  if (pool_strides[2] < kHeadDim)
    return fail(TC_ERR_INVALID_ARGUMENT, "pool token stride %lld overlaps rows", (long long)pool_strides[2]);
  for (int l = 0; l < num_layers; ++l) {
    const void* p[6] = {k_rows_host[l], v_rows_host[l], k_pools_host[l], v_pools_host[l],
                        q_heads ? q_rows_host[l] : k_rows_host[l], q_heads ? q_out_host[l] : k_rows_host[l]};
    for (const void* x : p) {
      if (!x) return fail(TC_ERR_INVALID_ARGUMENT, "null pointer of layer %d", l);
      if (!aligned16(x)) return fail(TC_ERR_ALIGNMENT, "layer %d: rows, pool or output not 16-byte aligned", l);
    }
  }
  auto fill = [&](auto& a, int l0, int nl) {
    for (int i = 0; i < static_cast<int>(sizeof(a.k) / sizeof(a.k[0])); ++i) {
      const bool on = i < nl;
      a.k[i] = on ? static_cast<const uint16_t*>(k_rows_host[l0 + i]) : nullptr;
      a.v[i] = on ? static_cast<const uint16_t*>(v_rows_host[l0 + i]) : nullptr;
      a.k_pool[i] = on ? static_cast<uint16_t*>(k_pools_host[l0 + i]) : nullptr;
      a.v_pool[i] = on ? static_cast<uint16_t*>(v_pools_host[l0 + i]) : nullptr;
      a.q[i] = on && q_heads ? static_cast<const uint16_t*>(q_rows_host[l0 + i]) : nullptr;
      a.q_out[i] = on && q_heads ? static_cast<uint16_t*>(q_out_host[l0 + i]) : nullptr;
    }
    for (int i = 0; i < 3; ++i) {
      a.sk[i] = k_strides[i];
      a.sv[i] = v_strides[i];
      a.sq[i] = q_heads ? q_strides[i] : 0;
      a.sp[i] = pool_strides[i];
      a.so[i] = q_heads ? q_out_strides[i] : 0;
    }
    a.slots = reinterpret_cast<const int4*>(slots_dev);
    a.freq_dev = inv_freq_dev;
    for (int i = 0; i < kHalf; ++i) a.freq[i] = inv_freq_host ? inv_freq_host[i] : 0.f;
    a.rows = static_cast<uint32_t>(rows);
    a.total = a.rows * static_cast<uint32_t>(batch);
    a.kv_heads = kv_heads;
    a.q_heads = q_heads;
    a.pages = num_pages;
    a.page_tokens = page_tokens;
  };
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (num_layers == 1) {
    RopeArgs<1> a;
    fill(a, 0, 1);
    launch(a, dtype, 1, s);
    return hip_status(hipGetLastError(), "rotated row write launch");
  }
  for (int l0 = 0; l0 < num_layers; l0 += kMaxLayers) {
    RopeArgs<kMaxLayers> a;
    const int nl = num_layers - l0 < kMaxLayers ? num_layers - l0 : kMaxLayers;
    fill(a, l0, nl);
    launch(a, dtype, nl, s);
    if ((rc = hip_status(hipGetLastError(), "rotated row write launch")) != TC_OK) return rc;
  }
  return TC_OK;
}
