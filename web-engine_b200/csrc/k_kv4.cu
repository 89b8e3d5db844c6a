// A paged 4-bit K/V cache (we_kv4_cache): rows in, rows out, and the attention of a step's new tokens over it.
#include "common.cuh"
#include "kernels.h"

namespace we {

// Row index (in rows of `dim` values) of token t of sequence b and kv head h, or -1 when the page table does not hold
// it (recorded in the device error word).
__device__ __forceinline__ int64_t kv4_row(const we_kv4_cache& c, int64_t b, int64_t h, int64_t t, uint32_t* err) {
  const int64_t slot = t / c.page;
  if (slot >= c.max_pages) {
    atomicCAS(err, 0u, (uint32_t)DEV_ERR_KV_FULL);
    return -1;
  }
  const int64_t id = c.page_table[b * c.max_pages + slot];
  if (id < 0 || id >= c.pages) {
    atomicCAS(err, 0u, (uint32_t)DEV_ERR_KV_PAGE);
    return -1;
  }
  return (id * c.kv_heads + h) * c.page + t % c.page;
}

// One warp per (sequence, token, kv head, k or v) group of 64 values: a lane holds two.
template <int DT>
__global__ void __launch_bounds__(256) kv4_append_kernel(const we_kv4_cache c, const void* __restrict__ k,
                                                         const void* __restrict__ v, int64_t tokens, int64_t stride,
                                                         uint32_t* err) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t groups = c.dim / 64, per_token = c.kv_heads * groups * 2, all = c.batch * tokens * per_token;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < all; u += (int64_t)gridDim.x * 8) {
    const int64_t bt = u / per_token, b = bt / tokens, t = bt % tokens;
    int64_t r = u % per_token;
    const bool is_v = r >= c.kv_heads * groups;
    if (is_v) r -= c.kv_heads * groups;
    const int64_t h = r / groups, g = r % groups;
    const int64_t have = c.lengths[b];
    if (have < 0) continue;
    const int64_t row = kv4_row(c, b, h, have + t, err);
    if (row < 0) continue;
    const int64_t at = bt * stride + h * c.dim + g * 64 + 2 * lane;
    const void* src = is_v ? v : k;
    const float x0 = load_act<DT>(src, at), x1 = load_act<DT>(src, at + 1);
    const float top = warp_max(fmaxf(fabsf(x0), fabsf(x1)));
    const __half s16 = __float2half_rn(fminf(__fdiv_rn(top, 7.f), 65504.f));
    const float s = __half2float(s16);
    int q0 = 0, q1 = 0;
    if (s != 0.f) {
      q0 = (int)fminf(fmaxf(rintf(__fdiv_rn(x0, s)), -8.f), 7.f);
      q1 = (int)fminf(fmaxf(rintf(__fdiv_rn(x1, s)), -8.f), 7.f);
    }
    (is_v ? c.v : c.k)[row * (c.dim / 2) + g * 32 + lane] = (uint8_t)((q0 & 15) | ((q1 & 15) << 4));
    if (lane == 0) (is_v ? c.v_scale : c.k_scale)[row * groups + g] = __half_as_ushort(s16);
  }
}

template <int DT>
__global__ void __launch_bounds__(256) kv4_unpack_kernel(const we_kv4_cache c, void* __restrict__ k, void* __restrict__ v,
                                                         int64_t tokens, const int32_t* __restrict__ start,
                                                         uint32_t* err) {
  pdl_wait();
  pdl_launch_dependents();
  // a thread: 8 values of one row, of k and of v
  const int64_t per_row = c.dim / 8, all = c.batch * tokens * c.kv_heads * per_row;
  for (int64_t u = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; u < all; u += (int64_t)gridDim.x * blockDim.x) {
    const int64_t bt = u / (c.kv_heads * per_row), b = bt / tokens, t = bt % tokens;
    const int64_t h = u / per_row % c.kv_heads, e = u % per_row;
    const int64_t have = c.lengths[b], from = start ? (int64_t)start[b] : have;
    const int64_t row = have < 0 || from < 0 ? -1 : kv4_row(c, b, h, from + t, err);
#pragma unroll
    for (int side = 0; side < 2; side++) {
      void* out = side ? v : k;
      if (!out) continue;
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (row >= 0) {
        const uint32_t word = *reinterpret_cast<const uint32_t*>((side ? c.v : c.k) + row * (c.dim / 2) + e * 4);
        const float s = __half2float(__ushort_as_half((side ? c.v_scale : c.k_scale)[row * (c.dim / 64) + e / 8]));
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = (float)(int(((word >> (4 * j)) & 15u) ^ 8u) - 8) * s;
      }
      store8<DT>(out, (bt * c.kv_heads + h) * c.dim + e * 8, x);
    }
  }
}

__global__ void kv4_advance_kernel(int32_t* lengths, int64_t batch, int32_t tokens) {
  pdl_wait();
  pdl_launch_dependents();
  for (int64_t b = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; b < batch; b += (int64_t)gridDim.x * blockDim.x)
    if (lengths[b] >= 0) lengths[b] += tokens;
}

// One warp per (sequence, token, head): online softmax over the keys, a lane holding dims 2 lane, 2 lane + 1 of each 64.
template <int DT, int OT, int D>
__global__ void __launch_bounds__(128) kv4_attention_simple_kernel(const Kv4AttnArgs a, uint32_t* err) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int G = D / 64;
  const we_kv4_cache& c = a.c;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= c.batch * a.tokens * a.heads) return;
  const int64_t bt = row / a.heads, h = row % a.heads, b = bt / a.tokens, i = bt % a.tokens;
  const int64_t kvh = h / (a.heads / c.kv_heads), have = c.lengths[b];
  float q[2 * G], o[2 * G], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 2 * G; e++) {
    q[e] = load_act<DT>(a.q, bt * a.q_stride + h * D + (e / 2) * 64 + 2 * lane + (e & 1)) * a.scale;
    o[e] = 0.f;
  }
  const int64_t keys = have < 0 ? 0 : have + i + 1;
  for (int64_t t = 0; t < keys; t++) {
    const int64_t r = kv4_row(c, b, kvh, t, err);
    if (r < 0) continue;
    float dot = 0.f, vv[2 * G];
#pragma unroll
    for (int g = 0; g < G; g++) {
      const float ks = __half2float(__ushort_as_half(c.k_scale[r * G + g]));
      const float vs = __half2float(__ushort_as_half(c.v_scale[r * G + g]));
      const uint32_t kb = c.k[r * (D / 2) + g * 32 + lane], vb = c.v[r * (D / 2) + g * 32 + lane];
      dot = fmaf((float)(int((kb & 15u) ^ 8u) - 8) * ks, q[2 * g], dot);
      dot = fmaf((float)(int((kb >> 4) ^ 8u) - 8) * ks, q[2 * g + 1], dot);
      vv[2 * g] = (float)(int((vb & 15u) ^ 8u) - 8) * vs;
      vv[2 * g + 1] = (float)(int((vb >> 4) ^ 8u) - 8) * vs;
    }
    const float s = warp_sum(dot), mn = fmaxf(m, s);
    const float corr = expf(m - mn), p = expf(s - mn);
    l = l * corr + p;
#pragma unroll
    for (int e = 0; e < 2 * G; e++) o[e] = o[e] * corr + p * vv[e];
    m = mn;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < 2 * G; e++)
    store_out<OT>(a.out, bt * a.out_stride + h * D + (e / 2) * 64 + 2 * lane + (e & 1), o[e] * inv);
}

static unsigned grid_of(int64_t work, int per_cta, int sms, int ctas_per_sm) {
  const int64_t g = (work + per_cta - 1) / per_cta, cap = (int64_t)sms * ctas_per_sm;
  return (unsigned)(g < cap ? g : cap);
}

cudaError_t launch_kv4_append(const we_kv4_cache& c, const void* k, const void* v, int dt, int64_t tokens,
                              int64_t stride, uint32_t* err, int sms, cudaStream_t st) {
  const unsigned grid = grid_of(c.batch * tokens * c.kv_heads * (c.dim / 64) * 2, 8, sms, 16);
  const cudaError_t e = dt == WE_F32 ? launch_pdl(kv4_append_kernel<WE_F32>, dim3(grid), 256, 0, st, c, k, v, tokens, stride, err)
                                     : launch_pdl(kv4_append_kernel<WE_BF16>, dim3(grid), 256, 0, st, c, k, v, tokens, stride, err);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

cudaError_t launch_kv4_unpack(const we_kv4_cache& c, void* k, void* v, int dt, int64_t tokens, const int32_t* start,
                              uint32_t* err, int sms, cudaStream_t st) {
  const unsigned grid = grid_of(c.batch * tokens * c.kv_heads * (c.dim / 8), 256, sms, 8);
  const cudaError_t e = dt == WE_F32 ? launch_pdl(kv4_unpack_kernel<WE_F32>, dim3(grid), 256, 0, st, c, k, v, tokens, start, err)
                                     : launch_pdl(kv4_unpack_kernel<WE_BF16>, dim3(grid), 256, 0, st, c, k, v, tokens, start, err);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

cudaError_t launch_kv4_advance(const we_kv4_cache& c, int64_t tokens, cudaStream_t st) {
  const unsigned grid = (unsigned)((c.batch + 127) / 128);
  const cudaError_t e = launch_pdl(kv4_advance_kernel, dim3(grid), 128, 0, st, c.lengths, c.batch, (int32_t)tokens);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

template <int DT, int OT>
static cudaError_t attention_simple(const Kv4AttnArgs& a, uint32_t* err, cudaStream_t st) {
  const dim3 grid((unsigned)((a.c.batch * a.tokens * a.heads + 3) / 4));
  if (a.c.dim == 64) return launch_pdl(kv4_attention_simple_kernel<DT, OT, 64>, grid, 128, 0, st, a, err);
  if (a.c.dim == 128) return launch_pdl(kv4_attention_simple_kernel<DT, OT, 128>, grid, 128, 0, st, a, err);
  return launch_pdl(kv4_attention_simple_kernel<DT, OT, 256>, grid, 128, 0, st, a, err);
}

cudaError_t launch_kv4_attention(const Kv4AttnArgs& a, uint32_t* err, int sms, cudaStream_t st) {
  const bool qf = a.dtype == WE_F32, of = a.out_dtype == WE_F32;
  const cudaError_t e = qf ? (of ? attention_simple<WE_F32, WE_F32>(a, err, st) : attention_simple<WE_F32, WE_BF16>(a, err, st))
                           : (of ? attention_simple<WE_BF16, WE_F32>(a, err, st) : attention_simple<WE_BF16, WE_BF16>(a, err, st));
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace we
