// Cross attention: queries of one sequence over another sequence's keys and values, with key lengths and a byte mask.
#include "common.cuh"
#include "kernels.h"

namespace we {

// One warp per (entry, query, head), fp32 online softmax, any dim up to 256 and any stride.
template <int DT, int OT, int VPL>
__global__ void __launch_bounds__(128) cross_simt_kernel(const we_cross_desc d) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t rows = d.batch * d.tq * d.heads, group = d.heads / d.kv_heads;
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); row < rows; row += (int64_t)gridDim.x * 4) {
    const int64_t bt = row / d.heads, h = row % d.heads, b = bt / d.tq, g = h / group;
    int64_t n = d.tk;
    if (d.key_lengths) {
      const int64_t len = d.key_lengths[b];
      n = len < n ? len : n;
    }
    float q[VPL], o[VPL], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < VPL; e++) {
      const int64_t x = lane + 32 * e;
      q[e] = x < d.dim ? load_act<DT>(d.q, bt * d.q_stride + h * d.dim + x) * d.scale : 0.f;
      o[e] = 0.f;
    }
    for (int64_t j = 0; j < n; j++) {
      const int64_t t = b * d.tk + j;
      if (d.key_mask && !d.key_mask[t]) continue;
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < VPL; e++) {
        const int64_t x = lane + 32 * e;
        if (x < d.dim) dot = fmaf(q[e], load_act<DT>(d.k, t * d.k_stride + g * d.dim + x), dot);
      }
      const float s = warp_sum(dot), mn = fmaxf(m, s);
      if (mn == -INFINITY) continue;  // only scores of -inf so far: no weight yet
      const float corr = expf(m - mn), p = expf(s - mn);
      l = l * corr + p;
#pragma unroll
      for (int e = 0; e < VPL; e++) {
        const int64_t x = lane + 32 * e;
        o[e] = o[e] * corr + (x < d.dim ? p * load_act<DT>(d.v, t * d.v_stride + g * d.dim + x) : 0.f);
      }
      m = mn;
    }
#pragma unroll
    for (int e = 0; e < VPL; e++) {
      const int64_t x = lane + 32 * e;
      // l = 0: no key was seen
      if (x < d.dim) store_out<OT>(d.out, bt * d.out_stride + h * d.dim + x, l == 0.f ? 0.f : o[e] / l);
    }
  }
}

template <int DT, int OT>
static cudaError_t cross_simt(const we_cross_desc& d, int sms, cudaStream_t st) {
  const int64_t rows = d.batch * d.tq * d.heads;
  int64_t g = (rows + 3) / 4;
  if (g > (int64_t)sms * 16) g = (int64_t)sms * 16;
  const dim3 grid((unsigned)g);
  if (d.dim <= 32) return launch_pdl(cross_simt_kernel<DT, OT, 1>, grid, 128, 0, st, d);
  if (d.dim <= 64) return launch_pdl(cross_simt_kernel<DT, OT, 2>, grid, 128, 0, st, d);
  if (d.dim <= 128) return launch_pdl(cross_simt_kernel<DT, OT, 4>, grid, 128, 0, st, d);
  return launch_pdl(cross_simt_kernel<DT, OT, 8>, grid, 128, 0, st, d);
}

cudaError_t launch_cross_simt(const we_cross_desc& d, int sms, cudaStream_t st) {
  const bool f = d.dtype == WE_F32, of = d.out_dtype == WE_F32;
  const cudaError_t e = f ? (of ? cross_simt<WE_F32, WE_F32>(d, sms, st) : cross_simt<WE_F32, WE_BF16>(d, sms, st))
                          : (of ? cross_simt<WE_BF16, WE_F32>(d, sms, st) : cross_simt<WE_BF16, WE_BF16>(d, sms, st));
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace we
