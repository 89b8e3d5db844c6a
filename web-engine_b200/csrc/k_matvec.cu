// Few rows of activations times int4 group-64 weights (a decoder's single tokens):
//   y[i, n] = sum_g s[n, g] sum_{j in g} q[n, j] x[i, j]   (+ bias, activation, aux, gate, accumulate)
#include "common.cuh"
#include "kernels.h"

namespace we {

// v = the product plus bias -> the value to store (the epilogue order of we_matmul)
__device__ __forceinline__ float matvec_epilogue(float v, const MatmulArgs& a, int64_t i, int64_t n, const void* y) {
  if (a.bias) v += a.bias[n];
  v = act_apply(a.epi.act, v);
  if (a.epi.aux_op) {
    const int64_t at = i * a.y_stride + n;
    const float aux = a.epi.aux_dtype == WE_F32 ? static_cast<const float*>(a.epi.aux)[at]
                                                : bf16_bits_to_f32(static_cast<const uint16_t*>(a.epi.aux)[at]);
    v = aux_apply(a.epi.aux_op, aux, v);
  }
  if (a.epi.gate) v *= a.epi.gate[n];
  if (a.accumulate) {
    const int64_t at = i * a.y_stride + n;
    v += a.y_dtype == WE_F32 ? static_cast<const float*>(y)[at] : bf16_bits_to_f32(static_cast<const uint16_t*>(y)[at]);
  }
  return v;
}

// One warp per output channel; a lane takes 8 values (4 packed bytes) of every 256.
template <int XT>
__global__ void __launch_bounds__(256) matvec_kernel(const void* __restrict__ x, const uint8_t* __restrict__ w, void* y,
                                                     const MatmulArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= a.n) return;
  float acc[WE_MATVEC_MAX_ROWS];
#pragma unroll
  for (int i = 0; i < WE_MATVEC_MAX_ROWS; i++) acc[i] = 0.f;
  const int64_t groups = a.k / 64;
  for (int64_t k0 = lane * 8; k0 < a.k; k0 += 256) {
    const uint32_t word = *reinterpret_cast<const uint32_t*>(w + n * (a.k / 2) + k0 / 2);
    const float s = __half2float(__ushort_as_half(a.group_scale[n * groups + k0 / 64]));
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float wv = (float)(int(((word >> (4 * j)) & 15u) ^ 8u) - 8) * s;
#pragma unroll
      for (int i = 0; i < WE_MATVEC_MAX_ROWS; i++)
        if (i < a.m) acc[i] = fmaf(wv, load_act<XT>(x, i * a.x_stride + k0 + j), acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < WE_MATVEC_MAX_ROWS; i++) {
    if (i >= a.m) break;
    const float v = warp_sum(acc[i]);
    if (lane == 0) {
      const float r = matvec_epilogue(v, a, i, n, y);
      if (a.y_dtype == WE_F32) store_out<WE_F32>(y, i * a.y_stride + n, r);
      else store_out<WE_BF16>(y, i * a.y_stride + n, r);
    }
  }
}

cudaError_t launch_matvec(const void* x, const void* w, void* y, const MatmulArgs& a, int sms, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.n + 7) / 8);
  const cudaError_t e =
      a.x_dtype == WE_F32
          ? launch_pdl(matvec_kernel<WE_F32>, dim3(grid), 256, 0, st, x, static_cast<const uint8_t*>(w), y, a)
          : launch_pdl(matvec_kernel<WE_BF16>, dim3(grid), 256, 0, st, x, static_cast<const uint8_t*>(w), y, a);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace we
