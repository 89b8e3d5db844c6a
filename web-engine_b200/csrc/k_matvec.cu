// Few rows of activations times int4 group-64 weights (a decoder's single tokens):
//   y[i, n] = sum_g s[n, g] sum_{j in g} q[n, j] x[i, j]   (+ bias, activation, aux, gate, accumulate)
//
// The weights are read once and bound the call (n k / 2 + n k / 32 bytes); what has to be kept small beside them is the
// number of instructions per weight. Tensor-core tiles of 16 channels x 8 columns x 16 values (mma.sync) take the
// weights straight from the registers they are unpacked in; a tcgen05 product would need them written to shared memory
// as a 128-row operand first, four times the bytes that are read. The columns are the tokens, so 1 to 8 tokens cost
// nearly the same.
// - Codes become f16 pairs by ONE logical operation: (word & 0x000f000f) ^ 0x00080008 are the subnormals u 2^-24 with
//   u = q + 8, and (word & 0x00f000f0) ^ 0x00800080 are u 2^-20; a shift by 8 brings the other two pairs of a word
//   there: 5 operations for 8 weights. The factor 16 is taken from the x of those places (x / 16), and the offset by
//   starting each group's sum at -8 sum(x): sum u x - 8 sum x = sum q x.
// - x is laid out once per CTA as f16 in the order of the tiles, times a power of two that brings its row's maximum to
//   2^15. bf16 values keep all their bits down to 2^-24 of the maximum (below, an error of at most 2^-36 of it); an f32
//   value is two columns, 11 bits and the next 11 times 2^10, together within 2^-22. So a product is exact or within
//   2^-22, sums are f32, and the group scale is one f32 multiply-add per group and output.
// - A warp takes 256 values of k of 32 channels at a time, through a ring of its own in shared memory (cp.async, no
//   barrier between warps); the 8 warps of a CTA split k, clusters of up to 8 CTAs split it further when there are few
//   channels or x does not fit; partial sums meet in shared memory in a fixed order, so a call always gives the same bits.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

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
__device__ __forceinline__ void matvec_store(float v, const MatmulArgs& a, int64_t i, int64_t n, void* y) {
  const float r = matvec_epilogue(v, a, i, n, y);
  if (a.y_dtype == WE_F32) store_out<WE_F32>(y, i * a.y_stride + n, r);
  else store_out<WE_BF16>(y, i * a.y_stride + n, r);
}

// ---------------- any k: one warp per output channel on the CUDA cores ----------------
// For x that does not fit the shared memory of 8 CTAs (about 1.1 MB). A lane takes 8 values (4 packed bytes) of every 256.
template <int XT>
__global__ void __launch_bounds__(256) matvec_long_kernel(const void* __restrict__ x, const uint8_t* __restrict__ w,
                                                          void* y, const MatmulArgs a) {
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
    if (lane == 0) matvec_store(v, a, i, n, y);
  }
}

// ---------------- tensor-core tiles ----------------
namespace mv {
constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int RT = 2, ROWS = RT * 16;          // channels of a tile pair
constexpr int KB_GROUPS = 4, KB = 256;         // a warp's step: 4 groups = 128 packed bytes of each channel
constexpr int STAGE = ROWS * 128;              // bytes of one step
#ifndef MV_DEPTH
#define MV_DEPTH 2
#endif
constexpr int DEPTH = MV_DEPTH;                // steps in a warp's ring
constexpr int RING = WARPS * DEPTH * STAGE;
constexpr int MAX_PAIRS = 8;                   // tile pairs of one CTA (their sums wait in shared memory)
constexpr int MAX_CLUSTER = 8;

struct Plan {
  int pairs;        // tile pairs per CTA
  int cluster;      // CTAs that split k
  int kb_per_cta;   // steps of 256 values per CTA
  int x_pitch;      // bytes from one column of x to the next in shared memory
  int smem;
};
}  // namespace mv

// d = a b + c: 16 x 8 x 16, f16 operands, f32 sums (the legacy warp-level tensor instruction; see the file's head)
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                        const float (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// f16 pair of two floats, to nearest, and its values back
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16x2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// XT: type of x; NT: tiles of 8 columns. Column c is token c (bf16), or the leading (c < m) or following bits of token
// c % m (f32).
template <int XT, int NT>
__global__ void __launch_bounds__(mv::THREADS) matvec_mma_kernel(const void* __restrict__ x, const uint8_t* __restrict__ w,
                                                                 void* y, const MatmulArgs a, const mv::Plan p) {
  using namespace mv;
  constexpr int XB = XT == WE_F32 ? 4 : 2, PIECES = XT == WE_F32 ? 2 : 1;
  constexpr int COLS = NT * 8;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t row_max[WE_MATVEC_MAX_ROWS];  // |x| of a row's slice, as bits of f32
  const int m = (int)a.m, n = (int)a.n;
  const int groups = (int)(a.k / 64);
  uint8_t* xs = smem + RING;                                                    // [m * PIECES] columns of x_pitch bytes
  float* start = reinterpret_cast<float*>(xs + m * PIECES * p.x_pitch);         // [groups of the slice][COLS]
  float* red = start + p.kb_per_cta * KB_GROUPS * COLS;                         // [WARPS][ROWS][COLS]
  float* part = red + WARPS * ROWS * COLS;                                      // [pairs][ROWS][m]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)tc::cluster_rank();
  const int pair0 = (int)blockIdx.y * p.pairs;
  const int all_pairs = (n + ROWS - 1) / ROWS;
  const int pairs = min(p.pairs, all_pairs - pair0);
  const int g0 = rank * p.kb_per_cta * KB_GROUPS;                               // first group of this CTA
  const int my_groups = max(0, min(p.kb_per_cta * KB_GROUPS, groups - g0));
  const int kbs = (my_groups + KB_GROUPS - 1) / KB_GROUPS;                      // steps of this CTA
  const int my_kbs = kbs > warp ? (kbs - warp + WARPS - 1) / WARPS : 0;         // steps warp, warp + 8, ...
  const int items = my_kbs * pairs;                                             // (pair, step), step fastest
  if (threadIdx.x < WE_MATVEC_MAX_ROWS) row_max[threadIdx.x] = 0;
  pdl_launch_dependents();
  pdl_wait();

  // Steps are fetched in the order of work. A lane copies 16 of 128 bytes of every fourth channel and loads the scales
  // 32 j + lane = (channel, group of the step). Past the last channel it reads the last one again (not stored), past the
  // last group the first one of the slice (its x is zero).
  const uint32_t ring = tc::smem_u32(smem) + (uint32_t)(warp * DEPTH * STAGE);
  const uint32_t lane_dst = ring + (lane >> 3) * 128 + (((((lane & 7) >> 1) ^ ((lane >> 3) & 3)) << 1) | (lane & 1)) * 16;
  uint32_t w_off[ROWS / 4], s_off[2 * RT];  // this lane's channels: offsets in 16 bytes, in scales
  uint32_t sc[DEPTH][2 * RT];
  int f_pair = pair0, f_kb = warp, f_item = 0;
  const uint32_t row16 = (uint32_t)(a.k / 32);
  auto place = [&] {
    const int c0 = f_pair * ROWS;
#pragma unroll
    for (int i = 0; i < ROWS / 4; i++) w_off[i] = (uint32_t)min(c0 + i * 4 + (lane >> 3), n - 1) * row16;
#pragma unroll
    for (int j = 0; j < 2 * RT; j++) s_off[j] = (uint32_t)min(c0 + j * 8 + (lane >> 2), n - 1) * (uint32_t)groups;
  };
  auto fetch = [&](int st) {
    if (f_item < items) {
      const int gw = f_kb * KB_GROUPS + ((lane & 7) >> 1), gs = f_kb * KB_GROUPS + (lane & 3);
      const uint8_t* wp = w + (int64_t)(g0 + (gw < my_groups ? gw : 0)) * 32 + (lane & 1) * 16;
      const uint16_t* sp = a.group_scale + g0 + (gs < my_groups ? gs : 0);
#pragma unroll
      for (int i = 0; i < ROWS / 4; i++) cp_async16(lane_dst + st * STAGE + i * 512, wp + (uint64_t)w_off[i] * 16);
#pragma unroll
      for (int j = 0; j < 2 * RT; j++) sc[st][j] = sp[s_off[j]];
      f_item++;
      f_kb += WARPS;
      if (f_kb >= kbs) {
        f_kb = warp;
        f_pair++;
        place();
      }
    }
    cp_async_commit();
  };
  place();
#pragma unroll
  for (int d = 0; d < DEPTH; d++) fetch(d);

  // x: units of 16 values (a lane's share of a group in a tile). First as they are, with the rows' maxima; then scaled,
  // as f16 pairs (v, v + 4) in the order of the codes, with the sums of each group.
  const int units_row = kbs * KB / 16, units = m * units_row;
  __syncthreads();
  {
    const char* src = static_cast<const char*>(x) + (int64_t)g0 * 64 * XB;
    const bool wide = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t)(a.x_stride * XB)) & 15) == 0;
    for (int base = 0; base < units; base += THREADS) {
      const int u = base + threadIdx.x;
      const int i = min(u / units_row, m - 1), e = u - i * units_row;
      uint32_t top = 0;
      if (u < units) {
        uint4 v[XB];
#pragma unroll
        for (int j = 0; j < XB; j++) v[j] = make_uint4(0, 0, 0, 0);
        if (e * 16 < my_groups * 64) {
          const char* from = src + ((int64_t)i * a.x_stride + e * 16) * XB;
#pragma unroll
          for (int j = 0; j < XB; j++) {
            if (wide) {
              v[j] = reinterpret_cast<const uint4*>(from)[j];
            } else {
              uint32_t t[4];
#pragma unroll
              for (int q = 0; q < 4; q++) {
                if constexpr (XB == 4) t[q] = reinterpret_cast<const uint32_t*>(from)[4 * j + q];
                else t[q] = reinterpret_cast<const uint16_t*>(from)[8 * j + 2 * q] |
                            (uint32_t)reinterpret_cast<const uint16_t*>(from)[8 * j + 2 * q + 1] << 16;
              }
              v[j] = make_uint4(t[0], t[1], t[2], t[3]);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < XB; j++) {
          const uint32_t t[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
          for (int q = 0; q < 4; q++) {
            if constexpr (XB == 4) top = max(top, t[q] & 0x7fffffffu);
            else top = max(top, max((t[q] << 16) & 0x7fffffffu, t[q] & 0x7fff0000u));
          }
          *reinterpret_cast<uint4*>(xs + (i + (j >> 1) * m) * p.x_pitch + e * 32 + (j & 1) * 16) = v[j];
        }
      }
      const int i0 = __shfl_sync(0xffffffffu, i, 0);
      if (__all_sync(0xffffffffu, i == i0)) {
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) atomicMax(&row_max[i0], top);
      } else if (u < units) {
        atomicMax(&row_max[i], top);
      }
    }
  }
  for (int u = threadIdx.x; u < kbs * KB_GROUPS * COLS; u += THREADS) start[u] = 0.f;  // columns without a token
  __syncthreads();
  for (int base = 0; base < units; base += THREADS) {
    const int u = base + threadIdx.x;
    const int i = min(u / units_row, m - 1), e = u - i * units_row;
    float sum[PIECES];
#pragma unroll
    for (int c = 0; c < PIECES; c++) sum[c] = 0.f;
    if (u < units) {
      const uint32_t ex = min(max(row_max[i] >> 23, 16u), 254u);
      const float up = __uint_as_float((269u - ex) << 23);  // 2^15 over the power of two of the maximum
      float v[16];
#pragma unroll
      for (int j = 0; j < XB; j++) {
        const uint4 q = *reinterpret_cast<const uint4*>(xs + (i + (j >> 1) * m) * p.x_pitch + e * 32 + (j & 1) * 16);
        const uint32_t t[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int h = 0; h < 4; h++) {
          if constexpr (XB == 4) {
            v[4 * j + h] = __uint_as_float(t[h]) * up;
          } else {
            v[8 * j + 2 * h] = __uint_as_float(t[h] << 16) * up;
            v[8 * j + 2 * h + 1] = __uint_as_float(t[h] & 0xffff0000u) * up;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < PIECES; c++) {
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {  // pair (8 (j / 4) + j % 4, + 4); odd j: x / 16
          const int at = (j >> 2) * 8 + (j & 3);
          const float down = (j & 1) ? 0.0625f : 1.f, back = (j & 1) ? 16.f : 1.f;
          // the leading bits toward zero, so that 2^16 is never reached
          const __half2 h = c + 1 < PIECES ? __halves2half2(__float2half_rz(v[at] * down), __float2half_rz(v[at + 4] * down))
                                           : __floats2half2_rn(v[at] * down, v[at + 4] * down);
          o[j] = *reinterpret_cast<const uint32_t*>(&h);
          const float2 f = unpack_f16x2(o[j]);
          sum[c] += f.x * back + f.y * back;
          if (c + 1 < PIECES) {  // what is left (below 2^5), times 2^10; nothing of an infinity
            v[at] = fabsf(v[at]) < 131072.f ? (v[at] - f.x * back) * 1024.f : 0.f;
            v[at + 4] = fabsf(v[at + 4]) < 131072.f ? (v[at + 4] - f.y * back) * 1024.f : 0.f;
          }
        }
        uint4* to = reinterpret_cast<uint4*>(xs + (i + c * m) * p.x_pitch + e * 32);
        to[0] = make_uint4(o[0], o[1], o[2], o[3]);
        to[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    }
#pragma unroll
    for (int c = 0; c < PIECES; c++) {
      sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], 1);
      sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], 2);
      if (u < units && (e & 3) == 0) start[(e >> 2) * COLS + i + c * m] = sum[c] * -4.76837158203125e-07f;  // -8 2^-24
    }
  }
  __syncthreads();

  const int cols = m * PIECES;
  float acc[RT][NT][4];
  auto clear = [&] {
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[r][t][e] = 0.f;
  };
  clear();

  auto step = [&](int kb, int st) {  // the step's values are in stage st
    const uint8_t* tile = smem + warp * DEPTH * STAGE + st * STAGE;
#pragma unroll
    for (int g = 0; g < KB_GROUPS; g++) {
      const int gs = kb * KB_GROUPS + g;
      uint4 b[NT][2];
      float c[NT][4];
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const int col = t * 8 + (lane >> 2);
        const uint4* src = reinterpret_cast<const uint4*>(xs + col * p.x_pitch + gs * 128 + (lane & 3) * 32);
        b[t][0] = b[t][1] = make_uint4(0, 0, 0, 0);
        if (col < cols) {
          b[t][0] = src[0];
          b[t][1] = src[1];
        }
        const float2 s = *reinterpret_cast<const float2*>(start + gs * COLS + t * 8 + (lane & 3) * 2);
        c[t][0] = c[t][2] = s.x;
        c[t][1] = c[t][3] = s.y;
      }
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const int row = r * 16 + (lane >> 2);  // and row + 8 (the same swizzle)
        const uint8_t* at = tile + row * 128 + ((g ^ (row & 3)) << 5) + (lane & 3) * 8;
        const uint2 lo = *reinterpret_cast<const uint2*>(at);
        const uint2 hi = *reinterpret_cast<const uint2*>(at + 8 * 128);
        float d[NT][4];
#pragma unroll
        for (int s = 0; s < 4; s++) {
          const uint32_t wl = (s < 2 ? lo.x : lo.y) >> ((s & 1) * 8), wh = (s < 2 ? hi.x : hi.y) >> ((s & 1) * 8);
          const uint32_t av[4] = {(wl & 0x000f000fu) ^ 0x00080008u, (wh & 0x000f000fu) ^ 0x00080008u,
                                  (wl & 0x00f000f0u) ^ 0x00800080u, (wh & 0x00f000f0u) ^ 0x00800080u};
#pragma unroll
          for (int t = 0; t < NT; t++) {
            const uint4& bb = b[t][s >> 1];
            mma_f16(d[t], av, (s & 1) ? bb.z : bb.x, (s & 1) ? bb.w : bb.y, s == 0 ? c[t] : d[t]);
          }
        }
        const uint32_t both = __shfl_sync(0xffffffffu, sc[st][2 * r] | sc[st][2 * r + 1] << 16, (lane & ~3) | g);
        const float2 s01 = unpack_f16x2(both);
#pragma unroll
        for (int t = 0; t < NT; t++) {
          acc[r][t][0] = fmaf(s01.x, d[t][0], acc[r][t][0]);
          acc[r][t][1] = fmaf(s01.x, d[t][1], acc[r][t][1]);
          acc[r][t][2] = fmaf(s01.y, d[t][2], acc[r][t][2]);
          acc[r][t][3] = fmaf(s01.y, d[t][3], acc[r][t][3]);
        }
      }
    }
  };

  // The pair's sums over this CTA's part of k: the warps' sums in turn, a token's pieces, and its power of two back.
  auto reduce = [&](int pr) {
    float* mine = red + warp * (ROWS * COLS);
    __syncthreads();  // the pair before has been read
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const int row = r * 16 + (lane >> 2), col = t * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(mine + row * COLS + col) = make_float2(acc[r][t][0], acc[r][t][1]);
        *reinterpret_cast<float2*>(mine + (row + 8) * COLS + col) = make_float2(acc[r][t][2], acc[r][t][3]);
      }
    __syncthreads();
    for (int u = threadIdx.x; u < ROWS * m; u += THREADS) {
      const int row = u / m, i = u - row * m;
      float v = 0.f;
#pragma unroll
      for (int c = PIECES - 1; c >= 0; c--) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; k++) s += red[k * (ROWS * COLS) + row * COLS + c * m + i];
        v = c ? s * 9.765625e-4f : v + s;  // 2^-10
      }
      const uint32_t ex = min(max(row_max[i] >> 23, 16u), 254u);
      part[pr * (ROWS * m) + u] = v * 512.f * __uint_as_float(ex << 23);  // 2^24 2^-15 2^(ex - 127)
    }
  };

  int pr = 0, left = my_kbs;  // the pair in work and its steps left (a warp without steps only joins the barriers)
  for (int base = 0; base < items; base += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
      if (base + d < items) {
        cp_async_wait<DEPTH - 1>();
        __syncwarp();
        step(warp + (my_kbs - left) * WARPS, d);
        __syncwarp();
        fetch(d);
        if (--left == 0) {
          reduce(pr);
          clear();
          pr++;
          left = my_kbs;
        }
      }
    }
  }
  if (items == 0)
    for (; pr < pairs; pr++) reduce(pr);
  __syncthreads();

  // the cluster's parts in rank order; rank q finishes the pairs q, q + size, ...
  const int size = p.cluster;
  if (size > 1) tc::cluster_sync_all();
  const uint32_t part_addr = tc::smem_u32(part);
  for (int q = rank; q < pairs; q += size) {
    for (int u = threadIdx.x; u < ROWS * m; u += THREADS) {
      const int i = u / ROWS, row = u - i * ROWS, c = (pair0 + q) * ROWS + row;
      if (c >= n) continue;
      const int at = q * (ROWS * m) + row * m + i;
      float v = 0.f;
      if (size == 1) {
        v = part[at];
      } else {
        for (int s = 0; s < size; s++) {
          float o;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o) : "r"(tc::map_rank(part_addr + 4u * at, s)));
          v += o;
        }
      }
      matvec_store(v, a, i, c, y);
    }
  }
  if (size > 1) tc::cluster_sync_all();  // no CTA leaves while another reads its part
}

template <int XT, int NT>
static cudaError_t matvec_mma(const void* x, const uint8_t* w, void* y, const MatmulArgs& a, const mv::Plan& p, int groups_y,
                              cudaStream_t st) {
  auto kern = matvec_mma_kernel<XT, NT>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.cluster, (unsigned)groups_y);
  cfg.blockDim = dim3(mv::THREADS);
  cfg.dynamicSmemBytes = (size_t)p.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  pdl_attribute(attr[1]);
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, x, w, y, a, p);
}

cudaError_t launch_matvec(const void* x, const void* wv, void* y, const MatmulArgs& a, int sms, cudaStream_t st) {
  using namespace mv;
  const uint8_t* w = static_cast<const uint8_t*>(wv);
  const bool f32 = a.x_dtype == WE_F32;
  const int cols = (int)a.m * (f32 ? 2 : 1);
  const int nt = (cols + 7) / 8;
  const int64_t all_pairs = (a.n + ROWS - 1) / ROWS, kbs = (a.k + KB - 1) / KB;
  Plan p{};
  auto fill = [&](int cluster, int64_t pairs, int64_t limit) {
    p.cluster = cluster;
    p.pairs = (int)pairs;
    p.kb_per_cta = (int)((kbs + cluster - 1) / cluster);
    // columns 16 bytes past a multiple of 128: two columns' 16-byte reads fall into different banks
    p.x_pitch = p.kb_per_cta * KB * 2 + 16;
    const int64_t bytes = RING + cols * (int64_t)p.x_pitch +
                          ((p.kb_per_cta * KB_GROUPS + WARPS * ROWS) * nt * 8 + pairs * ROWS * a.m) * 4;
    p.smem = (int)std::min<int64_t>(bytes, 1 << 30);
    return bytes <= limit;
  };
  // The fewest CTAs that split k (1, 2, 4, 8) which give every SM one, and more where x needs it for two CTAs (or else
  // one) an SM; then as many tile pairs a CTA as put the whole product in one wave.
  int least = 1;
  while (least < MAX_CLUSTER && least * WARPS < kbs && all_pairs * least < sms) least *= 2;
  bool ok = false;
  for (int per_sm = 2; per_sm >= 1 && !ok; per_sm--)
    for (int cluster = least; cluster <= MAX_CLUSTER && !ok; cluster *= 2) {
      const int64_t slots = std::max<int64_t>(1, (int64_t)sms * per_sm / cluster);
      ok = fill(cluster, std::min<int64_t>(MAX_PAIRS, (all_pairs + slots - 1) / slots), (per_sm == 2 ? 113 : 226) * 1024);
    }
  // offsets of weights are held as 32 bits, in 16 bytes
  if (!ok || (all_pairs + p.pairs - 1) / p.pairs > 65535 || a.n * (a.k / 32) > 0xffffffffLL) {
    const dim3 grid((unsigned)((a.n + 7) / 8));
    const cudaError_t e = f32 ? launch_pdl(matvec_long_kernel<WE_F32>, grid, 256, 0, st, x, w, y, a)
                              : launch_pdl(matvec_long_kernel<WE_BF16>, grid, 256, 0, st, x, w, y, a);
    return e == cudaSuccess ? cudaGetLastError() : e;
  }
  const int gy = (int)((all_pairs + p.pairs - 1) / p.pairs);
  cudaError_t e;
  if (f32) {
    e = nt == 1   ? matvec_mma<WE_F32, 1>(x, w, y, a, p, gy, st)
        : nt == 2 ? matvec_mma<WE_F32, 2>(x, w, y, a, p, gy, st)
        : nt == 3 ? matvec_mma<WE_F32, 3>(x, w, y, a, p, gy, st)
                  : matvec_mma<WE_F32, 4>(x, w, y, a, p, gy, st);
  } else {
    e = nt == 1 ? matvec_mma<WE_BF16, 1>(x, w, y, a, p, gy, st) : matvec_mma<WE_BF16, 2>(x, w, y, a, p, gy, st);
  }
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace we
