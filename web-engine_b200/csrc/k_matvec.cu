// Few rows of activations times int4 group-64 weights (a decoder's single tokens):
//   y[i, n] = sum_g s[n, g] sum_{j in g} q[n, j] x[i, j]   (+ bias, activation, aux, gate, accumulate)
//
// The weights are read once and bound the call (n k / 2 + n k / 32 bytes); what has to be kept small beside them is the
// number of instructions per weight. Tensor-core tiles of 16 channels x 8 columns x 16 values (mma.sync) take the
// weights straight from the registers they are unpacked in; a tcgen05 product would need them written to shared memory
// as a 128-row operand first, four times the bytes that are read. The columns are the tokens, so 1 to 8 tokens cost the
// same.
// - Codes become bf16 by one logical operation and one addition per pair: 0x4300 | (code ^ 8) is 136 + q, minus 136
//   exact. bf16 x is the other operand as it is; f32 x is three columns per token, the exact bf16 pieces of its 24 bits.
//   So every product is exact, a group's 64 products are summed in f32 by the tensor core, and the group scale is one
//   f32 multiply-add per group and output.
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
constexpr int DEPTH = 3;                       // steps in a warp's ring
constexpr int RING = WARPS * DEPTH * STAGE;
constexpr int MAX_PAIRS = 8;                   // tile pairs of one CTA (their sums wait in shared memory)
constexpr int MAX_CLUSTER = 8;

struct Plan {
  int pairs;        // tile pairs per CTA
  int cluster;      // CTAs that split k
  int kb_per_cta;   // steps of 256 values per CTA
  int x_pitch;      // bytes from one row of x to the next in shared memory
  int smem;
};
}  // namespace mv

__device__ __forceinline__ void cp_async16_zfill(uint32_t smem, const void* gmem, bool full) {
  const int n = full ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(n) : "memory");
}

// d += a b: 16 x 8 x 16, bf16 operands, f32 sums (the legacy warp-level tensor instruction; see the file's head)
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The pair of codes j and j + 4 of a packed word as exact bf16 values: 0x4300 | (code ^ 8) = 136 + q, minus 136.
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int j) {
  const uint32_t u = ((word >> (4 * j)) & 0x000f000fu) ^ 0x43084308u;
  const uint32_t off = 0xc308c308u;  // -136
  const __nv_bfloat162 r = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&off));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// XT: type of x; NT: tiles of 8 columns. Column c is token c (bf16), or piece c / m of token c % m (f32).
template <int XT, int NT>
__global__ void __launch_bounds__(mv::THREADS) matvec_mma_kernel(const void* __restrict__ x, const uint8_t* __restrict__ w,
                                                                 void* y, const MatmulArgs a, const mv::Plan p) {
  using namespace mv;
  constexpr int XB = XT == WE_F32 ? 4 : 2;
  constexpr int COLS = NT * 8;
  extern __shared__ __align__(16) uint8_t smem[];
  const int m = (int)a.m, n = (int)a.n;
  const int groups = (int)(a.k / 64);
  uint8_t* xs = smem + RING;                                                    // [m] rows of x_pitch bytes
  float* red = reinterpret_cast<float*>(xs + m * p.x_pitch);                    // [WARPS][ROWS][COLS]
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
  pdl_launch_dependents();
  pdl_wait();

  const uint32_t ring = tc::smem_u32(smem) + (uint32_t)(warp * DEPTH * STAGE);
  const int64_t row_bytes = a.k / 2;
  uint16_t sc[DEPTH][2 * RT];  // the stage's scales: value 32 j + lane = (channel, group of the step)
  // step `item` into stage `st`: a lane copies 16 of 128 bytes of every fourth channel
  auto fetch = [&](int item, int st) {
    const int pr = item / my_kbs, kb = warp + (item - pr * my_kbs) * WARPS;
    const int c0 = (pair0 + pr) * ROWS;
    const int gfirst = g0 + kb * KB_GROUPS;
    const int chunk = lane & 7;
    const bool inside = kb * KB_GROUPS + (chunk >> 1) < my_groups;
    const int64_t col = (int64_t)gfirst * 32 + chunk * 16;
#pragma unroll
    for (int i = 0; i < ROWS / 4; i++) {
      const int r = i * 4 + (lane >> 3);
      const bool ok = inside && c0 + r < n;
      const uint32_t dst = ring + st * STAGE + r * 128 + ((((chunk >> 1) ^ (r & 3)) << 1) | (chunk & 1)) * 16;
      cp_async16_zfill(dst, ok ? w + (int64_t)(c0 + r) * row_bytes + col : w, ok);
    }
#pragma unroll
    for (int j = 0; j < 2 * RT; j++) {
      const int r = j * 8 + (lane >> 2), g = lane & 3;
      const bool ok = kb * KB_GROUPS + g < my_groups && c0 + r < n;
      sc[st][j] = ok ? a.group_scale[(int64_t)(c0 + r) * groups + gfirst + g] : (uint16_t)0;
    }
  };
#pragma unroll
  for (int d = 0; d < DEPTH; d++) {
    if (d < items) fetch(d, d);
    cp_async_commit();
  }

  // x, in 8-byte words where its rows allow, else value by value; zeros up to whole steps. The tensor core takes
  // subnormal operands as zeros, so a row without a value of 2^-60 or more is worked on times 2^60 (exact).
  __shared__ int large[WE_MATVEC_MAX_ROWS];
  if (threadIdx.x < WE_MATVEC_MAX_ROWS) large[threadIdx.x] = 0;
  __syncthreads();
  auto each_word = [&](auto &&f) {
    const int per_row = kbs * KB * XB / 8;
    for (int u = threadIdx.x; u < m * per_row; u += THREADS) {
      const int i = u / per_row, e = u - i * per_row;
      f(i, reinterpret_cast<uint2*>(xs + i * p.x_pitch + e * 8), e);
    }
  };
  {
    const int vals = my_groups * 64;
    const char* src = static_cast<const char*>(x) + (int64_t)g0 * 64 * XB;
    const bool wide = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t)(a.x_stride * XB)) & 7) == 0;
    each_word([&](int i, uint2* to, int e) {
      uint2 v = make_uint2(0, 0);
      if (e * 8 < vals * XB) {
        const char* from = src + (int64_t)i * a.x_stride * XB + e * 8;
        if (wide) {
          v = *reinterpret_cast<const uint2*>(from);
        } else if constexpr (XB == 4) {
          v.x = reinterpret_cast<const uint32_t*>(from)[0];
          v.y = reinterpret_cast<const uint32_t*>(from)[1];
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(from);
          v.x = h[0] | (uint32_t)h[1] << 16;
          v.y = h[2] | (uint32_t)h[3] << 16;
        }
      }
      *to = v;
      // 2^-60 is 0x21800000 in f32, 0x2180 in bf16
      const bool big = XB == 4 ? (v.x & 0x7fffffffu) >= 0x21800000u || (v.y & 0x7fffffffu) >= 0x21800000u
                               : __vcmpgeu2(v.x & 0x7fff7fffu, 0x21802180u) || __vcmpgeu2(v.y & 0x7fff7fffu, 0x21802180u);
      if (big) large[i] = 1;
    });
  }
  __syncthreads();
  each_word([&](int i, uint2* to, int) {
    if (large[i]) return;
    uint2 v = *to;
    constexpr float UP = 1152921504606846976.f;  // 2^60
    if constexpr (XB == 4) {
      v.x = __float_as_uint(__uint_as_float(v.x) * UP);
      v.y = __float_as_uint(__uint_as_float(v.y) * UP);
    } else {
      v.x = pack_bf16x2(__uint_as_float(v.x << 16) * UP, __uint_as_float(v.x & 0xffff0000u) * UP);
      v.y = pack_bf16x2(__uint_as_float(v.y << 16) * UP, __uint_as_float(v.y & 0xffff0000u) * UP);
    }
    *to = v;
  });
  __syncthreads();

  // this lane's columns as the B operand: column nt * 8 + lane / 4
  int tok[NT], piece[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int col = t * 8 + (lane >> 2);
    piece[t] = XT == WE_F32 ? col / m : 0;
    tok[t] = col < (XT == WE_F32 ? 3 * m : m) ? (XT == WE_F32 ? col % m : col) : -1;
  }
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
      uint32_t b[NT][8];  // 16 values of x as 8 pairs (v, v + 4) in the order of code_pair
#pragma unroll
      for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int i = 0; i < 8; i++) b[t][i] = 0;
        if (tok[t] >= 0) {
          const uint8_t* src = xs + tok[t] * p.x_pitch + (kb * KB + g * 64 + (lane & 3) * 16) * XB;
          if constexpr (XT == WE_F32) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              float v[8];
              load8f(reinterpret_cast<const float*>(src), 8 * i, v);
#pragma unroll
              for (int j = 0; j < 8; j++) {
                // piece 0, 1 or 2: the leading 8 bits of what the pieces before leave (exact)
                const float h0 = __uint_as_float(__float_as_uint(v[j]) & 0xffff0000u);
                const float r1 = h0 == v[j] ? 0.f : v[j] - h0;  // an infinity is its own first piece
                const float h1 = __uint_as_float(__float_as_uint(r1) & 0xffff0000u);
                v[j] = piece[t] == 0 ? h0 : (piece[t] == 1 ? h1 : r1 - h1);
              }
#pragma unroll
              for (int j = 0; j < 4; j++) b[t][4 * i + j] = __byte_perm(__float_as_uint(v[j]), __float_as_uint(v[j + 4]), 0x7632);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const uint4 u = *reinterpret_cast<const uint4*>(src + 16 * i);
              b[t][4 * i] = __byte_perm(u.x, u.z, 0x5410);
              b[t][4 * i + 1] = __byte_perm(u.x, u.z, 0x7632);
              b[t][4 * i + 2] = __byte_perm(u.y, u.w, 0x5410);
              b[t][4 * i + 3] = __byte_perm(u.y, u.w, 0x7632);
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const int row = r * 16 + (lane >> 2);  // and row + 8 (the same swizzle)
        const uint8_t* at = tile + row * 128 + ((g ^ (row & 3)) << 5) + (lane & 3) * 8;
        const uint2 lo = *reinterpret_cast<const uint2*>(at);
        const uint2 hi = *reinterpret_cast<const uint2*>(at + 8 * 128);
        float d[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int e = 0; e < 4; e++) d[t][e] = 0.f;
#pragma unroll
        for (int s = 0; s < 4; s++) {
          const uint32_t wl = s < 2 ? lo.x : lo.y, wh = s < 2 ? hi.x : hi.y;
          const int j = (s & 1) * 2;
          const uint32_t av[4] = {code_pair(wl, j), code_pair(wh, j), code_pair(wl, j + 1), code_pair(wh, j + 1)};
#pragma unroll
          for (int t = 0; t < NT; t++) mma_bf16(d[t], av, b[t][2 * s], b[t][2 * s + 1]);
        }
        const uint32_t both = __shfl_sync(0xffffffffu, (uint32_t)sc[st][2 * r] | (uint32_t)sc[st][2 * r + 1] << 16,
                                          (lane & ~3) | g);
        const float s0 = __half2float(__ushort_as_half((uint16_t)both)), s1 = __half2float(__ushort_as_half((uint16_t)(both >> 16)));
#pragma unroll
        for (int t = 0; t < NT; t++) {
          acc[r][t][0] = fmaf(s0, d[t][0], acc[r][t][0]);
          acc[r][t][1] = fmaf(s0, d[t][1], acc[r][t][1]);
          acc[r][t][2] = fmaf(s1, d[t][2], acc[r][t][2]);
          acc[r][t][3] = fmaf(s1, d[t][3], acc[r][t][3]);
        }
      }
    }
  };

  // The pair's sums over this CTA's part of k: the warps' sums in turn, then (f32) the pieces of a token.
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
      constexpr int PIECES = XT == WE_F32 ? 3 : 1;
#pragma unroll
      for (int c = PIECES - 1; c >= 0; c--) {  // the smallest piece first
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; k++) s += red[k * (ROWS * COLS) + row * COLS + c * m + i];
        v += s;
      }
      part[pr * (ROWS * m) + u] = large[i] ? v : v * 8.673617379884035e-19f;  // 2^-60
    }
  };

  int pr = 0, left = my_kbs;  // the pair in work and its steps left (a warp without steps only joins the barriers)
  for (int base = 0; base < items; base += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
      const int item = base + d;
      if (item < items) {
        cp_async_wait<DEPTH - 1>();
        __syncwarp();
        step(warp + (my_kbs - left) * WARPS, d);
        __syncwarp();
        if (item + DEPTH < items) fetch(item + DEPTH, d);
        cp_async_commit();
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
  const int xb = f32 ? 4 : 2;
  const int cols = (int)a.m * (f32 ? 3 : 1);
  const int nt = cols <= 8 ? 1 : (cols <= 16 ? 2 : (cols <= 24 ? 3 : 6));
  const int64_t all_pairs = (a.n + ROWS - 1) / ROWS, kbs = (a.k + KB - 1) / KB;
  Plan p{};
  auto fill = [&](int cluster, int64_t pairs) {
    p.cluster = cluster;
    p.pairs = (int)pairs;
    p.kb_per_cta = (int)((kbs + cluster - 1) / cluster);
    // rows 16 bytes past a multiple of 128: two tokens' 16-byte reads fall into different banks
    p.x_pitch = p.kb_per_cta * KB * xb + 16;
    const int64_t bytes = RING + a.m * (int64_t)p.x_pitch + ((int64_t)WARPS * ROWS * nt * 8 + pairs * ROWS * a.m) * 4;
    p.smem = bytes <= 227 * 1024 ? (int)bytes : -1;
    return p.smem > 0;
  };
  // The fewest CTAs that split k (1, 2, 4, 8) which fill the SMs, and more where x needs it to fit; then as many tile
  // pairs a CTA as put the whole product in one wave of two CTAs an SM.
  int cluster = 1;
  while (cluster < MAX_CLUSTER && cluster * 2 * WARPS <= kbs * 2 && all_pairs * cluster < sms) cluster *= 2;
  bool ok = false;
  for (; cluster <= MAX_CLUSTER; cluster *= 2) {
    const int64_t slots = std::max<int64_t>(1, (int64_t)sms * 2 / cluster);
    const int64_t pairs = std::min<int64_t>(MAX_PAIRS, (all_pairs + slots - 1) / slots);
    if ((ok = fill(cluster, pairs))) break;
  }
  if (!ok || (all_pairs + p.pairs - 1) / p.pairs > 65535) {
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
                  : matvec_mma<WE_F32, 6>(x, w, y, a, p, gy, st);
  } else {
    e = nt == 1 ? matvec_mma<WE_BF16, 1>(x, w, y, a, p, gy, st) : matvec_mma<WE_BF16, 2>(x, w, y, a, p, gy, st);
  }
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace we
