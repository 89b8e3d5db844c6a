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
// - x is laid out once per CTA as f16 in the order of the tiles, each group of 64 times a power of two that brings its
//   maximum to 2^15. bf16 values keep all their bits down to 2^-24 of the maximum (below, an error of at most 2^-36 of
//   it); an f32 value is two columns, 11 bits and the next 11 times 2^10, together within 2^-22, and its codes take one
//   more operation to be signed f16, because the offset's sums would cost 2 to 3 bits of f32. So a product is exact or
//   within 2^-22, sums are f32, and a group's two scales are one f32 multiply-add per output.
// - A lane reads 16 bytes of a channel at once, so the four lanes of a tile's row hold two groups of 64. A token
//   therefore is two columns, one per group, each zero where the lane's values belong to the other group: one product
//   gives both groups' sums side by side and each takes its own scale.
// - Weights go from global memory to registers, 128 bytes of a channel a load and 4 KB a warp ahead of their use. A CTA is
//   16 warps (x is laid out once for all of them; with two CTAs of 8 an SM, 16 tokens took 44 us and now 35), which split
//   channels and k; clusters of up to 8 CTAs split k when there are few channels or x does not fit. Partial sums meet in
//   shared memory in a fixed order, so a call always gives the same bits.
// Measured: one token of 6144 values to 16384 channels 14.4 us (3.7 TB/s; a quarter of it until x is laid out and the first
// weights are there, then 6 TB/s), to 1536 channels 5.0; 8 tokens of 16384 to 6144 22.9, 16 tokens 37 (tensor tiles at 70% of
// the legacy instruction's rate in the main loop, x's layout and the sums a third of the time); f32, 3 tokens of 2496 values
// to 5003 channels 8.0. Tried and slower: all weights asked into L2 at once (18 us instead of 14), 256-byte bulk copies.
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
// For x that does not fit the shared memory of 8 CTAs (about 1.8 MB as f16: 53000 values of 16 tokens). A lane takes 8 values (4 packed bytes) of every 256.
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
constexpr int CHUNK = 128;       // values of k of a step: 64 packed bytes of each channel
constexpr int MAX_CLUSTER = 8;
constexpr int STEP = 2;          // chunks of a step: 128 bytes of each channel
constexpr int AHEAD = 2;         // steps that a warp loads ahead
constexpr int NOTHING = AHEAD * STEP * 256 + 128;  // bytes of zeros that lanes without a token read, on the banks that the others do not

struct Plan {
  int wk;           // warps of a CTA that split k (a power of two); the others take further channels
  int cluster;      // CTAs that split k
  int per_cta;      // chunks of 128 values per CTA
  int x_pitch;      // bytes from one token's piece to the next in shared memory
  int smem;
};
}  // namespace mv

// 16 bytes that are read once
__device__ __forceinline__ uint4 load_once16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// d += a b: 16 x 8 x 16, f16 operands, f32 sums (the legacy warp-level tensor instruction; see the file's head)
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (v & mask) ^ flip in one operation
__device__ __forceinline__ uint32_t and_xor(uint32_t v, uint32_t mask, uint32_t flip) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(v), "r"(mask), "r"(flip));
  return r;
}

__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ float2 unpack_f16x2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// A pair of codes in the low (odd = 0) or high nibbles of the halves of v, high ones times 16: as u 2^-24, u = q + 8, or
// (PIECES = 2) as q: 1024 + u - 1032, 1024 + 16 u - 1152.
template <int PIECES>
__device__ __forceinline__ uint32_t code_pair(uint32_t v, uint32_t mask, int odd) {
  if constexpr (PIECES == 1) return and_xor(v, mask, odd ? 0x00800080u : 0x00080008u);
  const uint32_t b = and_xor(v, mask, odd ? 0x64806480u : 0x64086408u);
  return as_u32(__hadd2(*reinterpret_cast<const __half2*>(&b), __float2half2_rn(odd ? -1152.f : -1032.f)));
}

// XT: type of x; NT: tiles of 8 columns; RT: row tiles of 16 channels of a warp; WARPS: of a CTA, one an SM. Columns 2 t
// and 2 t + 1 are the two groups of a chunk for piece t / m (f32: the leading bits, the following ones) of token t % m.
template <int XT, int NT, int RT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) matvec_mma_kernel(const void* __restrict__ x, const uint8_t* __restrict__ w,
                                                                 void* y, const MatmulArgs a, const mv::Plan p) {
  using namespace mv;
  constexpr int XB = XT == WE_F32 ? 4 : 2, PIECES = XT == WE_F32 ? 2 : 1;
  constexpr int THREADS = WARPS * 32, TOKS = NT * 4, ROWS = RT * 16, CHAINS = NT * RT <= 2 ? 2 : 1;
  extern __shared__ __align__(16) uint8_t smem[];
  const int m = (int)a.m, n = (int)a.n, toks = m * PIECES;
  const int groups = (int)(a.k / 64);
  uint8_t* xs = smem + NOTHING;    // [toks][chunks][quad][lane of a row][16 bytes]
  // [chunks of the slice][TOKS]: the two groups' starts (-8 sum of x) and powers of two
  float4* base = reinterpret_cast<float4*>(xs + toks * p.x_pitch);
  float* red = reinterpret_cast<float*>(base + p.per_cta * TOKS);  // [WARPS][ROWS][TOKS]
  float* part = red + WARPS * ROWS * TOKS;                         // [cluster][blocks of outputs][THREADS]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)tc::cluster_rank();
  const int kpart = warp & (p.wk - 1);                             // this warp's part of k
  const int cta_rows = WARPS / p.wk * ROWS;
  const int first = (int)blockIdx.y * cta_rows;
  const int g0 = rank * p.per_cta * 2;                             // first group of this CTA
  const int my_groups = max(0, min(p.per_cta * 2, groups - g0));
  const int chunks = (my_groups + 1) / 2;                          // of this CTA, the last one perhaps half
  const int ch0 = chunks * kpart / p.wk, end = chunks * (kpart + 1) / p.wk;  // this warp's chunks
  if (p.cluster > 1) tc::cluster_arrive();
  pdl_launch_dependents();
  pdl_wait();

  // A step's weights: a lane loads 16 bytes of channels lane / 8 + 0, 4, 8 and 12 of each row tile, eight lanes 128 bytes
  // of one (a load touches four lines; with 64 bytes of eight channels the load path took 14.4 us for 50 MB). Lanes 4 apart
  // then exchange half of it, and hold 64 bytes of both chunks of channels `channel` and + 8 between four of them.
  // Scales: lane c of the four loads the two of every fourth chunk. Past the last channel the last one is read again (not
  // stored); a lane whose group of the last chunk does not exist reads nothing there (its x is zero).
  const int channel = (lane >> 3) | (lane & 4), top_row = first + warp / p.wk * ROWS;
  uint4 raw[AHEAD][RT][4];
  uint32_t sc[RT][2], sc_next[RT][2];  // of channels `channel` and + 8
  const uint8_t* wp[RT];
  const uint16_t* sp[RT];
  int w_off[RT][4], s_off[RT];
#pragma unroll
  for (int r = 0; r < RT; r++) {
    const int at = min(top_row + r * 16 + (lane >> 3), n - 1), of = min(top_row + r * 16 + channel, n - 1);
    wp[r] = w + ((int64_t)at * groups + g0 + 2 * ch0) * 32 + (lane & 7) * 16;
    sp[r] = a.group_scale + (int64_t)of * groups + g0 + 2 * ch0 + (lane & 3) * 2;
#pragma unroll
    for (int i = 0; i < 4; i++) w_off[r][i] = (min(top_row + r * 16 + (lane >> 3) + 4 * i, n - 1) - at) * groups * 32;
    s_off[r] = (min(top_row + r * 16 + channel + 8, n - 1) - of) * groups;
  }
  const bool pairs = (groups & 1) == 0 && (reinterpret_cast<uintptr_t>(a.group_scale) & 3) == 0;  // scales two at a time
  // up to which chunk there are this lane's group (of its half of a step), and two groups
  const int lane_end = min(end, (my_groups - ((lane >> 1) & 1) + 1) / 2) - ((lane >> 2) & 1), two_end = min(end, my_groups / 2);
  auto fetch = [&](int d, int r, int c) {  // the step from chunk c on, where the pointers stand
    if (c < lane_end)
#pragma unroll
      for (int i = 0; i < 4; i++) raw[d][r][i] = load_once16(wp[r] + w_off[r][i]);
    wp[r] += STEP * 64;
  };
  auto fetch_scales = [&](int c) {  // of chunks c .. c + 3
#pragma unroll
    for (int r = 0; r < RT; r++) {
      const int mine = c + (lane & 3);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint16_t* from = sp[r] + (h ? s_off[r] : 0);
        if (pairs) {
          if (mine < end) sc_next[r][h] = __ldg(reinterpret_cast<const uint32_t*>(from));
        } else {
          if (mine < end) sc_next[r][h] = __ldg(from);
          if (mine < two_end) sc_next[r][h] |= (uint32_t)__ldg(from + 1) << 16;
        }
      }
      sp[r] += 8;
    }
  };
  // x: units of 16 values (half of a lane's share of a chunk), four neighbouring lanes a group: scaled, and as f16 pairs
  // (v, v + 4) in the order of the codes, with the sum of each group. A thread's first unit is asked for before the weights
  // (behind them it arrives some 2 us later), the next ones while one is worked on.
  const int units_row = chunks * CHUNK / 16, units = m * units_row;
  const char* src = static_cast<const char*>(x) + (int64_t)g0 * 64 * XB;
  const bool wide = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t)(a.x_stride * XB)) & 15) == 0;
  uint32_t ahead[4 * XB];  // the values as they are
  int i_ahead = 0, e_ahead = 0;  // their row, and unit of the row
  auto load_x = [&](int u) {
#pragma unroll
    for (int j = 0; j < 4 * XB; j++) ahead[j] = 0;
    i_ahead = u / units_row, e_ahead = u - i_ahead * units_row;
    if (u >= units || e_ahead * 16 >= my_groups * 64) return;
    const char* from = src + ((int64_t)i_ahead * a.x_stride + e_ahead * 16) * XB;
    if (wide) {
#pragma unroll
      for (int j = 0; j < XB; j++) {
        const uint4 q = reinterpret_cast<const uint4*>(from)[j];
        ahead[4 * j] = q.x, ahead[4 * j + 1] = q.y, ahead[4 * j + 2] = q.z, ahead[4 * j + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4 * XB; j++) {
        if constexpr (XB == 4) ahead[j] = reinterpret_cast<const uint32_t*>(from)[j];
        else ahead[j] = reinterpret_cast<const uint16_t*>(from)[2 * j] |
                        (uint32_t)reinterpret_cast<const uint16_t*>(from)[2 * j + 1] << 16;
      }
    }
  };
  if (units > 0) load_x(threadIdx.x);
#pragma unroll
  for (int r = 0; r < RT; r++) sc[r][0] = sc[r][1] = sc_next[r][0] = sc_next[r][1] = 0;
#pragma unroll
  for (int d = 0; d < AHEAD; d++) {
#pragma unroll
    for (int r = 0; r < RT; r++) {
#pragma unroll
      for (int i = 0; i < 4; i++) raw[d][r][i] = make_uint4(0, 0, 0, 0);
      fetch(d, r, ch0 + d * STEP);
    }
    if (d == 0) fetch_scales(ch0);
  }
  for (int u = threadIdx.x; u < NOTHING / 16; u += THREADS) reinterpret_cast<uint4*>(smem)[u] = make_uint4(0, 0, 0, 0);

  for (int u0 = 0; u0 < units; u0 += THREADS) {
    const bool mine = u0 + threadIdx.x < units;
    const int i = i_ahead, e = e_ahead;
    uint32_t top = 0;  // the largest magnitude's bits (bf16: of the halves, then as f32)
#pragma unroll
    for (int j = 0; j < 4 * XB; j++) top = XB == 4 ? max(top, ahead[j] & 0x7fffffffu) : __vmaxu2(top, ahead[j] & 0x7fff7fffu);
    if (XB == 2) top = max(top & 0xffff0000u, top << 16);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float2 v[8];  // the pairs of the tiles: values 8 (j / 4) + j % 4 and 4 on
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int l = (j >> 2) * 8 + (j & 3);
      if constexpr (XB == 4) v[j] = make_float2(__uint_as_float(ahead[l]), __uint_as_float(ahead[l + 4]));
      else if (j & 1) v[j] = make_float2(__uint_as_float(ahead[l >> 1] & 0xffff0000u), __uint_as_float(ahead[(l >> 1) + 2] & 0xffff0000u));
      else v[j] = make_float2(__uint_as_float(ahead[l >> 1] << 16), __uint_as_float(ahead[(l >> 1) + 2] << 16));
    }
    if (u0 + THREADS < units) load_x(u0 + THREADS + threadIdx.x);
    // 2^E of the maximum in [2^E, 2^(E + 1)); below 2^-111 the values are first brought up by 2^64
    uint32_t ex = top >> 23;
    float power = __uint_as_float(min(ex, 254u) << 23);
    if (ex < 16u) {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = __fmul2_rn(v[j], make_float2(18446744073709551616.f, 18446744073709551616.f));
      ex = max(__float_as_uint(__uint_as_float(top) * 18446744073709551616.f) >> 23, 16u);
      power = __uint_as_float(ex << 23) * 5.421010862427522e-20f;
    }
    const float up = __uint_as_float((269u - min(ex, 254u)) << 23);  // 2^(15 - E)
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      v[j] = __fmul2_rn(v[j], make_float2(up, up));
      if constexpr (PIECES == 1) sum = __fadd2_rn(sum, v[j]);
      if (j & 1) v[j] = __fmul2_rn(v[j], make_float2(0.0625f, 0.0625f));  // (the codes of these places are 16 times theirs)
    }
    float s = sum.x + sum.y;
    if constexpr (PIECES == 1) {
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
    }
    uint8_t* to = xs + i * p.x_pitch + (e >> 3) * 256 + (e & 1) * 128 + ((e >> 1) & 3) * 16;
#pragma unroll
    for (int c = 0; c < PIECES; c++) {
      uint32_t o[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (c + 1 < PIECES) {  // the leading bits toward zero (2^16 is never reached), and what is left (below 2^5) times 2^10
          asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(o[j]) : "f"(v[j].y), "f"(v[j].x));
          const float2 f = unpack_f16x2(o[j]);
          v[j] = __fmul2_rn(__fadd2_rn(v[j], make_float2(-f.x, -f.y)), make_float2(1024.f, 1024.f));
        } else {
          o[j] = as_u32(__floats2half2_rn(v[j].x, v[j].y));
        }
      }
      if (mine) {
        uint4* piece = reinterpret_cast<uint4*>(to + c * m * p.x_pitch);
        piece[0] = make_uint4(o[0], o[1], o[2], o[3]);
        piece[4] = make_uint4(o[4], o[5], o[6], o[7]);
        if ((e & 3) == 0) {  // group (e / 4) % 2 of chunk e / 8; an infinity or NaN makes its row NaN
          float* at = reinterpret_cast<float*>(base + (e >> 3) * TOKS + i + c * m) + ((e >> 2) & 1);
          at[0] = ex == 255u ? __uint_as_float(0x7fc00000u) : PIECES == 1 ? s * -4.76837158203125e-07f : 0.f;  // -8 2^-24
          at[2] = power * (c ? 9.765625e-4f : 1.f);
        }
      }
    }
  }
  if (toks < TOKS)  // places without a token
    for (int u = threadIdx.x; u < chunks * (TOKS - toks); u += THREADS)
      base[u / (TOKS - toks) * TOKS + toks + u % (TOKS - toks)] = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncthreads();

  float acc[RT][NT][2];  // channels lane / 4 and + 8 of a row tile, token piece 4 nt + lane % 4
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int t = 0; t < NT; t++) acc[r][t][0] = acc[r][t][1] = 0.f;
  // This lane's column holds a token only where its values belong to the column's group; other lanes read zeros.
  const uint8_t* bp[NT];
  int b_step[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int tok = t * 4 + (lane >> 3);
    const bool some = ((lane >> 2) & 1) == ((lane >> 1) & 1) && tok < toks;
    bp[t] = some ? xs + tok * p.x_pitch + ch0 * 256 + (lane & 3) * 16 : smem + 64;
    b_step[t] = some ? AHEAD * STEP * 256 : 0;
  }
  const float4* sp4 = base + ch0 * TOKS + (lane & 3);
  // the masks in registers, so that a code pair is one operation with its other constant
  uint32_t low = 0x000f000fu, high = 0x00f000f0u;
  asm volatile("" : "+r"(low), "+r"(high));

  const bool far = (lane & 4) != 0;
  static_assert(AHEAD * STEP == 4, "a lane's scales are of every fourth chunk");
  for (int c0 = ch0; c0 < end; c0 += AHEAD * STEP) {
#pragma unroll
    for (int r = 0; r < RT; r++) sc[r][0] = sc_next[r][0], sc[r][1] = sc_next[r][1];
    fetch_scales(c0 + AHEAD * STEP);
#pragma unroll
    for (int ah = 0; ah < AHEAD; ah++) {
      if (c0 + ah * STEP >= end) break;
      uint4 wq[STEP][2 * RT];
#pragma unroll
      for (int r = 0; r < RT; r++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {  // lane l has a channel's first chunk, lane l + 4 its second, and of the channel 4 on too
          const uint4 &one = raw[ah][r][2 * h], &two = raw[ah][r][2 * h + 1];
          uint4 x = far ? one : two;
          x.x = __shfl_xor_sync(0xffffffffu, x.x, 4);
          x.y = __shfl_xor_sync(0xffffffffu, x.y, 4);
          x.z = __shfl_xor_sync(0xffffffffu, x.z, 4);
          x.w = __shfl_xor_sync(0xffffffffu, x.w, 4);
          wq[0][2 * r + h] = far ? x : one;
          wq[1][2 * r + h] = far ? two : x;
        }
        fetch(ah, r, c0 + (ah + AHEAD) * STEP);
      }
#pragma unroll
      for (int st = 0; st < STEP; st++) {
        const int ch = ah * STEP + st;
        if (c0 + ch >= end) break;
        float d[RT][NT][4], e[RT][CHAINS == 2 ? NT : 1][4];  // one or two chains of products
        float2 power[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
          const float4 s = sp4[ch * TOKS + t * 4];
          power[t] = make_float2(s.z, s.w);
#pragma unroll
          for (int r = 0; r < RT; r++) {
            d[r][t][0] = d[r][t][2] = s.x;
            d[r][t][1] = d[r][t][3] = s.y;
            if constexpr (CHAINS == 2) e[r][t][0] = e[r][t][1] = e[r][t][2] = e[r][t][3] = 0.f;
          }
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
          uint4 b[NT];
#pragma unroll
          for (int t = 0; t < NT; t++) b[t] = *reinterpret_cast<const uint4*>(bp[t] + ch * 256 + q * 64);
#pragma unroll
          for (int r = 0; r < RT; r++) {
            const uint4 &l4 = wq[st][2 * r], &h4 = wq[st][2 * r + 1];
            const uint32_t lo = q == 0 ? l4.x : q == 1 ? l4.y : q == 2 ? l4.z : l4.w, lo8 = lo >> 8;
            const uint32_t hi = q == 0 ? h4.x : q == 1 ? h4.y : q == 2 ? h4.z : h4.w, hi8 = hi >> 8;
            const uint32_t a0[4] = {code_pair<PIECES>(lo, low, 0), code_pair<PIECES>(hi, low, 0),
                                    code_pair<PIECES>(lo, high, 1), code_pair<PIECES>(hi, high, 1)};
            const uint32_t a1[4] = {code_pair<PIECES>(lo8, low, 0), code_pair<PIECES>(hi8, low, 0),
                                    code_pair<PIECES>(lo8, high, 1), code_pair<PIECES>(hi8, high, 1)};
#pragma unroll
            for (int t = 0; t < NT; t++) {
              mma_f16(d[r][t], a0, b[t].x, b[t].y);
              mma_f16(CHAINS == 2 ? e[r][t] : d[r][t], a1, b[t].z, b[t].w);
            }
          }
        }
#pragma unroll
        for (int r = 0; r < RT; r++) {
          // with (2^24) 2^-15; the powers come last, in the addition, so that sums of tiny values are rounded once
          constexpr float F = PIECES == 1 ? 512.f : 3.0517578125e-5f;
          const int holder = (lane & ~3) | ch;
          const float2 s0 = __fmul2_rn(unpack_f16x2(__shfl_sync(0xffffffffu, sc[r][0], holder)), make_float2(F, F));
          const float2 s1 = __fmul2_rn(unpack_f16x2(__shfl_sync(0xffffffffu, sc[r][1], holder)), make_float2(F, F));
#pragma unroll
          for (int t = 0; t < NT; t++) {
            float(&u)[4] = d[r][t];
            if constexpr (CHAINS == 2) u[0] += e[r][t][0], u[1] += e[r][t][1], u[2] += e[r][t][2], u[3] += e[r][t][3];
            acc[r][t][0] = fmaf(u[1] * s0.y, power[t].y, fmaf(u[0] * s0.x, power[t].x, acc[r][t][0]));
            acc[r][t][1] = fmaf(u[3] * s1.y, power[t].y, fmaf(u[2] * s1.x, power[t].x, acc[r][t][1]));
          }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < NT; t++) bp[t] += b_step[t];
    sp4 += AHEAD * STEP * TOKS;
  }

  // The sums over this CTA's part of k: the warps' parts in turn, a token's pieces.
#pragma unroll
  for (int r = 0; r < RT; r++)
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int at = (warp * ROWS + r * 16 + channel) * TOKS + t * 4 + (lane & 3);
      red[at] = acc[r][t][0];
      red[at + 8 * TOKS] = acc[r][t][1];
    }
  __syncthreads();
  const int outs = cta_rows * m;
  const int row_shift = 31 - __clz(cta_rows), blocks = ((outs + THREADS - 1) / THREADS + p.cluster - 1) / p.cluster;
  if (p.cluster > 1) tc::cluster_wait();  // every CTA of the cluster has begun
  int owner = 0, slot = rank * blocks;  // the CTA that adds the cluster's parts of a block of outputs, and where it holds ours
  for (int u = threadIdx.x; u < outs; u += THREADS) {
    const int i = u >> row_shift, row = u - (i << row_shift);
    const float* from = red + (row / ROWS * p.wk * ROWS + row % ROWS) * TOKS + i;
    float v = 0.f;
#pragma unroll
    for (int c = PIECES - 1; c >= 0; c--)
#pragma unroll
      for (int k = 0; k < WARPS; k++)
        if (k < p.wk) v += from[k * (ROWS * TOKS) + c * m];
    if (p.cluster > 1) {
      tc::st_cluster_f32(tc::map_rank(tc::smem_u32(part + slot * THREADS + threadIdx.x), owner), v);
      if (++owner == p.cluster) owner = 0, slot++;
    } else if (first + row < n) {
      matvec_store(v, a, i, first + row, y);
    }
  }
  if (p.cluster > 1) {  // the cluster's parts in rank order
    __syncwarp();
    tc::cluster_sync_all();
    for (int b = 0; b < blocks; b++) {
      const int u = (b * p.cluster + rank) * THREADS + threadIdx.x, i = u >> row_shift, at = first + u - (i << row_shift);
      if (u >= outs || at >= n) continue;
      float v = 0.f;
#pragma unroll
      for (int s = 0; s < MAX_CLUSTER; s++)
        if (s < p.cluster) v += part[(s * blocks + b) * THREADS + threadIdx.x];
      matvec_store(v, a, i, at, y);
    }
  }
}

template <int XT, int NT, int RT, int WARPS>
static cudaError_t matvec_mma(const void* x, const uint8_t* w, void* y, const MatmulArgs& a, const mv::Plan& p, int groups_y,
                              cudaStream_t st) {
  auto kern = matvec_mma_kernel<XT, NT, RT, WARPS>;
  const cudaError_t e = allow_smem(kern, p.smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.cluster, (unsigned)groups_y);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = (size_t)p.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  pdl_attribute(attr[0]);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, x, w, y, a, p);
}

cudaError_t launch_matvec(const void* x, const void* wv, void* y, const MatmulArgs& a, int sms, cudaStream_t st) {
  using namespace mv;
  const uint8_t* w = static_cast<const uint8_t*>(wv);
  const bool f32 = a.x_dtype == WE_F32;
  const int toks = (int)a.m * (f32 ? 2 : 1);
  const int nt = toks <= 4 ? 1 : (toks <= 8 ? 2 : (toks <= 16 ? 4 : 8));
  const int WARPS = nt == 8 ? 8 : 16, THREADS = WARPS * 32;  // the instances below
  const int chunks = (int)((a.k + CHUNK - 1) / CHUNK), tiles = (int)((a.n + 15) / 16);
  // How k is split over clusters and warps: the shortest chain of a warp (its share of x's layout, its steps, its sums and
  // the cluster's, for as many waves of CTAs as it takes), in weights fitted to the timed splits.
  // ROOM: CTAs that 148 SMs hold at a time in clusters of 1 to 8, one CTA an SM (cudaOccupancyMaxActiveClusters; a cluster
  // stays within a GPC). All splits of 21 shapes were timed: this picks the fastest of 20 and one 7% slower of the other. 8
  // tokens of 16384 values to 6144 channels take 22.9 us with clusters of 5 and 26.4 with the best power of two.
  static constexpr int ROOM[MAX_CLUSTER] = {148, 148, 135, 132, 130, 132, 105, 120};
  Plan p{};
  int64_t best = -1;
  const int warps_shift = nt == 8 ? 3 : 4, threads_shift = warps_shift + 5, m = (int)a.m;
  for (int cluster = 1; cluster <= MAX_CLUSTER; cluster++) {
    const int per_cta = (chunks + cluster - 1) / cluster, slots = std::max(1, sms * ROOM[cluster - 1] / 148);
    const int64_t x_bytes = (int64_t)toks * per_cta * (CHUNK * 2) + (int64_t)per_cta * (nt * 64);
    if (x_bytes > 226 * 1024) continue;
    const int units = (m * per_cta * 8 + THREADS - 1) >> threads_shift;
    for (int split = 0; split <= warps_shift; split++) {  // log2 of the warps that split k
      const int wk = 1 << split;
      if (wk > 1 && wk > per_cta) break;
      const int rows = 16 << (warps_shift - split), outs = (rows * m + THREADS - 1) >> threads_shift;
      const int64_t ctas = (((int64_t)tiles << split) + WARPS - 1 >> warps_shift) * cluster, waves = (ctas + slots - 1) / slots;
      const int64_t bytes = NOTHING + x_bytes + WARPS * 16 * nt * 16 +
                            (cluster > 1 ? (outs + cluster - 1) / cluster * cluster * THREADS * 4 : 0);
      if (bytes > 226 * 1024) continue;
      const int64_t cost = waves * (units * (f32 ? 500 : 400) + ((per_cta + wk - 1) >> split) * (70 + 20 * nt) +
                                    outs * (60 + 2 * wk) + (cluster > 1 ? 100 : 0));
      if (best >= 0 && cost > best) continue;
      best = cost;
      p = Plan{wk, cluster, per_cta, per_cta * CHUNK * 2, (int)bytes};
    }
  }
  const bool ok = best >= 0;
  const int64_t cta_rows = ok ? WARPS / p.wk * 16 : 1, gy = (a.n + cta_rows - 1) / cta_rows;
  if (!ok || gy > 65535) {
    const dim3 grid((unsigned)((a.n + 7) / 8));
    const cudaError_t e = f32 ? launch_pdl(matvec_long_kernel<WE_F32>, grid, 256, 0, st, x, w, y, a)
                              : launch_pdl(matvec_long_kernel<WE_BF16>, grid, 256, 0, st, x, w, y, a);
    return e == cudaSuccess ? cudaGetLastError() : e;
  }
  const int ny = (int)gy;
  cudaError_t e;
  if (f32) {
    e = nt == 1   ? matvec_mma<WE_F32, 1, 1, 16>(x, w, y, a, p, ny, st)
        : nt == 2 ? matvec_mma<WE_F32, 2, 1, 16>(x, w, y, a, p, ny, st)
        : nt == 4 ? matvec_mma<WE_F32, 4, 1, 16>(x, w, y, a, p, ny, st)
                  : matvec_mma<WE_F32, 8, 1, 8>(x, w, y, a, p, ny, st);
  } else {
    e = nt == 1   ? matvec_mma<WE_BF16, 1, 1, 16>(x, w, y, a, p, ny, st)
        : nt == 2 ? matvec_mma<WE_BF16, 2, 1, 16>(x, w, y, a, p, ny, st)
                  : matvec_mma<WE_BF16, 4, 1, 16>(x, w, y, a, p, ny, st);
  }
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace we
