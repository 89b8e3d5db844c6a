// A paged 4-bit K/V cache (we_kv4_cache): rows in, rows out, and the attention of a step's new tokens over it.
#include <algorithm>

#include "attn_merge.cuh"
#include "common.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace we {

// Row index (in rows of `dim` values) of token t of sequence b at kv head 0, or -1 when the page table does not hold it
// (recorded in the device error word). Head h's row is h * page further.
__device__ __forceinline__ int64_t kv4_row(const we_kv4_cache& c, int64_t b, int64_t t, uint32_t* err) {
  const uint32_t page = (uint32_t)c.page, slot = (uint32_t)t / page;  // (a page of the table and t are below 2^32)
  if (slot >= c.max_pages) {
    atomicCAS(err, 0u, (uint32_t)DEV_ERR_KV_FULL);
    return -1;
  }
  const int64_t id = c.page_table[b * c.max_pages + slot];
  if (id < 0 || id >= c.pages) {
    atomicCAS(err, 0u, (uint32_t)DEV_ERR_KV_PAGE);
    return -1;
  }
  return id * c.kv_heads * c.page + ((uint32_t)t - slot * page);
}

// Rows in and out of the cache. A thread moves 8 values of k or of v a step: 16 bytes (bf16) or 32 on the wide side, a 4-byte
// word on the packed one, 8 neighbouring lanes a group. It keeps its place within a token (side, head, values) and steps
// over the tokens of its CTA, whose rows are looked up once, so that a step has little to compute but the values.
// Measured: 2 x 4099 tokens x 12 heads of 128 in bf16 in 23 us and back in 17 (the bytes of each are 10 us), 16 tokens both
// ways 4.7 us in a recorded graph (5.9 as two calls from Python); a warp per group and a look-up per value took 167 us.
constexpr int ROW_THREADS = 256, ROW_SPAN = 32;
struct RowShape {
  int units;       // of 8 values in a token: k's, then v's
  int head_shift;  // log2 of a head's
  int lanes;       // threads on one token (at most ROW_THREADS), a multiple of 8
  int along;       // tokens side by side in a CTA
  int span;        // tokens of a CTA, at most ROW_SPAN
};

// The rows of `here` tokens from t0 of all sequences' (from start[b], or the sequence's length, on), as the index of their
// first word of codes at kv head 0, -1 where there is none.
__device__ __forceinline__ void find_rows(const we_kv4_cache& c, int64_t* rows, int64_t t0, uint32_t here, int64_t tokens,
                                          const int32_t* start, int head_shift, uint32_t* err) {
  if (threadIdx.x >= here) return;
  const int64_t i = t0 + threadIdx.x, b = i >> 32 ? i / tokens : (uint32_t)i / (uint32_t)tokens;
  const int64_t have = c.lengths[b], from = start ? (int64_t)start[b] : have;
  const int64_t row = have < 0 || from < 0 ? -1 : kv4_row(c, b, from + (i - b * tokens), err);
  rows[threadIdx.x] = row < 0 ? row : row << head_shift;
}

__device__ __forceinline__ float rcp_approx(float x) {  // to 1 ulp
  float d;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // keeps a NaN
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The codes of 8 values, 8 lanes to a group of 64, and the group's scale: s = f16(max|x| / 7), q = rint(x / s) in -8..7.
// The first division is by a constant: q + (a - 7 q) / 7 with q = a / 7 to a rounding is the rounded quotient (Markstein).
// For the second, x (1 / s) added to 1.5 2^23 is rounded to an integer q, the quotient's own rounding unless |x - q s| is
// within 2e-6 s of s / 2 (1 / s is to 2^-23, the quotient to 2^-24). Halves are common where few-bit values meet (one in 650
// bf16 values): where x - q s is exactly s / 2, q goes to the even side. What is left takes the division (f32 values close
// to a half), as do values that need the clamp: infinities, and groups whose s is not a normal f16 (in all others
// |x / s| <= 7.01). A NaN makes its group's scale NaN. The q + 8 of four values add up to 16 bits in f32.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], uint16_t* scale) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j += 2) top = max3_nan(top, fabsf(x[j]), fabsf(x[j + 1]));
#pragma unroll
  for (int o = 4; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  constexpr float SEVENTH = 1.f / 7.f, MAGIC = 12582912.f, MOST = 7.f * 65504.f;
  const float held = min_nan(top, MOST), near = held * SEVENTH;
  const __half s16 = __float2half_rn(fmaf(fmaf(-7.f, near, held), SEVENTH, near));
  const float s = __half2float(s16), inv = rcp_approx(s);
  *scale = __half_as_ushort(s16);
  const float2 inv2 = make_float2(inv, inv), magic2 = make_float2(MAGIC, MAGIC), back2 = make_float2(-MAGIC, -MAGIC),
               less2 = make_float2(-s, -s);
  float far = 0.f;
  float2 sum[2];  // of values 0..3 and 4..7, the even and the odd ones apart
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float2 v = make_float2(x[2 * j], x[2 * j + 1]);
    const float2 q = __fadd2_rn(__ffma2_rn(v, inv2, magic2), back2);
    const float2 e = __ffma2_rn(q, less2, v);
    far = max3_nan(far, fabsf(e.x), fabsf(e.y));
    const float w = j & 1 ? 256.f : 1.f;  // 8 (1 + 16 + 256 + 4096) = 34952
    sum[j / 2] = __ffma2_rn(q, make_float2(w, 16.f * w), j & 1 ? sum[j / 2] : make_float2(34952.f + 8388608.f, 0.f));
  }
  uint32_t word = __byte_perm(__float_as_uint(sum[0].x + sum[0].y), __float_as_uint(sum[1].x + sum[1].y), 0x5410);
  if (!(far <= 0.499998f * s && s >= 6.104e-5f && top <= MOST)) {
    if (!(s > 0.f)) return 0;  // (0 or NaN)
    bool rest = !(far <= s && s >= 6.104e-5f && top <= MOST);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float r = fmaf(x[j], inv, MAGIC), e = fmaf(__fadd_rn(r, -MAGIC), -s, x[j]), twice = 2.f * fabsf(e);
      const uint32_t odd = (__float_as_uint(r) & 1u) << (4 * j);
      if (twice == s) word += e < 0.f ? 0u - odd : odd;
      else rest |= twice >= 0.999996f * s;
    }
    if (rest) {
      word = 0x88888888u;
#pragma unroll 1
      for (int j = 0; j < 8; j++) {
        float one = x[0];
#pragma unroll
        for (int e = 1; e < 8; e++) one = j == e ? x[e] : one;
        word += (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(one, s)), -8.f), 7.f) << (4 * j);
      }
    }
  }
  return word ^ 0x88888888u;
}

// PER_SM: CTAs an SM at the least: 6 (in 40 registers) where there are more than two for each SM, 1 (in 56) otherwise. Prompts
// of 2 x 4099 tokens both ways 40.0 us against 43.6, 16 tokens 4.9 against 4.7.
template <int DT, bool WIDE, int PER_SM>
__global__ void __launch_bounds__(ROW_THREADS, PER_SM) kv4_append_kernel(const we_kv4_cache c, const void* __restrict__ k,
                                                                 const void* __restrict__ v, int64_t tokens, int64_t stride,
                                                                 const RowShape z, uint32_t* err) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ int64_t rows[ROW_SPAN];
  const int64_t all = c.batch * tokens;
  const uint32_t slot = threadIdx.x / z.lanes, unit = threadIdx.x - slot * z.lanes;
  for (int64_t t0 = (int64_t)blockIdx.x * z.span; t0 < all; t0 += (int64_t)gridDim.x * z.span) {
    const uint32_t here = (uint32_t)(all - t0 < z.span ? all - t0 : z.span);
    bool found = false;
    for (uint32_t a = blockIdx.y * z.lanes + unit; a - unit < (uint32_t)z.units; a += gridDim.y * z.lanes) {
      const bool mine = a < (uint32_t)z.units && slot < (uint32_t)z.along, is_v = a >= (uint32_t)z.units / 2;
      const uint32_t at = is_v ? a - z.units / 2 : a, h = at >> z.head_shift, e = at - (h << z.head_shift);
      const void* src = is_v ? v : k;
      const int64_t head = ((int64_t)h * c.page << z.head_shift) + e;
      uint32_t* codes = reinterpret_cast<uint32_t*>(is_v ? c.v : c.k) + head;
      uint16_t* scales = (is_v ? c.v_scale : c.k_scale) + head / 8;
      float x[8] = {};
      auto load = [&](uint32_t t) {
        if (!mine || t >= here) return;
        const int64_t from = (t0 + t) * stride + (int64_t)at * 8;
        if constexpr (WIDE) {
          load8<DT>(src, from, x);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) x[j] = load_act<DT>(src, from + j);
        }
      };
      load(slot);  // (on its way during the look-up)
      if (!found) {
        __syncthreads();  // (rows of the tokens before are read)
        find_rows(c, rows, t0, here, tokens, nullptr, z.head_shift, err);
        __syncthreads();
        found = true;
      }
      for (uint32_t t = slot; t - slot < here; t += z.along) {  // (all lanes together: the groups' maxima are shuffled)
        uint16_t scale;
        const uint32_t word = kv4_codes(x, &scale);
        load(t + z.along);
        const int64_t row = mine && t < here ? rows[t] : -1;
        if (row >= 0) {
          codes[row] = word;
          if (e % 8 == 0) scales[(uint64_t)row / 8] = scale;
        }
      }
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(ROW_THREADS) kv4_unpack_kernel(const we_kv4_cache c, void* __restrict__ k,
                                                                 void* __restrict__ v, int64_t tokens,
                                                                 const int32_t* __restrict__ start, const RowShape z,
                                                                 uint32_t* err) {
  pdl_wait();
  pdl_launch_dependents();
  __shared__ int64_t rows[ROW_SPAN];
  const int64_t all = c.batch * tokens;
  const uint32_t slot = threadIdx.x / z.lanes, unit = threadIdx.x - slot * z.lanes;
  for (int64_t t0 = (int64_t)blockIdx.x * z.span; t0 < all; t0 += (int64_t)gridDim.x * z.span) {
    const uint32_t here = (uint32_t)(all - t0 < z.span ? all - t0 : z.span);
    __syncthreads();
    find_rows(c, rows, t0, here, tokens, start, z.head_shift, err);
    __syncthreads();
    for (uint32_t a = blockIdx.y * z.lanes + unit; a < (uint32_t)z.units; a += gridDim.y * z.lanes) {
      const bool is_v = a >= (uint32_t)z.units / 2;
      const uint32_t at = is_v ? a - z.units / 2 : a, h = at >> z.head_shift, e = at - (h << z.head_shift);
      void* out = is_v ? v : k;
      if (!out || slot >= (uint32_t)z.along) continue;
      const int64_t head = ((int64_t)h * c.page << z.head_shift) + e, to = t0 * z.units / 2 + at;
      const uint32_t* codes = reinterpret_cast<const uint32_t*>(is_v ? c.v : c.k) + head;
      const uint16_t* scales = (is_v ? c.v_scale : c.k_scale) + head / 8;
#pragma unroll 4
      for (uint32_t t = slot; t < here; t += z.along) {
        const int64_t row = rows[t];
        uint32_t word = 0x88888888u;
        float s = 0.f;
        if (row >= 0) {
          word = codes[row] ^ 0x88888888u;
          s = __half2float(__ushort_as_half(scales[(uint64_t)row / 8]));
        }
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {  // q + 8 as the low bits of 2^23
          const float2 u = make_float2(__uint_as_float(0x4b000000u | ((word >> (4 * j)) & 15u)),
                                       __uint_as_float(0x4b000000u | ((word >> (4 * j + 4)) & 15u)));
          const float2 y = __fmul2_rn(__fadd2_rn(u, make_float2(-8388616.f, -8388616.f)), make_float2(s, s));
          x[j] = y.x;
          x[j + 1] = y.y;
        }
        store8<DT>(out, (to + (int64_t)t * (z.units / 2)) * 8, x);
      }
    }
  }
}

__global__ void kv4_advance_kernel(int32_t* lengths, int64_t batch, int32_t tokens) {
  pdl_wait();
  pdl_launch_dependents();
  for (int64_t b = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; b < batch; b += (int64_t)gridDim.x * blockDim.x)
    if (lengths[b] >= 0) lengths[b] = (int32_t)min((int64_t)lengths[b] + tokens, (int64_t)0x7fffffff);  // (never to idle)
}

// ---------------- attention ----------------
// Per (sequence, kv head): q rows (the new tokens times the heads of the group) over that head's keys. The cache is read
// once for every 8 or 16 rows (dim / 2 + dim / 32 bytes per key, for k and for v); the products run on 16 x 8 x 16 tensor
// tiles with KEYS (for v: dims) as the 16 rows and up to 8 q rows as the columns, so a tile has no more idle rows than
// the group leaves of 8, and the codes go from the registers they are unpacked in straight into the tile:
// - S^T = K Q^T. A lane holds 16 codes of 2 keys; a pair of codes becomes the f16 subnormals u 2^-24, u = q + 8, by one
//   logical operation (and u 2^-20 for the next nibble, whose q is divided by 16); the sum of a group of 64 starts at
//   -8 sum(q). The key's scale multiplies the group's sum in f32. A row of q is held over the power of two of its largest
//   value; what is below 2^-36 of that is lost.
// - O^T = V^T P^T. Two keys' words are interleaved by byte permutations, so that a pair is the same dim of two keys; p
//   times the key's scale of v, times a power of two that keeps it in f16's range (2^15 at most), is the other operand,
//   turned by movmatrix from S^T's layout. The offset 8 is taken out at the end with the sum of those weights, which one
//   more tile of ones accumulates.
// - f32 q or out (TERMS = 2): q and the weights are two f16 terms each (22 bits), and codes become signed f16 by one more
//   operation, because the offset's sums would cost 2 bits of a score and, weights being positive, up to 5 of an output.
// - A warp takes 16 or 32 keys at a time through a ring of its own (cp.async), with its own running maximum; the O and
//   sums are only rescaled when the maximum grows by more than 2^8 or v's scales outgrow their power of two. Values of v of
//   very different magnitudes take a second sweep with powers for each row and group (sweep()).
// - A cluster of 8 CTAs shares the keys of a sequence evenly and merges over distributed shared memory; a longer sequence
//   takes several clusters, whose parts the last one to finish merges. Every merge is in a fixed order.
namespace kv {
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int CLUSTER = 8;    // CTAs that share a run of keys and merge over distributed shared memory
// Steps in a warp's ring (a power of two): 35 KB a CTA, so that registers say how many an SM holds. With two steps whatever
// their size, 5 tokens over 3333 keys of 64 in f32, out of memory, took 14.0 us instead of 12.0.
template <int D, int KT>
constexpr int ring_depth() {
  return 512 / (KT * D);
}

struct Params {
  we_kv4_cache c;
  const void* q;
  void* out;
  int tokens, heads, group, rows;  // group: heads per kv head; rows = tokens * group
  int row_tiles;                   // tiles of 8 NQ rows
  int chunk;                       // keys per CTA at most
  int wide_q;                      // rows of q are 16-byte aligned
  int64_t q_stride, out_stride;
  float scale_log2;                // |scale| log2(e); its sign goes to q, so that maxima and hidden scores of -inf hold
  int negative;
  int dtype, out_dtype;
  float* part;                     // [sequence, kv head, row tile][clusters][8 NQ](dim values, maximum, sum), when more than one
  uint32_t* done;                  // [sequence, kv head, row tile]: clusters that have written, zero between calls
  uint32_t* err;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a b + c
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t and_xor(uint32_t v, uint32_t mask, uint32_t flip) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(v), "r"(mask), "r"(flip));
  return r;
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {  // of an 8 x 8 f16 tile
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ float2 halves(uint32_t u) { return __half22float2(as_half2(u)); }

// 2^(11 - e) (one term; the weights are held times 2^6) or 2^(17 - e) (two) from (31 - e) << 10
__device__ __forceinline__ float power_up(uint32_t power, int terms) {
  return __uint_as_float((power << 13) + ((terms == 1 ? 107u : 113u) << 23));
}
__device__ __forceinline__ float power_down(uint32_t power, int terms) {  // 1 over it
  return __uint_as_float(((terms == 1 ? 147u : 141u) << 23) - (power << 13));
}

// Where the 32 bytes of group g of row `row` (0..15) of a tile lie: so that the rows that lanes read together
// ({0 4 1 5}, {2 6 3 7} for k, {0 1 2 3}, {4 5 6 7} for v, and 8 more) are on different banks.
template <int D>
__device__ __forceinline__ int segment(int row, int g) {
  const int h = (row & 1) | ((((row >> 1) ^ (row >> 2)) & 1) << 1);
  if (D == 64) return ((row >> 2) * 4 + h) * 32;
  if (D == 128) return ((row >> 1) * 4 + (row & 1) * 2 + (g ^ (h >> 1))) * 32;
  return (row * 4 + (g ^ h)) * 32;
}
// This lane's values of q: 16 of each group of the rows nq * 8 + lane / 4 of its tile.
template <int D, int NQ>
__device__ __forceinline__ void load_q(const Params& p, int b, int head, int rtile, uint4 (&q_raw)[NQ][D / 64][4]) {
  constexpr int G = D / 64, QROWS = 8 * NQ;
  const int c = threadIdx.x & 3, u = (threadIdx.x >> 2) & 7;
#pragma unroll
  for (int nq = 0; nq < NQ; nq++) {
    const int r = rtile * QROWS + nq * 8 + u;
    const int64_t row = ((int64_t)b * p.tokens + r / p.group) * p.q_stride + (int64_t)(head * p.group + r % p.group) * D + c * 16;
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        q_raw[nq][g][j] = make_uint4(0, 0, 0, 0);
        if (r >= p.rows || (p.dtype == WE_BF16 && j >= 2)) continue;
        const int64_t at = row + g * 64 + j * (p.dtype == WE_F32 ? 4 : 8);
        uint32_t w[4];
        if (p.wide_q) {
          const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.q) + at * (p.dtype == WE_F32 ? 4 : 2));
          w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if (p.dtype == WE_F32) w[e] = static_cast<const uint32_t*>(p.q)[at + e];
            else w[e] = static_cast<const uint16_t*>(p.q)[at + 2 * e] | (uint32_t) static_cast<const uint16_t*>(p.q)[at + 2 * e + 1] << 16;
          }
        }
        q_raw[nq][g][j] = make_uint4(w[0], w[1], w[2], w[3]);
      }
  }
}

// What a warp's keys give its tile of q rows.
template <int D, int NQ>
struct Part {
  float o[NQ][D / 16][4], w_sum[NQ][D / 64][4];  // O, and the sums of weights (times 8: the codes' offset) by groups
  float down[NQ][D / 64][2];                     // what O is to be multiplied by
  float m[NQ][2], l[NQ][2];
};

// One sweep over this warp's keys.
// EXACT false: the weights times scales of v, and O, are held over ONE power of two, that of the largest scale so far. With
// scales down to 2^-RANGE of that a row's largest product is at least 2^-5 (TERMS 2: 2^-2) and every other is within 2^-11 (2^-22)
// of itself or an absolute 2^-25. A smaller scale, or one that is not finite, ends the sweep (false), and the CTA begins again:
// EXACT: every row and group has a power of its own, by the largest product of a weight and a scale that it has met, so that a
// key of large values to which a row gives no weight takes no bits from the row's other keys (with one power for all, values
// 10^7 below such a key's came out as zeros, or with a few bits in f32).
// Choosing between the two step by step cost every call 5% (16 sequences of 3001 to 16384 keys, 48 heads on 12: 68.4 us against
// 65.0); the check of the range and the code beside it cost it nothing, a call of one short sequence 0.2 us of 6.2. Values
// that need the second sweep: 4 sequences of 16000 keys 28.6 -> 35.7 us, in f32 40.2 -> 47.3 (scales of zero cost a check each step,
// 30.8 and 43.2). (256-wide heads with more than 8 rows, which spilled before, lost 6%: 8 tokens of
// 32 heads on 8, 4 x 4000 keys, 62.7 us against 58.9.)
template <int D, int NQ, int KT, int TERMS, bool EXACT>
__device__ __forceinline__ bool sweep(const Params& p, int b, int head, int rtile, int have, int key0, int key1, uint8_t* smem,
                                      const uint4 (&q_raw)[NQ][D / 64][4], Part<D, NQ>& part) {
  constexpr int G = D / 64, STEP = KT * 16, ROW = D / 2, TILE = 16 * ROW, QROWS = 8 * NQ;
  constexpr int STAGE = KT * (2 * TILE + 2 * 16 * G * 2), DEPTH = ring_depth<D, KT>();
  constexpr int MTILES = D / 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3, u = lane >> 2;
  float(&o)[NQ][MTILES][4] = part.o;
  float(&w_sum)[NQ][G][4] = part.w_sum;
  float(&down)[NQ][G][2] = part.down;
  float(&m)[NQ][2] = part.m;
  float(&l)[NQ][2] = part.l;

  // this warp's steps: key0 + (warp + WARPS i) STEP
  const int steps = (key1 - key0 + STEP - 1) / STEP;
  const int mine = steps > warp ? (steps - warp + WARPS - 1) / WARPS : 0;
  uint8_t* ring = smem + warp * (DEPTH * STAGE);
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);

  // Where this warp's next 32 tiles of 16 keys lie, a lane each: index of the tile in the cache, or -1: not there.
  uint32_t at16 = 0xffffffffu;
  const int page = (int)p.c.page;
  auto load_ids = [&](int i) {  // from step i on
    const int tile = i * KT + lane, key = key0 + (warp + WARPS * (tile / KT)) * STEP + (tile % KT) * 16;
    at16 = 0xffffffffu;
    if (key < key1) {
      const int slot = key / page;
      const int id = p.c.page_table[(int64_t)b * p.c.max_pages + slot];
      if (id < 0 || id >= p.c.pages) atomicCAS(p.err, 0u, (uint32_t)DEV_ERR_KV_PAGE);
      else at16 = ((uint32_t)id * (uint32_t)p.c.kv_heads + head) * (uint32_t)(page / 16) + (key - slot * page) / 16;
    }
  };
  auto piece_to = [&](int j) {  // where a lane's j-th 16-byte piece of a tile goes
    const int at = j * 32 + lane, r = at / (ROW / 16), ch = at % (ROW / 16);  // piece `ch` of row r
    return segment<D>(r, ch >> 1) + (ch & 1) * 16;
  };
  uint32_t copy_to[D == 128 ? 1 : TILE / 512];  // (dim 128: 8 rows on is 512 bytes on)
#pragma unroll
  for (int j = 0; j < (D == 128 ? 1 : TILE / 512); j++) copy_to[j] = piece_to(j);
  uint32_t there = 0;  // bit per tile of the ring's stages: its page exists
  auto copy = [&](int i) {
    if (i < mine) {
      if ((i * KT) % 32 == 0) load_ids(i);
      const int stage = i & (DEPTH - 1);
      const uint32_t to = ring_addr + stage * STAGE;
#pragma unroll
      for (int t = 0; t < KT; t++) {
        const uint32_t at = __shfl_sync(0xffffffffu, at16, (i * KT + t) & 31);
        const uint32_t bit = 1u << (stage * KT + t);
        there &= ~bit;
        if (at == 0xffffffffu) continue;
        there |= bit;
#pragma unroll
        for (int side = 0; side < 2; side++) {
          const uint8_t* from = (side ? p.c.v : p.c.k) + (uint64_t)at * TILE + lane * 16;
#pragma unroll
          for (int j = 0; j < TILE / 512; j++) cp_async16(to + (t * 2 + side) * TILE + (D == 128 ? copy_to[0] + j * 512 : copy_to[j]), from + j * 512);
        }
        // scales: 4-byte words, 8 G of k then 8 G of v
#pragma unroll
        for (int j = 0; j < (16 * G + 31) / 32; j++) {
          const int word = j * 32 + lane, w = word % (8 * G);
          const uint16_t* from = (word / (8 * G) ? p.c.v_scale : p.c.k_scale) + (uint64_t)at * (16 * G) + w * 2;
          if (word < 16 * G)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + KT * 2 * TILE + t * (64 * G) + word * 4), "l"(from)
                         : "memory");
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < DEPTH - 1; i++) copy(i);

  // q as the B operand: column lane / 4 of tile nq is row nq * 8 + lane / 4; of a group's 8 words a lane holds words 2 c and
  // 2 c + 1 in the order of the codes: for word w and half h the pairs (q0, q4), (q1, q5) / 16 or (q2, q6), (q3, q7) / 16,
  // times a power of two that brings the row's largest to 2^15.
  uint32_t qf[NQ][G][4][2][TERMS];
  float q_start[NQ][G][4], q_back[NQ][2];  // of the columns of S^T that a lane holds: 2 c, 2 c + 1 (of two rows)
#pragma unroll
  for (int nq = 0; nq < NQ; nq++) {
    float x[G][16], top = 0.f;
#pragma unroll
    for (int g = 0; g < G; g++) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t w[4] = {q_raw[nq][g][j].x, q_raw[nq][g][j].y, q_raw[nq][g][j].z, q_raw[nq][g][j].w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (p.dtype == WE_F32) {
            x[g][4 * j + e] = __uint_as_float(w[e]);
          } else if (j < 2) {
            x[g][8 * j + 2 * e] = __uint_as_float(w[e] << 16);
            x[g][8 * j + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(x[g][e]));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t ex = min(max(__float_as_uint(top) >> 23, 16u), 254u);
    const float up = __uint_as_float((269u - ex) << 23 | (uint32_t)p.negative << 31);
    float sum[G];
#pragma unroll
    for (int g = 0; g < G; g++) {
      sum[g] = 0.f;
#pragma unroll
      for (int w = 0; w < 2; w++)
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const float down = k ? 0.0625f : 1.f;
            float lo = x[g][w * 8 + h * 2 + k] * up, hi = x[g][w * 8 + h * 2 + k + 4] * up;
            sum[g] += lo + hi;
#pragma unroll
            for (int t = 0; t < TERMS; t++) {
              // the first of two terms toward zero, so that 2^16 is never reached
              const __half2 v = t + 1 < TERMS ? __halves2half2(__float2half_rz(lo * down), __float2half_rz(hi * down))
                                              : __floats2half2_rn(lo * down, hi * down);
              qf[nq][g][w * 2 + h][k][t] = as_u32(v);
              const float2 f = __half22float2(v);
              lo -= f.x * (k ? 16.f : 1.f);
              hi -= f.y * (k ? 16.f : 1.f);
            }
          }
      sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
      sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
    }
    const float back = p.scale_log2 * (TERMS == 1 ? 512.f : 3.0517578125e-5f) * __uint_as_float(ex << 23);  // (2^24) 2^-15 2^E
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int from = (c * 2 + k) * 4;
      q_back[nq][k] = __shfl_sync(0xffffffffu, back, from);
#pragma unroll
      for (int g = 0; g < G; g++) q_start[nq][g][k] = q_start[nq][g][2 + k] = TERMS == 1 ? __shfl_sync(0xffffffffu, sum[g], from) * -4.76837158203125e-07f : 0.f;  // -8 2^-24
    }
  }

  uint32_t low = 0x000f000fu, high = 0x00f000f0u;  // in registers: a pair of codes is one operation with its other constant
  asm volatile("" : "+r"(low), "+r"(high));
  const __half2 sub1 = __float2half2_rn(-1032.f), sub16 = __float2half2_rn(-1152.f);
  const int full = have + (rtile * QROWS) / p.group + 1;  // keys below are seen by every row of the tile

  // offsets of this lane's pieces of a tile: for k words 2 c, 2 c + 1 of a group of its key and (+ 8 rows) the other; for v
  // word u of the keys of rows 2 c and (+ 8 rows) 2 c + 8, and of rows 2 c + 1 and 2 c + 9
  const int k0 = (u >> 1) + 4 * (u & 1);  // row r of a tile of S^T is key r / 2 + 4 (r & 1) (+ 8)
  int k_at[G], v_at[G], v_next = 0;
#pragma unroll
  for (int g = 0; g < G; g++) {
    k_at[g] = segment<D>(k0, g) + c * 8;
    v_at[g] = TILE + segment<D>(c, g) + u * 4;
  }
  if (D == 64) v_next = TILE + segment<D>(c + 4, 0) + u * 4;
  // row c + 4 (dim 128: as segment() puts it, the other group's place of row c and 256 bytes on)
  auto v_at_4 = [&](int g) { return D == 64 ? v_next : D == 128 ? v_at[g ^ 1] + 256 : TILE + segment<D>(c + 4, g) + u * 4; };
  const int s_at = KT * 2 * TILE + k0 * (2 * G);

  constexpr uint32_t RANGE = TERMS == 1 ? 10 : 7;
  // EXACT: scales of v are kept times 2^(11 - e) (TERMS 2: 2^(17 - e)), e a row's and group's power as an f16 exponent: for scales
  // up to 2^ABOVE above it and weights of up to 2^8 the products stay below 2^15.
  constexpr int ABOVE = 4;
  constexpr float UP = TERMS == 1 ? 6.f : 0.f;  // weights are kept times 2^UP
#pragma unroll
  for (int nq = 0; nq < NQ; nq++) {
#pragma unroll
    for (int t = 0; t < MTILES; t++) o[nq][t][0] = o[nq][t][1] = o[nq][t][2] = o[nq][t][3] = 0.f;
#pragma unroll
    for (int g = 0; g < G; g++) w_sum[nq][g][0] = w_sum[nq][g][1] = w_sum[nq][g][2] = w_sum[nq][g][3] = 0.f;
    m[nq][0] = m[nq][1] = NONE;
    l[nq][0] = l[nq][1] = 0.f;
  }
  // scales of v, as f16 bits, that need no change: up to the upper half (whose exponent field is O's power: that of the
  // largest scale so far, at least 1), and from the lower half on
  uint32_t v_range = 0x07ff0000u;
  // power[nq][g]: (31 - e) << 10 of this lane's two columns, e in 1..30.
  // limit: the scales of v, as f16 bits of two groups a word, up to which no power has to move
  uint32_t power[NQ][G], limit[(G + 1) / 2];
#pragma unroll
  for (int nq = 0; nq < NQ; nq++)
#pragma unroll
    for (int g = 0; g < G; g++) power[nq][g] = 0x78007800u;
#pragma unroll
  for (int g = 0; g < (G + 1) / 2; g++) limit[g] = 0x17ff17ffu;  // e = 1 + ABOVE
  for (int i = 0; i < mine; i++) {
    copy(i + DEPTH - 1);
    cp_async_wait<DEPTH - 1>();
    __syncwarp();
    const int stage = i & (DEPTH - 1);
    const uint8_t* st = ring + stage * STAGE;
    const int first = key0 + (warp + WARPS * i) * STEP;
    constexpr uint32_t TILES = (1u << KT) - 1u;
    const uint32_t here = (there >> (stage * KT)) & TILES;
    const bool whole = here == TILES && first + STEP <= min(full, key1);  // (uniform) every row sees every key
    float s[KT][NQ][4];  // S^T in the units of the products
    uint32_t vs[KT][2][(G + 1) / 2];  // scales of v of this lane's two keys
#pragma unroll
    for (int t = 0; t < KT; t++) {
      const uint8_t* kt = st + (t * 2) * TILE;
      float d[NQ][G][4];
#pragma unroll
      for (int g = 0; g < G; g++) {
        const uint2 a2 = *reinterpret_cast<const uint2*>(kt + k_at[g]);
        const uint2 b2 = *reinterpret_cast<const uint2*>(kt + k_at[g] + 8 * ROW);
#pragma unroll
        for (int x = 0; x < 4; x++) {  // word x / 2, half x % 2
          const uint32_t wa = (x < 2 ? a2.x : a2.y) >> ((x & 1) * 8), wb = (x < 2 ? b2.x : b2.y) >> ((x & 1) * 8);
          uint32_t av[4];
          if constexpr (TERMS == 1) {
            av[0] = and_xor(wa, low, 0x00080008u), av[1] = and_xor(wb, low, 0x00080008u);
            av[2] = and_xor(wa, high, 0x00800080u), av[3] = and_xor(wb, high, 0x00800080u);
          } else {  // 1024 + u - 1032 = q, 1024 + 16 u - 1152 = 16 q
            av[0] = as_u32(__hadd2(as_half2(and_xor(wa, low, 0x64086408u)), sub1));
            av[1] = as_u32(__hadd2(as_half2(and_xor(wb, low, 0x64086408u)), sub1));
            av[2] = as_u32(__hadd2(as_half2(and_xor(wa, high, 0x64806480u)), sub16));
            av[3] = as_u32(__hadd2(as_half2(and_xor(wb, high, 0x64806480u)), sub16));
          }
#pragma unroll
          for (int nq = 0; nq < NQ; nq++)
#pragma unroll
            for (int k = 0; k < TERMS; k++) {
              if (x == 0 && k == 0) mma_f16(d[nq][g], av, qf[nq][g][x][0][k], qf[nq][g][x][1][k], q_start[nq][g]);
              else mma_f16(d[nq][g], av, qf[nq][g][x][0][k], qf[nq][g][x][1][k]);
            }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint8_t* kat = st + s_at + t * (64 * G) + h * (16 * G);
        float ks[G];
        if constexpr (G == 1) {
          ks[0] = __half2float(__ushort_as_half(*reinterpret_cast<const uint16_t*>(kat)));
          vs[t][h][0] = *reinterpret_cast<const uint16_t*>(kat + 32);
        } else {
#pragma unroll
          for (int g = 0; g < G; g += 2) {
            const float2 f = halves(*reinterpret_cast<const uint32_t*>(kat + g * 2));
            ks[g] = f.x;
            ks[g + 1] = f.y;
            vs[t][h][g / 2] = *reinterpret_cast<const uint32_t*>(kat + 32 * G + g * 2);
          }
        }
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
          for (int k = 0; k < 2; k++) {
            float x = d[nq][0][h * 2 + k] * ks[0];
#pragma unroll
            for (int g = 1; g < G; g++) x = fmaf(d[nq][g][h * 2 + k], ks[g], x);
            s[t][nq][h * 2 + k] = x;
          }
      }
    }
    if (!whole) {
#pragma unroll
      for (int t = 0; t < KT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int key = first + t * 16 + k0 + 8 * h;
          const bool valid = ((here >> t) & 1) && key < key1;
#pragma unroll
          for (int g = 0; g < (G + 1) / 2; g++) vs[t][h][g] = valid ? vs[t][h][g] : 0u;
#pragma unroll
          for (int nq = 0; nq < NQ; nq++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
              const int r = rtile * QROWS + nq * 8 + c * 2 + k;
              if (!(valid && key <= have + r / p.group)) s[t][nq][h * 2 + k] = -INFINITY;
            }
        }
    }
    // Does a score pass its column's maximum by 2^8, or a scale of v its power of two, in this lane? (q_back > 0)
    bool grow = false;
    float mt[NQ][2];
#pragma unroll
    for (int nq = 0; nq < NQ; nq++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        float x = fmaxf(s[0][nq][k], s[0][nq][2 + k]);
#pragma unroll
        for (int t = 1; t < KT; t++) x = fmaxf(x, fmaxf(s[t][nq][k], s[t][nq][2 + k]));
        mt[nq][k] = x * q_back[nq][k];
        grow = grow || mt[nq][k] > m[nq][k] + 8.f;
      }
    if constexpr (EXACT) {
      uint32_t vt[(G + 1) / 2];
      bool large = false;
#pragma unroll
      for (int g = 0; g < (G + 1) / 2; g++) {
        vt[g] = 0;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
          for (int h = 0; h < 2; h++) vt[g] = __vmaxu2(vt[g], vs[t][h][g] & 0x7fff7fffu);
        large = large || __vmaxu2(vt[g], limit[g]) != limit[g];
      }
      if (__any_sync(0xffffffffu, grow || large)) {
        int least[G], most[G];  // the lowest power of the warp's columns, the exponent of the step's largest scale
        uint32_t top[NQ][G];    // both columns' largest product of a weight and a scale in the step, upper halves of f32
        float old[NQ][2];       // what the maximum's growth takes from a column, as a factor and (at most that) as a power
        int drop[NQ][2];
        // (all columns side by side, so that their exchanges overlap)
#pragma unroll
        for (int away = 4; away <= 16; away *= 2)
#pragma unroll
          for (int nq = 0; nq < NQ; nq++)
#pragma unroll
            for (int k = 0; k < 2; k++) mt[nq][k] = fmaxf(mt[nq][k], __shfl_xor_sync(0xffffffffu, mt[nq][k], away));
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const float now = fmaxf(mt[nq][k], m[nq][k]);
            old[nq][k] = now > m[nq][k] ? ex2_ftz(m[nq][k] - now) : 1.f;
            drop[nq][k] = now > m[nq][k] ? (int)fminf(now - m[nq][k], 64.f) : 0;
            m[nq][k] = now;
            l[nq][k] *= old[nq][k];
          }
          uint32_t of[G][2] = {};
#pragma unroll
          for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float p = ex2_ftz(fmaf(s[t][nq][e], q_back[nq][e & 1], -m[nq][e & 1]));
#pragma unroll
              for (int g = 0; g < G; g++) {
                const uint32_t raw = vs[t][e >> 1][g / 2];
                const float sv = __half2float(__ushort_as_half((uint16_t)((g & 1) ? raw >> 16 : raw)));
                of[g][e & 1] = max(of[g][e & 1], p > 0.f ? __float_as_uint(p * sv) & 0x7fffffffu : 0u);
              }
            }
#pragma unroll
          for (int g = 0; g < G; g++) top[nq][g] = __byte_perm(of[g][0], of[g][1], 0x7632);
        }
#pragma unroll
        for (int away = 4; away <= 16; away *= 2)
#pragma unroll
          for (int nq = 0; nq < NQ; nq++)
#pragma unroll
            for (int g = 0; g < G; g++) top[nq][g] = __vmaxu2(top[nq][g], __shfl_xor_sync(0xffffffffu, top[nq][g], away));
#pragma unroll
        for (int g = 0; g < G; g++) most[g] = (int)(__reduce_max_sync(0xffffffffu, (g & 1) ? vt[g / 2] >> 16 : vt[g / 2] & 0xffffu) >> 10);
#pragma unroll
        for (int g = 0; g < G; g++) {
          least[g] = 30;
#pragma unroll
          for (int nq = 0; nq < NQ; nq++) {
            float corr[2];
            uint32_t field = 0;
#pragma unroll
            for (int k = 0; k < 2; k++) {
              // the exponent that the largest product needs, as a scale's: with up to 2^ABOVE of room for larger scales
              const int need = (int)((top[nq][g] >> (16 * k + 7)) & 255u) - 112, had = 31 - (int)((power[nq][g] >> (16 * k + 10)) & 31u);
              const int now = min(max(max(had - drop[nq][k], max(need, min(most[g], need + ABOVE))), 1), 30);
              least[g] = min(least[g], now);
              corr[k] = old[nq][k] * __uint_as_float((uint32_t)(127 + had - now) << 23);
              field |= (uint32_t)(31 - now) << (16 * k + 10);
            }
            power[nq][g] = field;
#pragma unroll
            for (int e = 0; e < 4; e++) {
#pragma unroll
              for (int t = 0; t < 4; t++) o[nq][g * 4 + t][e] *= corr[e & 1];
              w_sum[nq][g][e] *= corr[e & 1];
            }
          }
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
          // (scales of NaN and infinities always pass the limit)
          const int upto = min(__reduce_min_sync(0xffffffffu, least[g]) + ABOVE, 30);
          const uint32_t bits = (uint32_t)upto << 10 | 0x3ffu;
          limit[g / 2] = (g & 1) ? (limit[g / 2] & 0xffffu) | bits << 16 : bits;
        }
      }
    } else {
      uint32_t vt = 0, vb = 0xffffffffu;
#pragma unroll
      for (int t = 0; t < KT; t++)
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int g = 0; g < (G + 1) / 2; g++) {
            vt = G == 1 ? max(vt, vs[t][h][g]) : __vmaxu2(vt, vs[t][h][g]);
            vb = G == 1 ? min(vb, vs[t][h][g]) : __vminu2(vb, vs[t][h][g]);
          }
      if (G > 1) vt = max(vt & 0xffffu, vt >> 16), vb = min(vb & 0xffffu, vb >> 16);
      const bool move = grow || vt > v_range >> 16;
      if (__any_sync(0xffffffffu, move || vb < (v_range & 0xffffu))) {
        const bool rescale = __any_sync(0xffffffffu, move);  // (else some scales are 0, which are no values, or too small)
        // O and the sums of weights are kept over 2^(exponent of the largest scale)
        const uint32_t had = v_range >> 26, top = max(__reduce_max_sync(0xffffffffu, vt), had << 10), e = top >> 10;
        // the smallest scale that is held well beside it: 2^-RANGE of it (smaller ones before it are in O, in f32)
        const uint32_t least = e > RANGE ? top - (RANGE << 10) : 0x400u >> min(RANGE + 1u - e, 11u);
        v_range = (top | 0x3ffu) << 16 | least;
        bool small = false;
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int g = 0; g < G; g++) {
              const uint32_t bits = (g & 1) ? vs[t][h][g / 2] >> 16 : vs[t][h][g / 2] & 0xffffu;
              small = small || (bits != 0 && bits < least);
            }
        if (top >= 0x7c00u || __any_sync(0xffffffffu, small)) return false;  // (a negative scale is one of the former)
        const float f = __uint_as_float((127u + had - e) << 23);
#pragma unroll
        for (int nq = 0; nq < NQ && rescale; nq++) {
          float corr[2];
#pragma unroll
          for (int k = 0; k < 2; k++) {
            float x = mt[nq][k];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            corr[k] = 1.f;
            if (x > m[nq][k]) {
              corr[k] = ex2_ftz(m[nq][k] - x);
              m[nq][k] = x;
            }
            l[nq][k] *= corr[k];
            corr[k] *= f;
          }
#pragma unroll
          for (int t = 0; t < MTILES; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[nq][t][e] *= corr[e & 1];
#pragma unroll
          for (int g = 0; g < G; g++)
#pragma unroll
            for (int e = 0; e < 4; e++) w_sum[nq][g][e] *= corr[e & 1];
        }
      }
    }
    // scales of v times 2^(15 - e) (TERMS 2: 2^(21 - e)), e the exponent field of the largest: below 2, so that a weight of
    // 2^(8 + UP) at most times it stays below 2^15 (2^15)
    const float v_up = __uint_as_float((148u - (v_range >> 26)) << 23);
    const __half2 v_up2 = __float2half2_rn(v_up * 0.015625f);
#pragma unroll
    for (int t = 0; t < KT; t++) {
      float pw[NQ][4];
#pragma unroll
      for (int nq = 0; nq < NQ; nq++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          pw[nq][e] = ex2_ftz(fmaf(s[t][nq][e], q_back[nq][e & 1], UP - m[nq][e & 1]));
          l[nq][e & 1] += pw[nq][e];
        }
      const uint8_t* kt = st + (t * 2) * TILE;
      // TERMS 1: weights and scales as f16, their products rounded once more (2^-11 each)
      __half2 ph[NQ][2];
      uint32_t vn[2][(G + 1) / 2];
      if constexpr (TERMS == 1 && !EXACT) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int nq = 0; nq < NQ; nq++) ph[nq][h] = __floats2half2_rn(pw[nq][h * 2], pw[nq][h * 2 + 1]);
#pragma unroll
          for (int g = 0; g < (G + 1) / 2; g++) vn[h][g] = as_u32(__hmul2(as_half2(vs[t][h][g]), v_up2));
        }
      }
#pragma unroll
      for (int g = 0; g < G; g++) {
        // weights times scales as the B operand: S^T's rows (keys) become the 16 values of the product
        uint32_t bw[NQ][TERMS][2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          if constexpr (TERMS == 1 && !EXACT) {
            const __half2 both = as_half2(vn[h][g / 2]), sv = (g & 1) ? __high2half2(both) : __low2half2(both);
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) bw[nq][0][h] = transposed(as_u32(__hmul2(ph[nq][h], sv)));
          } else {
            const uint32_t raw = vs[t][h][g / 2];
            const float sv = __half2float(__ushort_as_half((uint16_t)((g & 1) ? raw >> 16 : raw)));
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) {
              float x0, x1;
              if constexpr (EXACT) {  // (a scale of NaN is its key's rows' alone)
                x0 = s[t][nq][h * 2] == -INFINITY ? 0.f : pw[nq][h * 2] * (sv * power_up(power[nq][g] & 0xffffu, TERMS));
                x1 = s[t][nq][h * 2 + 1] == -INFINITY ? 0.f : pw[nq][h * 2 + 1] * (sv * power_up(power[nq][g] >> 16, TERMS));
              } else {
                x0 = pw[nq][h * 2] * (sv * v_up), x1 = pw[nq][h * 2 + 1] * (sv * v_up);
              }
              const __half2 v = __floats2half2_rn(x0, x1);
              if constexpr (TERMS == 1) {
                bw[nq][0][h] = transposed(as_u32(v));
                continue;
              }
              const float2 f = __half22float2(v);
              bw[nq][0][h] = transposed(as_u32(v));
              bw[nq][TERMS - 1][h] = transposed(as_u32(__floats2half2_rn(x0 - f.x, x1 - f.y)));
            }
          }
        }
        if constexpr (TERMS == 1) {
          const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
          for (int nq = 0; nq < NQ; nq++) mma_f16(w_sum[nq][g], ones, bw[nq][0][0], bw[nq][0][1]);
        }
        // v: word u (dims 8 u .. 8 u + 7 of the group) of the keys of rows 2 c, 2 c + 1, 2 c + 8, 2 c + 9
        const uint32_t v0 = *reinterpret_cast<const uint32_t*>(kt + v_at[g]);
        const uint32_t v1 = *reinterpret_cast<const uint32_t*>(kt + v_at_4(g));
        const uint32_t v2 = *reinterpret_cast<const uint32_t*>(kt + v_at[g] + 8 * ROW);
        const uint32_t v3 = *reinterpret_cast<const uint32_t*>(kt + v_at_4(g) + 8 * ROW);
#pragma unroll
        for (int h = 0; h < 2; h++) {  // dims 8 u + 4 h ..
          const uint32_t x = __byte_perm(v0, v1, h ? 0x7632 : 0x5410), y = __byte_perm(v2, v3, h ? 0x7632 : 0x5410);
#pragma unroll
          for (int j = 0; j < 2; j++) {  // rows u and u + 8 of the tile: dims 8 u + 4 h + 2 j and the next (times 16)
            const uint32_t xs = x >> (8 * j), ys = y >> (8 * j);
            uint32_t av[4];
            if constexpr (TERMS == 1) {
              av[0] = and_xor(xs, low, 0x00080008u), av[1] = and_xor(xs, high, 0x00800080u);
              av[2] = and_xor(ys, low, 0x00080008u), av[3] = and_xor(ys, high, 0x00800080u);
            } else {
              av[0] = as_u32(__hadd2(as_half2(and_xor(xs, low, 0x64086408u)), sub1));
              av[1] = as_u32(__hadd2(as_half2(and_xor(xs, high, 0x64806480u)), sub16));
              av[2] = as_u32(__hadd2(as_half2(and_xor(ys, low, 0x64086408u)), sub1));
              av[3] = as_u32(__hadd2(as_half2(and_xor(ys, high, 0x64806480u)), sub16));
            }
#pragma unroll
            for (int nq = 0; nq < NQ; nq++)
#pragma unroll
              for (int k = 0; k < TERMS; k++) mma_f16(o[nq][g * 4 + h * 2 + j], av, bw[nq][k][0], bw[nq][k][1]);
          }
        }
      }
    }
    __syncwarp();  // every lane has read the stage that is copied into next
  }
#pragma unroll
  for (int nq = 0; nq < NQ; nq++)
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int k = 0; k < 2; k++)  // (2^-(15 - e), 2^-(21 - e) in a first sweep)
        down[nq][g][k] = EXACT ? power_down((power[nq][g] >> (16 * k)) & 0xffffu, TERMS)
                               : __uint_as_float(((v_range >> 26) + (TERMS == 1 ? 112u : 106u)) << 23);
  return true;
}

// What a CTA does: its share of the keys of a sequence, for one tile of q rows of a kv head, and its part of the merge.
// D: dim; NQ: tiles of 8 q rows; KT: tiles of 16 keys of a step; TERMS: f16 terms of q and of the weights.
template <int D, int NQ, int KT, int TERMS, bool EXACT>
__device__ __forceinline__ void attend_tile(const Params& p) {
  constexpr int STEP = KT * 16, QROWS = 8 * NQ, MTILES = D / 16, PITCH = MERGE_PITCH<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3, u = lane >> 2;
  const int rank = blockIdx.x % CLUSTER, run = blockIdx.x / CLUSTER, b = blockIdx.z;  // CTA of the cluster, run of keys
  const int head = blockIdx.y / p.row_tiles, rtile = blockIdx.y % p.row_tiles;  // kv head, tile of q rows
  const int unit = (b * gridDim.y) + blockIdx.y;

  // the page table's row is asked for beside the length, not behind it
  if (warp == 0 && lane * 32 < p.c.max_pages)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(p.c.page_table + (int64_t)b * p.c.max_pages + lane * 32));
  // this lane's q values (see below) come first: they need no length
  uint4 q_raw[NQ][D / 64][4];
  load_q<D, NQ>(p, b, head, rtile, q_raw);

  const int length = p.c.lengths[b];
  const int64_t room = p.c.max_pages * p.c.page;
  const int have = (int)min((int64_t)length, room);  // (a length may be any 32 bits; past the table all its keys are seen)
  const int64_t want = (int64_t)length + min(p.tokens, (rtile * QROWS + QROWS - 1) / p.group + 1);  // keys of the tile's last row
  const int keys = have < 0 ? 0 : (int)min(want, room);
  if (have >= 0 && want > room && blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(p.err, 0u, (uint32_t)DEV_ERR_KV_FULL);
  const int runs = max(1, (int)(((uint32_t)keys + CLUSTER * p.chunk - 1) / (uint32_t)(CLUSTER * p.chunk)));
  if (run >= runs) return;  // (the whole cluster)
  const int share = ((keys + runs * CLUSTER - 1) / (runs * CLUSTER) + STEP - 1) / STEP * STEP;  // keys of each CTA
  const int key0 = min(keys, (run * CLUSTER + rank) * share), key1 = min(keys, key0 + share);

  // The warps' O, maxima and sums, merged in shared memory (the rings are done): [warp][row](D values, m, l)
  float* mem = reinterpret_cast<float*>(smem);
  Part<D, NQ> part;
  const bool done = sweep<D, NQ, KT, TERMS, EXACT>(p, b, head, rtile, have, key0, key1, smem, q_raw, part);
  cp_async_wait<0>();
  if (__builtin_expect(__syncthreads_or(!done), 0)) {
    if constexpr (!EXACT) attend_tile<D, NQ, KT, TERMS, true>(p);
    return;
  }
#pragma unroll
  for (int nq = 0; nq < NQ; nq++)
#pragma unroll
    for (int k = 0; k < 2; k++) {
      float sum = part.l[nq][k];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      float* to = mem + (warp * QROWS + nq * 8 + c * 2 + k) * PITCH;
#pragma unroll
      for (int t = 0; t < MTILES; t++) {  // group t / 4, dims 8 u + 2 (t % 4) and the next
        float x0 = part.o[nq][t][k], x1 = part.o[nq][t][2 + k];
        if constexpr (TERMS == 1) {
          const float off = 8.f * part.w_sum[nq][t / 4][k];
          x0 = fmaf(x0, 16777216.f, -off);
          x1 = fmaf(x1, 1048576.f, -off);
        } else {
          x1 *= 0.0625f;
        }
        *reinterpret_cast<float2*>(to + (t / 4) * 64 + u * 8 + (t % 4) * 2) = make_float2(x0 * part.down[nq][t / 4][k], x1 * part.down[nq][t / 4][k]);
      }
      if (u == 0) {
        to[D] = part.m[nq][k];
        to[D + 1] = sum;
      }
    }
  __syncthreads();
  auto finish = [&](int r, int d, float4 acc, float sum) {  // 4 values of row r of the tile from dim d on
    const int row = rtile * QROWS + r;
    if (row >= p.rows) return;
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // no key seen: zeros; NaN stays
    const int64_t at = ((int64_t)b * p.tokens + row / p.group) * p.out_stride + (int64_t)(head * p.group + row % p.group) * D + d;
    const float v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (p.out_dtype == WE_F32) store_out<WE_F32>(p.out, at + e, v[e]);
      else store_out<WE_BF16>(p.out, at + e, v[e]);
    }
  };
  merge_parts<D, QROWS, WARPS, CLUSTER>(mem, p.part, p.done, &last, unit, (int)gridDim.x / CLUSTER, runs, run, rank, finish);
}
}  // namespace kv

// PER_SM: CTAs that an SM holds by their registers.
template <int D, int NQ, int KT, int TERMS, int PER_SM>
__global__ void __launch_bounds__(kv::THREADS, PER_SM) kv4_attention_kernel(const __grid_constant__ kv::Params p) {
  pdl_launch_dependents();
  pdl_wait();
  kv::attend_tile<D, NQ, KT, TERMS, false>(p);
}

// How rows are cut: a token over as many threads as it has units, evenly over several rounds of at most ROW_THREADS (over
// CTAs where there are few tokens); 8 tokens a thread where that leaves two CTAs an SM.
struct RowPlan {
  RowShape shape;
  dim3 grid;
  int threads;
};
static RowPlan kv4_rows(const we_kv4_cache& c, int64_t tokens, int sms) {
  RowPlan p;
  const int64_t units = 2 * c.kv_heads * (c.dim / 8), all = c.batch * tokens, rounds = (units + ROW_THREADS - 1) / ROW_THREADS;
  p.shape.units = (int)units;
  p.shape.head_shift = c.dim == 64 ? 3 : c.dim == 128 ? 4 : 5;
  p.shape.lanes = (int)(((units + rounds - 1) / rounds + 7) / 8 * 8);
  p.shape.along = (int)std::min<int64_t>({ROW_THREADS / p.shape.lanes, ROW_SPAN, std::max<int64_t>(1, all / (2 * sms))});
  p.shape.span = (int)std::min<int64_t>(ROW_SPAN, p.shape.along * std::max<int64_t>(1, std::min<int64_t>(8, all / (2 * sms * p.shape.along))));
  p.threads = (p.shape.lanes * p.shape.along + 31) / 32 * 32;
  const int64_t x = std::min<int64_t>((all + p.shape.span - 1) / p.shape.span, 0x7fffffff);
  p.grid = dim3((unsigned)x, (unsigned)rounds);
  return p;
}

cudaError_t launch_kv4_append(const we_kv4_cache& c, const void* k, const void* v, int dt, int64_t tokens,
                              int64_t stride, uint32_t* err, int sms, cudaStream_t st) {
  const RowPlan p = kv4_rows(c, tokens, sms);
  const int64_t es = dt == WE_F32 ? 4 : 2;
  const bool wide = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | (uintptr_t)(stride * es)) & 15) == 0;
  const bool many = (int64_t)p.grid.x * p.grid.y > 2 * sms;
#define APPEND_CASE(DT, WIDE) (many ? kv4_append_kernel<DT, WIDE, 6> : kv4_append_kernel<DT, WIDE, 1>)
  const auto kernel = dt == WE_F32 ? (wide ? APPEND_CASE(WE_F32, true) : APPEND_CASE(WE_F32, false))
                                   : (wide ? APPEND_CASE(WE_BF16, true) : APPEND_CASE(WE_BF16, false));
#undef APPEND_CASE
  const cudaError_t e = launch_pdl(kernel, p.grid, p.threads, 0, st, c, k, v, tokens, stride, p.shape, err);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

cudaError_t launch_kv4_unpack(const we_kv4_cache& c, void* k, void* v, int dt, int64_t tokens, const int32_t* start,
                              uint32_t* err, int sms, cudaStream_t st) {
  const RowPlan p = kv4_rows(c, tokens, sms);
  const auto kernel = dt == WE_F32 ? kv4_unpack_kernel<WE_F32> : kv4_unpack_kernel<WE_BF16>;
  const cudaError_t e = launch_pdl(kernel, p.grid, p.threads, 0, st, c, k, v, tokens, start, p.shape, err);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

cudaError_t launch_kv4_advance(const we_kv4_cache& c, int64_t tokens, cudaStream_t st) {
  const unsigned grid = (unsigned)((c.batch + 127) / 128);
  const cudaError_t e = launch_pdl(kv4_advance_kernel, dim3(grid), 128, 0, st, c.lengths, c.batch, (int32_t)tokens);
  return e == cudaSuccess ? cudaGetLastError() : e;
}

namespace {
// CTAs an SM by registers. f32: three (4 sequences of 16000 keys, 48 heads of 128 on 12, took 52 us with four and take 40). bf16:
// four, for which 128-wide heads spill 16 bytes; calls of so few CTAs that three an SM hold them do better with three (2
// sequences of 4096 keys, 8 heads: 10.4 us against 12.5; 16 of 3001 to 16384, 48 on 12: 75.1 against 65.3).
constexpr int kv4_per_sm(int dim, int nq, int terms) {
  return dim * nq == 512 ? 1 : dim * nq == 256 ? 2 : terms == 2 ? 3 : 4;
}

// How the work of a call is cut: q rows into tiles of 8 or 16, keys into chunks of a CTA.
struct Kv4Plan {
  int nq, row_tiles, runs, chunk;
  int64_t units, part_floats;
};
Kv4Plan kv4_plan(const Kv4AttnArgs& a, int sms) {
  Kv4Plan q{};
  const int64_t rows = a.tokens * (a.heads / a.c.kv_heads);
  q.nq = rows <= 8 ? 1 : 2;
  q.row_tiles = (int)((rows + 8 * q.nq - 1) / (8 * q.nq));
  q.units = a.c.batch * a.c.kv_heads * q.row_tiles;
  // The CTAs that the SMs hold, four an SM (f32: three), less what no cluster of 8 fits into (71 of 74 do). A sequence's length is
  // known on the device only, so runs are cut for the longest possible one, into about one wave of CTAs; more and shorter ones
  // cost more in their first and last steps than ragged lengths gain (68 us against 81 with four waves for 16 sequences of 3001
  // to 16384 keys, 60 against 78 for one of 131000). Merging runs takes as long as some 800 keys of a CTA (500 in f32, whose keys
  // take longer), so that many have to be saved. One sequence, 12 kv heads, in one run and in as many as fit: bf16, dim 128: 4096
  // keys 9.8 and 11.7, 8192 13.4 and 14.0, 16384 21.1 and 17.3 us; dim 64: 8.2 and 10.8, 11.1 and 11.6, 16.7 and 13.8; f32, dim
  // 128: 4096 12.1 and 12.9, 8192 17.8 and 14.2; dim 64: 9.7 and 11.1, 13.8 and 11.9. Where one more run would take a few CTAs more
  // than three an SM, f32 stays below (2 sequences of 16384 keys, 16 heads of 128: 40 us, 46 in two runs).
  const int64_t cap = std::max<int64_t>(1, a.c.max_pages * a.c.page), alone = (cap + kv::CLUSTER - 1) / kv::CLUSTER;
  const bool three = (a.dtype == WE_F32 || a.out_dtype == WE_F32) && a.c.dim <= 128;
  const int per_sm = three ? 3 : 4;
  const int64_t fit = std::max<int64_t>(1, (int64_t)(sms - 6) * per_sm / (q.units * kv::CLUSTER));
  const int64_t runs = alone - alone / fit > (three ? 500 : 800) ? fit : 1;
  const int64_t chunk = std::max<int64_t>(256, (alone + runs - 1) / runs);
  q.chunk = (int)((std::min<int64_t>(chunk, 0x4000000) + 31) / 32 * 32);
  q.runs = (int)((cap + (int64_t)q.chunk * kv::CLUSTER - 1) / ((int64_t)q.chunk * kv::CLUSTER));
  q.part_floats = q.runs > 1 ? q.units * q.runs * 8 * q.nq * (a.c.dim + 4) : 0;
  return q;
}

template <int D, int NQ, int KT, int TERMS, int PER_SM = kv4_per_sm(D, NQ, TERMS)>
cudaError_t kv4_launch(const kv::Params& p, dim3 grid, cudaStream_t st) {
  auto kern = kv4_attention_kernel<D, NQ, KT, TERMS, PER_SM>;
  constexpr int ring = kv::WARPS * kv::ring_depth<D, KT>() * KT * (D * 16 + D);
  constexpr int merge = (kv::WARPS + 1) * 8 * NQ * (D + 4) * 4;
  constexpr int bytes = ring > merge ? ring : merge;
  const cudaError_t e = allow_smem(kern, bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kv::THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kv::CLUSTER;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  pdl_attribute(attr[1]);
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, p);
}
}  // namespace

void kv4_attention_scratch(const Kv4AttnArgs& a, int sms, int64_t* part_bytes, int64_t* units) {
  const Kv4Plan q = kv4_plan(a, sms);
  *part_bytes = q.part_floats * 4;
  *units = q.runs > 1 ? q.units : 0;
}

cudaError_t launch_kv4_attention(const Kv4AttnArgs& a, void* part, uint32_t* done, uint32_t* err, int sms, cudaStream_t st) {
  const Kv4Plan q = kv4_plan(a, sms);
  kv::Params p{};
  p.c = a.c;
  p.q = a.q;
  p.out = a.out;
  p.tokens = (int)a.tokens;
  p.heads = (int)a.heads;
  p.group = (int)(a.heads / a.c.kv_heads);
  p.rows = p.tokens * p.group;
  p.row_tiles = q.row_tiles;
  p.chunk = q.chunk;
  p.wide_q = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * (a.dtype == WE_F32 ? 4 : 2))) & 15) == 0;
  p.q_stride = a.q_stride;
  p.out_stride = a.out_stride;
  p.scale_log2 = fabsf(a.scale) * 1.4426950408889634f;
  p.negative = a.scale < 0.f;
  p.dtype = a.dtype;
  p.out_dtype = a.out_dtype;
  p.part = static_cast<float*>(part);
  p.done = done;
  p.err = err;
  const dim3 grid((unsigned)(q.runs * kv::CLUSTER), (unsigned)(a.c.kv_heads * q.row_tiles), (unsigned)a.c.batch);
  const bool f32 = a.dtype == WE_F32 || a.out_dtype == WE_F32;
  cudaError_t e;
#define KV4_CASE(D)                                                                                             \
  e = f32 ? (q.nq == 1 ? kv4_launch<D, 1, 1, 2>(p, grid, st) : kv4_launch<D, 2, 1, 2>(p, grid, st))             \
          : (q.nq == 1 ? kv4_launch<D, 1, D == 256 ? 1 : 2, 1>(p, grid, st) : kv4_launch<D, 2, 1, 1>(p, grid, st))
  if (a.c.dim == 64) KV4_CASE(64);
  else if (a.c.dim == 128 && !f32 && q.nq == 1 && (int64_t)grid.x * grid.y * grid.z <= 3 * sms - 24) e = kv4_launch<128, 1, 2, 1, 3>(p, grid, st);
  else if (a.c.dim == 128) KV4_CASE(128);
  else KV4_CASE(256);
#undef KV4_CASE
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace we
