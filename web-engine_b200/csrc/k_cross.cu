// Cross attention: queries of one sequence over another sequence's keys and values, with key lengths and a byte mask.
//
// cross_tile_kernel: any size, stride and dim up to 256. Few query rows read much and compute little, so it is bound by the
// bytes of k and v; its tiles are the ones of the cached attention (S^T = K Q^T and O^T = V^T P^T, keys and dims as the 16
// rows of warp-level tensor products, up to 8 query rows as the columns), the keys split over warps, a cluster's CTAs and
// clusters, and merged in a fixed order (attn_merge.cuh).
// - bf16: k and v go from shared memory into the products as they are (ldmatrix, for v transposed), p as bf16: both operands
//   of a product have one type, and v's range is bf16's. Its rounding (2^-9 each, sums in f32) is 0.0013 of an output's size
//   beside 0.0017 of the output's own; a second term for p would be half as many products again.
// - f32: every operand is two tf32 terms (22 bits) and a product three (the two small terms' product is below 2^-22).
// Hidden keys: their scores are -inf and their rows of v zeros, so that nothing of them reaches a product.
#include <algorithm>

#include "attn_merge.cuh"
#include "common.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace we {

namespace cross {
constexpr int WARPS = 4, THREADS = WARPS * 32, TILE = 16;

struct Params {
  we_cross_desc d;  // strides and scale resolved
  int group, rows, row_tiles;  // heads per kv head; rows = tq * group; tiles of 8 NQ rows
  int chunk;                   // keys per CTA at most
  int wide_kv, wide_q;         // k and v by 16-byte copies; q by 4-byte loads
  float scale_log2;            // |scale| log2(e)
  int negative;                // scores change sign before any is hidden (q as it is loaded: 3 us of 38 for one query, 4096 keys)
  float* part;
  uint32_t* done;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {  // of an 8 x 8 tile of 16-bit values
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// x as two tf32 terms: the nearest one (to 11 bits, ties up), and what is left, of whose 12 bits the product drops one.
// (cvt.rna.tf32 takes several instructions here: 1024 queries x 512 keys of 12 heads 192 us with it.)
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
// d += a b in three products
__device__ __forceinline__ void mma_3tf32(float (&d)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], const uint32_t (&b)[4]) {
  mma_tf32(d, al, b[0], b[1]);
  mma_tf32(d, ah, b[2], b[3]);
  mma_tf32(d, ah, b[0], b[1]);
}

// Which 16-byte piece of row r the piece `ch` is kept as: rows that lanes read together lie on different banks. bf16: the 8
// rows of an ldmatrix. f32: for k rows r and r + 1, for v rows 0 2 4 6 (and 1 3 5 7).
template <bool F32>
__device__ __forceinline__ int piece(int r, int ch, int is_v) {
  if (!F32) return ch ^ (r & 7);
  return is_v ? ch ^ (((r >> 1) & 3) << 1) : ch ^ ((r & 1) << 2);
}
}  // namespace cross

// F32: type of q, k and v; D: dim rounded up; NQ: tiles of 8 query rows; DEPTH: steps of 16 keys in a warp's ring; CLUSTER:
// CTAs that share a run of keys.
template <bool F32, int D, int NQ, int DEPTH, int CLUSTER>
__global__ void __launch_bounds__(cross::THREADS) cross_tile_kernel(const cross::Params p) {
  using namespace cross;
  constexpr int ES = F32 ? 4 : 2, ROW = D * ES, SIDE = TILE * ROW, STAGE = 2 * SIDE, QROWS = 8 * NQ, MTILES = D / 16;
  constexpr int QBYTES = F32 ? NQ * (D / 8) * 32 * 16 : 0;  // f32: q's terms, in the order of the products
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int last;
  const we_cross_desc& a = p.d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3, u = lane >> 2;
  const int rank = blockIdx.x % CLUSTER, run = blockIdx.x / CLUSTER;
  const int rtile = blockIdx.y % p.row_tiles, head = blockIdx.y / p.row_tiles, b = blockIdx.z;  // kv head
  const int unit = b * gridDim.y + blockIdx.y, dim = (int)a.dim;
  pdl_launch_dependents();
  pdl_wait();

  int keys = (int)a.tk;
  if (a.key_lengths) keys = max(0, min(keys, a.key_lengths[b]));
  const int runs = max(1, (int)(((int64_t)keys + CLUSTER * p.chunk - 1) / (CLUSTER * p.chunk)));
  if (run >= runs) return;  // (the whole cluster)
  const int share = ((keys + runs * CLUSTER - 1) / (runs * CLUSTER) + TILE - 1) / TILE * TILE;  // keys of each CTA
  const int key0 = min(keys, (run * CLUSTER + rank) * share), key1 = min(keys, key0 + share);
  const int steps = (key1 - key0 + TILE - 1) / TILE;
  const int mine = steps > warp ? (steps - warp + WARPS - 1) / WARPS : 0;  // tiles warp, warp + 4, ...

  uint8_t* ring = smem + QBYTES + warp * (DEPTH * STAGE);
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
  const uint8_t* mask = a.key_mask ? a.key_mask + (int64_t)b * a.tk : nullptr;
  // f32: a side's place is filled again as soon as it is read, so that one stage a warp (three CTAs an SM; two stages leave
  // one) keeps copies on their way: one token to 4096 keys of 8 x 12 heads of 128 158 -> 72 us. bf16 has room for two
  // stages, the next one's copies queued before this one is waited for (3% faster there).
  constexpr bool EARLY = F32;
  static_assert(EARLY || DEPTH > 1, "");
  uint32_t seen[DEPTH];  // which of a stage's 16 keys are seen
  auto copy = [&](int i, int st, int side) {  // k first: that also finds which keys are seen
    if (i < mine) {
      const int first = key0 + (warp + WARPS * i) * TILE;
      if (side == 0) {
        const int key = first + lane;
        seen[st] = __ballot_sync(0xffffffffu, lane < TILE && key < key1 && (!mask || mask[key] != 0));
      }
      const int there = min(TILE, key1 - first);  // rows that exist
      if (seen[st]) {
        const int64_t stride = side ? a.v_stride : a.k_stride;
        const uint8_t* from = static_cast<const uint8_t*>(side ? a.v : a.k) + (((int64_t)b * a.tk + first) * stride + (int64_t)head * dim) * ES;
        uint8_t* to = ring + st * STAGE + side * SIDE;
        const uint32_t to_addr = ring_addr + st * STAGE + side * SIDE;
        if (p.wide_kv) {
#pragma unroll
          for (int j = 0; j < SIDE / 512; j++) {
            const int at = j * 32 + lane, r = at / (ROW / 16), ch = at % (ROW / 16);
            if (r < there && ch * 16 < dim * ES)
              cp_async16(to_addr + r * ROW + piece<F32>(r, ch, side) * 16, from + r * stride * ES + ch * 16);
          }
        } else {  // value by value
          for (int at = lane; at < TILE * dim; at += 32) {
            const int r = at / dim, e = at - r * dim;
            if (r >= there) break;
            uint8_t* dst = to + r * ROW + piece<F32>(r, e * ES / 16, side) * 16 + (e * ES) % 16;
            if constexpr (F32) *reinterpret_cast<uint32_t*>(dst) = reinterpret_cast<const uint32_t*>(from)[r * stride + e];
            else *reinterpret_cast<uint16_t*>(dst) = reinterpret_cast<const uint16_t*>(from)[r * stride + e];
          }
        }
      }
    }
    cp_async_commit();
  };
  if (dim < D) {  // the places past dim stay zero
    for (int at = threadIdx.x; at < WARPS * DEPTH * STAGE / 16; at += THREADS)
      reinterpret_cast<uint4*>(smem + QBYTES)[at] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
#pragma unroll
  for (int d = 0; d < (EARLY ? DEPTH : DEPTH - 1); d++) {
    copy(d, d, 0);
    copy(d, d, 1);
  }

  // q as the B operand: column lane / 4 of tile nq is row nq * 8 + lane / 4
  auto q_row = [&](int nq) -> int64_t {
    const int r = rtile * QROWS + nq * 8 + u;
    if (r >= p.rows) return -1;
    return ((int64_t)b * a.tq + r / p.group) * a.q_stride + (int64_t)(head * p.group + r % p.group) * dim;
  };
  uint32_t qf[F32 ? 1 : NQ][F32 ? 1 : D / 16][2];
  uint4* q_terms = reinterpret_cast<uint4*>(smem);  // [nq][step of 8 dims][lane]: b0, b1 and what is left of them
  if constexpr (F32) {
    // values 4 c .. 4 c + 3 of each 16: the first two belong to one step of 8, the others to the next
    for (int s = warp; s < D / 16; s += WARPS)
#pragma unroll
      for (int nq = 0; nq < NQ; nq++) {
        const int64_t row = q_row(nq);
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int d = s * 16 + c * 4 + e;
          x[e] = row >= 0 && d < dim ? static_cast<const float*>(a.q)[row + d] : 0.f;
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint4 t;
          split_tf32(x[2 * h], t.x, t.z);
          split_tf32(x[2 * h + 1], t.y, t.w);
          q_terms[(nq * (D / 8) + s * 2 + h) * 32 + lane] = t;
        }
      }
    __syncthreads();
  } else {
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
      const int64_t row = q_row(nq);
#pragma unroll
      for (int s = 0; s < D / 16; s++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int d = s * 16 + h * 8 + c * 2;
          uint32_t v = 0;
          if (row >= 0 && d < dim) {
            const uint16_t* from = static_cast<const uint16_t*>(a.q) + row + d;
            if (p.wide_q) v = *reinterpret_cast<const uint32_t*>(from);
            else v = from[0] | (d + 1 < dim ? (uint32_t)from[1] << 16 : 0u);
          }
          qf[nq][s][h] = v;
        }
    }
  }

  float o[NQ][MTILES][4], m[NQ][2], l[NQ][2];
#pragma unroll
  for (int nq = 0; nq < NQ; nq++) {
#pragma unroll
    for (int t = 0; t < MTILES; t++) o[nq][t][0] = o[nq][t][1] = o[nq][t][2] = o[nq][t][3] = 0.f;
    m[nq][0] = m[nq][1] = NONE;
    l[nq][0] = l[nq][1] = 0.f;
  }

  for (int i0 = 0; i0 < mine; i0 += DEPTH) {
#pragma unroll
    for (int st = 0; st < DEPTH; st++) {
      const int i = i0 + st;
      if (i >= mine) break;
      if constexpr (!EARLY) {
        copy(i + DEPTH - 1, (st + DEPTH - 1) % DEPTH, 0);
        copy(i + DEPTH - 1, (st + DEPTH - 1) % DEPTH, 1);
      }
      cp_async_wait<EARLY ? 2 * DEPTH - 1 : 2 * DEPTH - 2>();
      __syncwarp();
      const uint32_t bits = seen[st];
      if (bits == 0) {  // (uniform) no key of the tile is seen
        if constexpr (EARLY) {
          copy(i + DEPTH, st, 0);
          copy(i + DEPTH, st, 1);
        }
        continue;
      }
      const uint8_t *kt = ring + st * STAGE, *vt = kt + SIDE;
      const uint32_t k_addr = ring_addr + st * STAGE, v_addr = k_addr + SIDE;
      // S^T: row u of the tile is key u, and key u + 8
      float s[NQ][4];
#pragma unroll
      for (int nq = 0; nq < NQ; nq++) s[nq][0] = s[nq][1] = s[nq][2] = s[nq][3] = 0.f;
      if constexpr (F32) {
        // The tensor cores cut each sum's last bits off: a chain for the large products of even dims, one for the odd
        // ones and one for the small products, added at the end.
        float part[NQ][3][4] = {};
#pragma unroll
        for (int x = 0; x < D / 16; x++) {
          const float4 k0 = *reinterpret_cast<const float4*>(kt + u * ROW + piece<true>(u, x * 4 + c, 0) * 16);
          const float4 k1 = *reinterpret_cast<const float4*>(kt + (u + 8) * ROW + piece<true>(u + 8, x * 4 + c, 0) * 16);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t ah[4], al[4];
            split_tf32(h ? k0.z : k0.x, ah[0], al[0]);
            split_tf32(h ? k1.z : k1.x, ah[1], al[1]);
            split_tf32(h ? k0.w : k0.y, ah[2], al[2]);
            split_tf32(h ? k1.w : k1.y, ah[3], al[3]);
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) {
              const uint4 t = q_terms[(nq * (D / 8) + x * 2 + h) * 32 + lane];
              mma_tf32(part[nq][2], al, t.x, t.y);
              mma_tf32(part[nq][2], ah, t.z, t.w);
              mma_tf32(part[nq][h], ah, t.x, t.y);
            }
          }
        }
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[nq][e] = part[nq][2][e] + (part[nq][0][e] + part[nq][1][e]);
      } else {
        const int r = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int x = 0; x < D / 16; x++) {
          uint32_t av[4];
          ldmatrix4<false>(av, k_addr + r * ROW + piece<false>(r, x * 2 + (lane >> 4), 0) * 16);
#pragma unroll
          for (int nq = 0; nq < NQ; nq++) mma_bf16(s[nq], av, qf[nq][x][0], qf[nq][x][1]);
        }
      }
      if (p.negative) {
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[nq][e] = -s[nq][e];
      }
      if (bits != 0xffffu) {
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (!((bits >> (u + (e >> 1) * 8)) & 1)) s[nq][e] = -INFINITY;
      }
      if constexpr (EARLY) {
        __syncwarp();
        copy(i + DEPTH, st, 0);
      }
      bool grow = false;
#pragma unroll
      for (int nq = 0; nq < NQ; nq++)
#pragma unroll
        for (int k = 0; k < 2; k++) grow = grow || fmaxf(s[nq][k], s[nq][2 + k]) * p.scale_log2 > m[nq][k] + 8.f;
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
          float corr[2];
#pragma unroll
          for (int k = 0; k < 2; k++) {
            float x = fmaxf(s[nq][k], s[nq][2 + k]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16)) * p.scale_log2;
            corr[k] = 1.f;
            if (x > m[nq][k]) {
              corr[k] = ex2_ftz(m[nq][k] - x);
              m[nq][k] = x;
            }
            l[nq][k] *= corr[k];
          }
#pragma unroll
          for (int t = 0; t < MTILES; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[nq][t][e] *= corr[e & 1];
        }
      }
      float w[NQ][4];
#pragma unroll
      for (int nq = 0; nq < NQ; nq++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          w[nq][e] = ex2_ftz(fmaf(s[nq][e], p.scale_log2, -m[nq][e & 1]));
          l[nq][e & 1] += w[nq][e];
        }
      if constexpr (EARLY) {
        cp_async_wait<2 * DEPTH - 1>();
        __syncwarp();
      }
      if (bits != 0xffffu) {  // hidden rows of v become zeros
#pragma unroll
        for (int j = 0; j < SIDE / 512; j++) {
          const int at = j * 32 + lane;
          if (!((bits >> (at / (ROW / 16))) & 1)) reinterpret_cast<uint4*>(ring + st * STAGE + SIDE)[at] = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      if constexpr (F32) {
        uint32_t bt[2][NQ][4];  // keys 8 h ..: a lane's are 8 h + 2 c and the next
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int nq = 0; nq < NQ; nq++) {
            // the 8 x 8 weights turned, 16 bits at a time
            const uint32_t w0 = __float_as_uint(w[nq][2 * h]), w1 = __float_as_uint(w[nq][2 * h + 1]);
            const uint32_t lo = transposed(__byte_perm(w0, w1, 0x5410)), hi = transposed(__byte_perm(w0, w1, 0x7632));
            split_tf32(__uint_as_float(__byte_perm(lo, hi, 0x5410)), bt[h][nq][0], bt[h][nq][2]);
            split_tf32(__uint_as_float(__byte_perm(lo, hi, 0x7632)), bt[h][nq][1], bt[h][nq][3]);
          }
#pragma unroll
        for (int x = 0; x < D / 32; x++) {  // dims 32 x + 4 u .. + 3: rows u, u + 8 of two tiles
          float4 v0[2], v1[2];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int r0 = h * 8 + c * 2;
            v0[h] = *reinterpret_cast<const float4*>(vt + r0 * ROW + piece<true>(r0, x * 8 + u, 1) * 16);
            v1[h] = *reinterpret_cast<const float4*>(vt + (r0 + 1) * ROW + piece<true>(r0 + 1, x * 8 + u, 1) * 16);
          }
#pragma unroll
          for (int t = 0; t < 2; t++) {
            float part[NQ][4] = {};  // of the tile's keys, added in f32's own rounding
#pragma unroll
            for (int h = 0; h < 2; h++) {
              uint32_t ah[4], al[4];
              split_tf32(t ? v0[h].z : v0[h].x, ah[0], al[0]);
              split_tf32(t ? v0[h].w : v0[h].y, ah[1], al[1]);
              split_tf32(t ? v1[h].z : v1[h].x, ah[2], al[2]);
              split_tf32(t ? v1[h].w : v1[h].y, ah[3], al[3]);
#pragma unroll
              for (int nq = 0; nq < NQ; nq++) mma_3tf32(part[nq], ah, al, bt[h][nq]);
            }
#pragma unroll
            for (int nq = 0; nq < NQ; nq++)
#pragma unroll
              for (int e = 0; e < 4; e++) o[nq][x * 2 + t][e] += part[nq][e];
          }
        }
      } else {
        uint32_t bw[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++)
#pragma unroll
          for (int h = 0; h < 2; h++) bw[nq][h] = transposed(pack_bf16x2(w[nq][2 * h], w[nq][2 * h + 1]));
        const int r = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
        for (int t = 0; t < MTILES; t++) {
          uint32_t av[4];
          ldmatrix4<true>(av, v_addr + r * ROW + piece<false>(r, t * 2 + ((lane >> 3) & 1), 1) * 16);
#pragma unroll
          for (int nq = 0; nq < NQ; nq++) mma_bf16(o[nq][t], av, bw[nq][0], bw[nq][1]);
        }
      }
      __syncwarp();  // every lane has read the stage that is copied into next
      if constexpr (EARLY) copy(i + DEPTH, st, 1);
    }
  }

  // The warps' O, maxima and sums into shared memory (the rings are done)
  cp_async_wait<0>();
  __syncthreads();
  constexpr int PITCH = MERGE_PITCH<D>;
  float* mem = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nq = 0; nq < NQ; nq++)
#pragma unroll
    for (int k = 0; k < 2; k++) {
      float sum = l[nq][k];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      float* to = mem + (warp * QROWS + nq * 8 + c * 2 + k) * PITCH;
#pragma unroll
      for (int t = 0; t < MTILES; t++) {
        if constexpr (F32) {  // dims 32 (t / 2) + 4 u + 2 (t % 2) and the next
          *reinterpret_cast<float2*>(to + (t / 2) * 32 + u * 4 + (t % 2) * 2) = make_float2(o[nq][t][k], o[nq][t][2 + k]);
        } else {
          to[t * 16 + u] = o[nq][t][k];
          to[t * 16 + u + 8] = o[nq][t][2 + k];
        }
      }
      if (u == 0) {
        to[D] = m[nq][k];
        to[D + 1] = sum;
      }
    }
  __syncthreads();
  auto finish = [&](int r, int d, float4 acc, float sum) {  // 4 values of row r of the tile from dim d on
    const int row = rtile * QROWS + r;
    if (row >= p.rows) return;
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // no key seen: zeros; NaN stays
    const int64_t at = ((int64_t)b * a.tq + row / p.group) * a.out_stride + (int64_t)(head * p.group + row % p.group) * dim + d;
    const float v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (d + e >= dim) break;
      if (a.out_dtype == WE_F32) store_out<WE_F32>(a.out, at + e, v[e]);
      else store_out<WE_BF16>(a.out, at + e, v[e]);
    }
  };
  merge_parts<D, QROWS, WARPS, CLUSTER>(mem, p.part, p.done, &last, unit, (int)gridDim.x / CLUSTER, runs, run, rank, finish);
}

// ---------------- host side ----------------
namespace {
struct CrossPlan {
  int dim, nq, row_tiles, cluster, runs, chunk;  // dim: rounded up to 64, 128 or 256
  int64_t units, part_floats;
};
CrossPlan cross_plan(const we_cross_desc& d, int sms) {
  CrossPlan q{};
  const int64_t rows = d.tq * (d.heads / d.kv_heads);
  const bool f32 = d.dtype == WE_F32;
  q.dim = d.dim <= 64 ? 64 : d.dim <= 128 ? 128 : 256;
  q.nq = rows <= 8 ? 1 : 2;
  q.row_tiles = (int)((rows + 8 * q.nq - 1) / (8 * q.nq));
  q.units = d.batch * d.kv_heads * q.row_tiles;
  // about one wave of runs (as the cached attention's plan), by the CTAs that fit an SM's shared memory
  const int per_sm = f32 ? (q.dim == 64 ? 4 : q.dim == 128 ? 3 : 1) : (q.dim == 64 ? 4 : q.dim == 128 ? 3 : 1);
  const int64_t slots = (int64_t)sms * per_sm - 8 * per_sm, tk = std::max<int64_t>(1, d.tk);
  // where the row tiles alone fill the SMs, a CTA takes all keys of its rows
  q.cluster = q.nq == 2 && q.units >= slots ? 1 : 8;
  // several runs only where they spare a CTA more than merging them costs, some 150 KB of keys and values: one query to 2048
  // keys of 12 heads of 128 8.4 us in one run and 9.5 in several, to 8192 20.4 and 16.0
  const int64_t alone = (tk + q.cluster - 1) / q.cluster, fit = std::max<int64_t>(1, slots / (q.units * q.cluster));
  const int64_t runs = (alone - alone / fit) * 2 * q.dim * (f32 ? 4 : 2) > 150000 ? fit : 1;
  const int64_t chunk = std::max<int64_t>(128, (alone + runs - 1) / runs);
  q.chunk = (int)((std::min<int64_t>(chunk, 0x4000000) + 15) / 16 * 16);
  q.runs = (int)((tk + (int64_t)q.chunk * q.cluster - 1) / ((int64_t)q.chunk * q.cluster));
  q.part_floats = q.runs > 1 ? q.units * q.runs * 8 * q.nq * (q.dim + 4) : 0;
  return q;
}

template <bool F32, int D, int NQ, int DEPTH, int CLUSTER>
cudaError_t cross_tile(const cross::Params& p, dim3 grid, cudaStream_t st) {
  auto kern = cross_tile_kernel<F32, D, NQ, DEPTH, CLUSTER>;
  constexpr int es = F32 ? 4 : 2;
  constexpr int ring = (F32 ? NQ * (D / 8) * 512 : 0) + cross::WARPS * DEPTH * 2 * cross::TILE * D * es;
  constexpr int merge = (cross::WARPS + 1) * 8 * NQ * MERGE_PITCH<D> * 4;
  constexpr int bytes = ring > merge ? ring : merge;
  const cudaError_t e = allow_smem(kern, bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(cross::THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CLUSTER;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  pdl_attribute(attr[1]);
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, p);
}
}  // namespace

void cross_tile_scratch(const we_cross_desc& d, int sms, int64_t* part_bytes, int64_t* units, int64_t* grid_y) {
  const CrossPlan q = cross_plan(d, sms);
  *part_bytes = q.part_floats * 4;
  *units = q.runs > 1 ? q.units : 0;
  *grid_y = d.kv_heads * q.row_tiles;
}

cudaError_t launch_cross_tile(const we_cross_desc& d, void* part, uint32_t* done, int sms, cudaStream_t st) {
  const CrossPlan q = cross_plan(d, sms);
  const bool f32 = d.dtype == WE_F32;
  const int es = f32 ? 4 : 2;
  cross::Params p{};
  p.d = d;
  p.group = (int)(d.heads / d.kv_heads);
  p.rows = (int)(d.tq * p.group);
  p.row_tiles = q.row_tiles;
  p.chunk = q.chunk;
  const uintptr_t kv = reinterpret_cast<uintptr_t>(d.k) | reinterpret_cast<uintptr_t>(d.v) |
                       (uintptr_t)(d.k_stride * es) | (uintptr_t)(d.v_stride * es) | (uintptr_t)(d.dim * es);
  p.wide_kv = (kv & 15) == 0;
  p.wide_q = ((reinterpret_cast<uintptr_t>(d.q) | (uintptr_t)(d.q_stride * es) | (uintptr_t)(d.dim * es)) & 3) == 0;
  p.scale_log2 = fabsf(d.scale) * 1.4426950408889634f;
  p.negative = d.scale < 0.f;
  p.part = static_cast<float*>(part);
  p.done = done;
  const dim3 grid((unsigned)(q.runs * q.cluster), (unsigned)(d.kv_heads * q.row_tiles), (unsigned)d.batch);
  cudaError_t e;
#define CROSS_CASE(F32, D, DEPTH)                                          \
  e = q.cluster == 1 ? cross_tile<F32, D, 2, DEPTH, 1>(p, grid, st)        \
      : q.nq == 1    ? cross_tile<F32, D, 1, DEPTH, 8>(p, grid, st)        \
                     : cross_tile<F32, D, 2, DEPTH, 8>(p, grid, st)
  if (f32) {
    if (q.dim == 64) CROSS_CASE(true, 64, 1);
    else if (q.dim == 128) CROSS_CASE(true, 128, 1);
    else CROSS_CASE(true, 256, 1);
  } else {
    if (q.dim == 64) CROSS_CASE(false, 64, 2);
    else if (q.dim == 128) CROSS_CASE(false, 128, 2);
    else CROSS_CASE(false, 256, 2);
  }
#undef CROSS_CASE
  return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace we
