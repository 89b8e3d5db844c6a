// Cross attention with many queries on tcgen05: bf16, heads of 64 or 128.
//
// A CTA takes items of 128 rows, one after the other, over a kv head's keys in tiles of 128: rows are tokens x the kv head's
// group of heads, so that a group reads its keys once however few its tokens. Warp 0 brings Q and
// the K and V tiles by TMA, one thread of warp 1 issues S = Q K^T and O += P V (kind::f16, accumulators in TMEM, P read from
// TMEM over the first half of S's columns, V an MN-major operand as it is stored), warps 2 to 9 run the softmax, a thread one
// query row and one half of the tile's keys (the two exchange their maxima through shared memory).
// Text states are a few tiles, so an item is a few steps only and each step is a chain (S, softmax, P V): what keeps the
// tensor cores fed is a second CTA on the SM (256 TMEM columns and about 100 KB of shared memory each), and that a CTA's next
// item is under way while the last one is written: its Q, K and V are loaded and its first S computed by then.
// Hidden keys (past a length, or masked) have scores of -inf, and the softmax warps write zeros over their rows of V in
// shared memory before they hand P over, so that nothing of them reaches a product; tiles without any skip both.
// Calls whose items would leave SMs idle give each item to a cluster, its CTAs a share of the keys each, merged over
// distributed shared memory.
// P is rounded to bf16 (2^-9 each, sums in f32), as V is stored: kind::f16 takes both operands of one type.
// Measured in recorded graphs: 2 x 4096 queries x (512, 333) keys, 24 heads of 128: 69 us, 613 TFLOP/s (76 as single calls on
// inputs that were not read just before; 67.8 when a tile held one head's rows only); 2048 x 4096 keys 140 us (735 TFLOP/s),
// 180 us with a random mask; 128 x 4096 keys 22.7 us (64 without the clusters). A step of a CTA takes about 4600 cycles:
// from P to the next S 2000 (the products are 1024 of it, more when the other CTA's are in front), reading S and the maxima
// 500, exponentials 1650, P's way to TMEM 400. Storing each lane's row by itself took 10400 cycles an item; one CTA per item
// without the next one's loads and S in flight 87 us instead of 82.

#include <cudaTypedefs.h>

#include <algorithm>

#include "attn_merge.cuh"
#include "common.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace we {

namespace cf {
constexpr int B = 128;            // queries of a CTA, keys of a tile
constexpr int ATOM = B * 128;     // 128 rows of 64 bf16 (one swizzle-128B box)
constexpr int SOFTMAX_WARPS = 8;   // 4 row quarters x 2 halves of the keys (and of O's columns)
constexpr int THREADS = 64 + SOFTMAX_WARPS * 32;
constexpr uint32_t TMEM_COLS = 256, O_COL = 128;
constexpr float RESCALE_LOG2 = 8.f;

struct Params {
  int64_t tq, tk, out_stride, items;
  int kv_heads, group, span, q_tiles, splits;  // group: heads per kv head; span: tokens of an item (span * group rows);
                                               // items = batch * kv_heads * q_tiles; splits: CTAs per item
  float scale_log2;  // |scale| log2(e); with a negative scale the scores change sign as they are read
  void* out;
  int out_dtype;
  const int32_t* key_lengths;
  const uint8_t* key_mask;
  int negative;
  uint32_t* err;
};

template <int D>
struct Layout {
  static constexpr int STAGES = D == 64 ? 2 : 1, TILE = D / 64 * ATOM;
  static constexpr int Q = 0, K = TILE, V = K + STAGES * TILE, BARS = V + STAGES * TILE;
  static constexpr int NUM_BARS = 4 * STAGES + 8;                    // (a multiple of 2)
  static constexpr int RED = BARS + NUM_BARS * 8 + 16;               // row maxima of two tile parities and row sums, by halves
  static constexpr int BYTES = RED + 3 * 2 * B * 4 + 1024;
  static constexpr uint32_t IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(B >> 3) << 17) | ((uint32_t)(B >> 4) << 24);
  static constexpr uint32_t IDESC_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(B >> 4) << 24);
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t c0, int32_t c1, int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t c0, int32_t c1, int32_t c2,
                                            int32_t c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16_up(float lo, float hi) {  // non-negative, to nearest (ties up)
  return __byte_perm(__float_as_uint(lo) + 0x8000u, __float_as_uint(hi) + 0x8000u, 0x7632);
}
// Lane t of four holds pieces 0..3 of row t; afterwards piece t of rows 0..3.
__device__ __forceinline__ void transpose4(uint4 (&w)[4], int lane) {
  auto swap = [&](uint4& lo, uint4& hi, int bit) {  // the lane with the bit gives its lo for the other's hi
    const bool up = (lane & bit) != 0;
    uint4 x = up ? lo : hi;
    x.x = __shfl_xor_sync(0xffffffffu, x.x, bit);
    x.y = __shfl_xor_sync(0xffffffffu, x.y, bit);
    x.z = __shfl_xor_sync(0xffffffffu, x.z, bit);
    x.w = __shfl_xor_sync(0xffffffffu, x.w, bit);
    if (up) lo = x;
    else hi = x;
  };
  swap(w[0], w[1], 1);
  swap(w[2], w[3], 1);
  swap(w[0], w[2], 2);
  swap(w[1], w[3], 2);
}
// 64 bytes of each of the warp's 32 rows (lane = row); to: where rows 4 (lane / 4) + 0..3 go, values from `out`, or -1.
template <typename T>
__device__ __forceinline__ void store_quads(uint4 (&w)[4], T* out, const int64_t (&to)[4], int lane) {
  transpose4(w, lane);
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (to[e] >= 0) *reinterpret_cast<uint4*>(out + to[e] + (lane & 3) * (16 / (int)sizeof(T))) = w[e];
}
}  // namespace cf

template <int D, bool SPLIT>
__global__ void __launch_bounds__(cf::THREADS, 2)
    cross_flash_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const cf::Params p) {
  using namespace tc;
  using namespace cf;
  using L = Layout<D>;
  constexpr int NS = L::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem), bars = sbase + L::BARS;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::BARS + L::NUM_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const uint32_t MISC = bars + 8 * 4 * NS, Q_FULL = MISC, Q_EMPTY = MISC + 8, S_FULL = MISC + 16, P_FULL = MISC + 24,
                 O_DONE = MISC + 32, O_FREE = MISC + 40, DRAIN = MISC + 48;
  auto K_FULL = [&](int s) { return bars + 8u * s; };
  auto K_EMPTY = [&](int s) { return bars + 8u * (NS + s); };
  auto V_FULL = [&](int s) { return bars + 8u * (2 * NS + s); };
  auto V_EMPTY = [&](int s) { return bars + 8u * (3 * NS + s); };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; i++) {
      mbar_init(K_FULL(i), 1);
      mbar_init(K_EMPTY(i), 1);
      mbar_init(V_FULL(i), 1);
      mbar_init(V_EMPTY(i), 1);
    }
    mbar_init(Q_FULL, 1);
    mbar_init(Q_EMPTY, 1);
    mbar_init(S_FULL, 1);
    mbar_init(P_FULL, SOFTMAX_WARPS);
    mbar_init(O_DONE, 1);
    mbar_init(O_FREE, SOFTMAX_WARPS);
    mbar_init(DRAIN, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  // TMEM is taken only when the kernel before has ended, and the one after may start only when this CTA has its own: no CTA
  // then waits for columns that one of another kernel holds while it waits in turn.
  pdl_wait();
  if (warp == 1) tmem_alloc(smem_u32(tmem_holder), TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem = *tmem_holder;

  // The items of this CTA, in every role alike: query tile fastest, then heads, then entries. An item without keys takes part
  // in no barrier. `tiles` and `done` count the tiles and the items with keys so far: the parities of the barriers.
  // SPLIT: a cluster of p.splits CTAs has one item, each CTA its share of the tiles (from tile t0).
  struct Item {
    int q0, h, b, keys, t0, nt;  // first token, kv head
  };
  const int64_t first = SPLIT ? blockIdx.x / p.splits : blockIdx.x, step = SPLIT ? p.items : gridDim.x;
  auto item = [&](int64_t i) {
    Item x;
    x.q0 = (int)(i % p.q_tiles) * p.span;
    const int bh = (int)(i / p.q_tiles);
    x.h = bh % p.kv_heads;
    x.b = bh / p.kv_heads;
    x.keys = (int)p.tk;
    if (p.key_lengths) x.keys = max(0, min(x.keys, p.key_lengths[x.b]));
    x.t0 = 0;
    x.nt = (x.keys + B - 1) / B;
    if constexpr (SPLIT) {
      const int rank = (int)cluster_rank(), all = x.nt;
      x.t0 = (int)((int64_t)all * rank / p.splits);
      x.nt = (int)((int64_t)all * (rank + 1) / p.splits) - x.t0;
    }
    return x;
  };

  // Row r of an item: head r % group of the kv head's, token q0 + r / group. Its first value's place in out, -1: no row.
  const uint32_t recip = (65536u + p.group - 1) / p.group;  // r / group = r recip >> 16, exact for r < 128, group <= 128
  auto out_at = [&](const Item& x, int r) -> int64_t {
    const int t = (int)((r * recip) >> 16);
    if (t >= p.span || x.q0 + t >= p.tq) return -1;
    return ((int64_t)x.b * p.tq + x.q0 + t) * p.out_stride + ((int64_t)x.h * p.group + r - t * p.group) * D;
  };

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int tiles = 0, done = 0, k_issued = 0, v_issued = 0;
      for (int64_t i = first; i < p.items && ok; i += step) {
        const Item x = item(i);
        if (x.nt == 0) continue;
        auto load = [&](const CUtensorMap* map, uint32_t dst, uint32_t bar, int head, int row) {
          mbar_expect_tx(bar, L::TILE);
#pragma unroll
          for (int c = 0; c < D / 64; c++) tma_load_3d(dst + c * ATOM, map, bar, head * D + c * 64, row, x.b);
        };
        ok = wait_fast(Q_EMPTY, (done & 1) ^ 1u, abort_flag, p.err, DEV_ERR_TIMEOUT_PRODUCER, WAIT_LIMIT_NS, true);
        if (!ok) break;
        mbar_expect_tx(Q_FULL, (uint32_t)(p.span * p.group) * (D * 2));
#pragma unroll
        for (int c = 0; c < D / 64; c++) tma_load_4d(sbase + L::Q + c * ATOM, &tm_q, Q_FULL, c * 64, x.h * p.group, x.q0, x.b);
        done++;
        for (int j = 0; j < x.nt; j++, tiles++) {
          const int s = tiles % NS;
          const uint32_t free_parity = ((tiles / NS) & 1) ^ 1u;
          ok = wait_fast(K_EMPTY(s), free_parity, abort_flag, p.err, DEV_ERR_TIMEOUT_PRODUCER, WAIT_LIMIT_NS, true);
          if (!ok) break;
          load(&tm_k, sbase + L::K + s * L::TILE, K_FULL(s), x.h, (x.t0 + j) * B);
          k_issued = tiles + 1;
          ok = wait_fast(V_EMPTY(s), free_parity, abort_flag, p.err, DEV_ERR_TIMEOUT_PRODUCER, WAIT_LIMIT_NS, true);
          if (!ok) break;
          load(&tm_v, sbase + L::V + s * L::TILE, V_FULL(s), x.h, (x.t0 + j) * B);
          v_issued = tiles + 1;
        }
      }
      if (!ok) {  // the copies already issued land before the CTA exits
        if (done > 0) wait_fast(Q_FULL, (done - 1) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_DRAIN, DRAIN_LIMIT_NS, false);
        for (int t = max(0, k_issued - NS); t < k_issued; t++)
          wait_fast(K_FULL(t % NS), (t / NS) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_DRAIN, DRAIN_LIMIT_NS, false);
        for (int t = max(0, v_issued - NS); t < v_issued; t++)
          wait_fast(V_FULL(t % NS), (t / NS) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_DRAIN, DRAIN_LIMIT_NS, false);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = true;
      int tiles = 0, done = 0;
      auto s_mma = [&](int t) -> bool {  // S(t) = Q K_t^T
        const int s = t % NS;
        if (!wait_fast(K_FULL(s), (t / NS) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA, WAIT_LIMIT_NS, true)) return false;
        tc_fence_after();
        const uint64_t qdesc = sw128_desc(sbase + L::Q), kdesc = sw128_desc(sbase + L::K + s * L::TILE);
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++) {  // boxes of 64 dims, 4 products of 16 each
          const uint64_t off = (uint64_t)((kk >> 2) * (ATOM >> 4) + (kk & 3) * 2);
          umma<true>(tmem, qdesc + off, kdesc + off, L::IDESC_S, kk != 0);
        }
        umma_commit(S_FULL);
        umma_commit(K_EMPTY(s));
        return true;
      };
      for (int64_t i = first; i < p.items && ok; i += step) {
        const Item x = item(i);
        if (x.nt == 0) continue;
        ok = wait_fast(Q_FULL, done & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA, WAIT_LIMIT_NS, true) && s_mma(tiles);
        for (int j = 0; j < x.nt && ok; j++, tiles++) {
          const int s = tiles % NS;
          if (j + 1 == x.nt) umma_commit(Q_EMPTY);  // the item's last S is issued: Q is free once it is done
          // the item before must be out of O before this one's first product overwrites it
          ok = wait_spin(P_FULL, tiles & 1, 4096, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA, WAIT_LIMIT_NS, true) &&
               wait_fast(V_FULL(s), (tiles / NS) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA, WAIT_LIMIT_NS, true) &&
               (j > 0 || wait_fast(O_FREE, (done & 1) ^ 1u, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA, WAIT_LIMIT_NS, true));
          if (!ok) break;
          tc_fence_after();
          const uint64_t vdesc = mn_sw128_desc(sbase + L::V + s * L::TILE, ATOM);
#pragma unroll
          for (int kk = 0; kk < 8; kk++)  // 128 keys: 8 products of 16 (16 rows of 128 bytes of V, 8 columns of P)
            umma_tmem_a(tmem + O_COL, tmem + (uint32_t)(kk * 8), vdesc + (uint64_t)(kk * (16 * 128 >> 4)), L::IDESC_O, (j | kk) != 0);
          umma_commit(V_EMPTY(s));
          if (j + 1 < x.nt) ok = s_mma(tiles + 1);
          else umma_commit(O_DONE);
        }
        done++;
      }
      // every product this thread issued completes before TMEM is freed
      umma_commit(DRAIN);
      wait_fast(DRAIN, 0, abort_flag, p.err, DEV_ERR_TIMEOUT_DRAIN, DRAIN_LIMIT_NS, false);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2, r = quarter * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16), o_addr = lane_addr + O_COL + half * (D / 2);
    const uint32_t pair_bar = 1u + quarter;  // the two warps of a row quarter
    float* red = reinterpret_cast<float*>(smem + L::RED);  // [2 parities][2 halves][128 rows], then [2 halves][128 rows] of sums
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true, stop = false;  // ok: of this warp; the two warps of a pair only leave together, by a barrier's answer
    int tiles = 0, done = 0;
    for (int64_t i = first; i < p.items; i += step) {
      const Item it = item(i);
      const uint8_t* mask = p.key_mask ? p.key_mask + (int64_t)it.b * p.tk : nullptr;
      float m = NONE, l = 0.f;
      for (int j = 0; j < it.nt; j++, tiles++) {
        // which of this half's keys are seen
        const int key = (it.t0 + j) * B + half * 64 + lane, s = tiles % NS;
        const uint32_t w0 = __ballot_sync(0xffffffffu, key < it.keys && (!mask || mask[key] != 0));
        const uint32_t w1 = __ballot_sync(0xffffffffu, key + 32 < it.keys && (!mask || mask[key + 32] != 0));
        const bool whole = (w0 & w1) == 0xffffffffu;
        ok = ok && wait_fast(S_FULL, tiles & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_EPILOGUE, WAIT_LIMIT_NS, true);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        uint32_t sc[64];
        tmem_ld32_async(lane_addr + half * 64, *reinterpret_cast<uint32_t(*)[32]>(sc));
        tmem_ld32_async(lane_addr + half * 64 + 32, *reinterpret_cast<uint32_t(*)[32]>(sc + 32));
        tmem_wait_ld(*reinterpret_cast<uint32_t(*)[32]>(sc));
        reg_fence(*reinterpret_cast<uint32_t(*)[32]>(sc + 32));
        if (p.negative) {
#pragma unroll
          for (int c = 0; c < 64; c++) sc[c] ^= 0x80000000u;
        }
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 32; c++) {
            if (!((w0 >> c) & 1)) sc[c] = 0xff800000u;
            if (!((w1 >> c) & 1)) sc[32 + c] = 0xff800000u;
          }
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; c++) mx[c] = fmaxf(__uint_as_float(sc[2 * c]), __uint_as_float(sc[2 * c + 1]));
#pragma unroll
        for (int c = 8; c < 64; c += 8)
#pragma unroll
          for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], __uint_as_float(sc[c + 2 * e]), __uint_as_float(sc[c + 2 * e + 1]));
        float* rm = red + (tiles & 1) * 2 * B;
        rm[half * B + r] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        // the exchange also ANDs the two warps' wait results, so that a pair always leaves the loop together, and orders both
        // halves' reads of S before the writes of P over its columns
        if (!named_bar_and(pair_bar, 64, ok)) {
          stop = true;
          break;
        }
        const float top = fmaxf(rm[r], rm[B + r]) * p.scale_log2;
        float corr = 1.f;
        const bool grow = top > m + RESCALE_LOG2;
        if (grow) {
          corr = ex2_ftz(m - top);
          l *= corr;
          m = top;
        }
        const float2 nm2 = make_float2(-m, -m);
        float2 sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 32; e++) {
          const float2 x = __ffma2_rn(make_float2(__uint_as_float(sc[2 * e]), __uint_as_float(sc[2 * e + 1])), sc2, nm2);
          const float2 w = make_float2(ex2_ftz(x.x), ex2_ftz(x.y));
          sum[e & 3] = __fadd2_rn(sum[e & 3], w);
          pk[e] = pack_bf16_up(w.x, w.y);
        }
        tmem_st32(lane_addr + half * 32, pk);
        l += ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y)) + ((sum[2].x + sum[2].y) + (sum[3].x + sum[3].y));
        // O is scaled for the old maximum (P V of the tile before is done: its commit came before S's)
        if (__any_sync(0xffffffffu, grow && j > 0)) {
#pragma unroll
          for (int c = 0; c < D / 64; c++) {
            uint32_t o[32];
            tmem_ld32(o_addr + c * 32, o);
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
            tmem_st32(o_addr + c * 32, o);
          }
        }
        if (!whole) {  // zeros over the hidden keys' rows of V (here by now): a warp 16 of its half's rows
          ok = ok && wait_fast(V_FULL(s), (tiles / NS) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_EPILOGUE, WAIT_LIMIT_NS, true);
          ok = __all_sync(0xffffffffu, ok);
          uint8_t* v = smem + L::V + s * L::TILE + (half * 64 + quarter * 16) * 128;
          const uint32_t hidden = ~(quarter < 2 ? w0 : w1) >> ((quarter & 1) * 16);
          if (ok) {
#pragma unroll
            for (int at = lane; at < 16 * 8; at += 32)
              if ((hidden >> (at >> 3)) & 1)
#pragma unroll
                for (int c = 0; c < D / 64; c++) *reinterpret_cast<uint4*>(v + c * ATOM + at * 16) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        tmem_st_wait();  // P (and O) are in TMEM before the products read them
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(P_FULL);
      }
      if (stop) break;
      // the row's sum over both halves; the second barrier keeps the next item's sums behind these reads
      float* row_sum = red + 4 * B;
      row_sum[half * B + r] = l;
      if (it.nt > 0) ok = ok && wait_fast(O_DONE, done & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_EPILOGUE, WAIT_LIMIT_NS, true);
      ok = __all_sync(0xffffffffu, ok);
      if (!named_bar_and(pair_bar, 64, ok)) break;
      tc_fence_after();
      l = row_sum[r] + row_sum[B + r];
      if constexpr (SPLIT) {  // this CTA's part of the rows, for the cluster's merge (K and V are read by now)
        if (half == 0) {
          red[r] = m;
          red[B + r] = l;
        }
#pragma unroll
        for (int c = 0; c < D / 64; c++) {
          uint32_t o[32];
          if (it.nt > 0) {
            tmem_ld32(o_addr + c * 32, o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = 0;
          }
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const int piece = (half * (D / 8) + c * 8 + e) ^ (r & 7);
            *reinterpret_cast<uint4*>(smem + L::K + r * (D * 4) + piece * 16) =
                make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
        break;
      }
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key seen: zeros; NaN stays
      int64_t to[4];  // where the four rows go that this lane stores pieces of, or -1
#pragma unroll
      for (int e = 0; e < 4; e++) {
        to[e] = out_at(it, quarter * 32 + (lane & ~3) + e);
        if (to[e] >= 0) to[e] += half * (D / 2);
      }
#pragma unroll
      for (int c = 0; c < D / 64; c++) {
        uint32_t o[32];
        if (it.nt > 0) {
          tmem_ld32(o_addr + c * 32, o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; e++) o[e] = 0;
        }
        if (c + 1 == D / 64 && it.nt > 0) {  // this warp has read its part of O
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(O_FREE);
        }
        // 16-byte pieces of the lanes' rows are exchanged among four lanes, so that a store writes 64 bytes of a row: with
        // each lane storing its own row an item took 10400 cycles to write, of about 29000
        if (p.out_dtype == WE_BF16) {
          uint4 w[4];
#pragma unroll
          for (int e = 0; e < 4; e++)
            w[e] = make_uint4(pack_bf16x2(__uint_as_float(o[8 * e]) * inv, __uint_as_float(o[8 * e + 1]) * inv),
                              pack_bf16x2(__uint_as_float(o[8 * e + 2]) * inv, __uint_as_float(o[8 * e + 3]) * inv),
                              pack_bf16x2(__uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 5]) * inv),
                              pack_bf16x2(__uint_as_float(o[8 * e + 6]) * inv, __uint_as_float(o[8 * e + 7]) * inv));
          store_quads(w, static_cast<uint16_t*>(p.out) + c * 32, to, lane);
        } else {
#pragma unroll
          for (int i2 = 0; i2 < 2; i2++) {
            uint4 w[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int at = i2 * 16 + 4 * e;
              w[e] = make_uint4(__float_as_uint(__uint_as_float(o[at]) * inv), __float_as_uint(__uint_as_float(o[at + 1]) * inv),
                                __float_as_uint(__uint_as_float(o[at + 2]) * inv), __float_as_uint(__uint_as_float(o[at + 3]) * inv));
            }
            store_quads(w, static_cast<float*>(p.out) + c * 32 + i2 * 16, to, lane);
          }
        }
      }
      named_bar_sync(pair_bar, 64);
      if (it.nt > 0) done++;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
  if constexpr (SPLIT) {  // each CTA joins the parts of its share of the rows, always in the same order
    __syncwarp();
    cluster_sync_all();
    const Item x = item(first);
    const int rows = B / p.splits;
    for (int at = threadIdx.x; at < rows * (D / 4); at += THREADS) {
      const int row = (int)cluster_rank() * rows + at / (D / 4), piece = at % (D / 4);
      const int64_t to = out_at(x, row);
      if (to < 0) break;
      float top = NONE;
      for (int c = 0; c < p.splits; c++) top = fmaxf(top, ld_cluster_f32(map_rank(sbase + L::RED + row * 4, c)));
      PartSum sum;
      for (int c = 0; c < p.splits; c++)
        sum.add(ld_cluster_f32x4(map_rank(sbase + L::K + row * (D * 4) + (piece ^ (row & 7)) * 16, c)),
                ld_cluster_f32(map_rank(sbase + L::RED + row * 4, c)),
                ld_cluster_f32(map_rank(sbase + L::RED + (B + row) * 4, c)), top);
      const float l = sum.l, inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      const int64_t o = to + piece * 4;
      if (p.out_dtype == WE_BF16)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + o) =
            make_uint2(pack_bf16x2(sum.v.x * inv, sum.v.y * inv), pack_bf16x2(sum.v.z * inv, sum.v.w * inv));
      else
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + o) =
            make_float4(sum.v.x * inv, sum.v.y * inv, sum.v.z * inv, sum.v.w * inv);
    }
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while another reads from it
  }
}

// ---------------- host side ----------------
namespace {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn_cross() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }
  return fn;
}
// [batch, tq, heads, D] of bf16, tokens `stride` values apart, in boxes of 64 values of `group` heads of `span` tokens
bool cross_q_map(CUtensorMap* map, const we_cross_desc& d, int group, int span) {
  auto fn = encode_fn_cross();
  if (!fn) return false;
  cuuint64_t dims[4] = {(cuuint64_t)d.dim, (cuuint64_t)d.heads, (cuuint64_t)d.tq, (cuuint64_t)d.batch};
  cuuint64_t strides[3] = {(cuuint64_t)(d.dim * 2), (cuuint64_t)(d.q_stride * 2), (cuuint64_t)(d.tq * d.q_stride * 2)};
  cuuint32_t box[4] = {64, (cuuint32_t)group, (cuuint32_t)span, 1}, estr[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(d.q), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// [batch, rows, cols] of bf16, rows `stride` values apart, in boxes of 64 columns x 128 rows with 128-byte swizzle
bool cross_map(CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t batch, int64_t stride) {
  auto fn = encode_fn_cross();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
  cuuint64_t strides[2] = {(cuuint64_t)(stride * 2), (cuuint64_t)(rows * stride * 2)};
  cuuint32_t box[3] = {64, cf::B, 1}, estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
cudaError_t cross_flash(const we_cross_desc& d, uint32_t* err, int sms, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  const int group = (int)(d.heads / d.kv_heads), span = cf::B / group;
  if (!cross_q_map(&mq, d, group, span) ||
      !cross_map(&mk, d.k, d.kv_heads * D, d.tk, d.batch, d.k_stride) ||
      !cross_map(&mv, d.v, d.kv_heads * D, d.tk, d.batch, d.v_stride))
    return cudaErrorNotSupported;
  const int64_t q_tiles = (d.tq + span - 1) / span, items = q_tiles * d.kv_heads * d.batch;
  // CTAs that would be idle take a share of the keys (powers of two up to 8 a cluster, a tile of keys each at the least; 24
  // CTAs fewer than two an SM, because clusters of 8 leave some places of a GPC empty)
  const int64_t tiles = (d.tk + cf::B - 1) / cf::B;
  int splits = 1;
  while (splits < 8 && items * splits * 2 <= 2 * sms - 24 && splits * 2 <= tiles) splits *= 2;
  cf::Params p{d.tq, d.tk, d.out_stride, items, (int)d.kv_heads, group, span, (int)q_tiles, splits,
               fabsf(d.scale) * 1.4426950408889634f, d.out, d.out_dtype, d.key_lengths, d.key_mask, d.scale < 0.f, err};
  constexpr int bytes = cf::Layout<D>::BYTES;
  const auto kernel = splits > 1 ? cross_flash_kernel<D, true> : cross_flash_kernel<D, false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(splits > 1 ? items * splits : std::min<int64_t>(items, 2 * sms)));
  cfg.blockDim = dim3(cf::THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  pdl_attribute(attr[0]);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, kernel, mq, mk, mv, p);
  return e == cudaSuccess ? cudaGetLastError() : e;
}
}  // namespace

// Whether launch_cross_flash takes the call: types, head size, 16-byte rows, sizes of a tensor map.
bool cross_flash_supported(const we_cross_desc& d) {
  if (d.dtype != WE_BF16 || (d.dim != 64 && d.dim != 128) || d.tk < 1 || d.heads / d.kv_heads > cf::B) return false;
  const int64_t os = d.out_dtype == WE_F32 ? 4 : 2;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(d.q) | reinterpret_cast<uintptr_t>(d.k) | reinterpret_cast<uintptr_t>(d.v) |
                         reinterpret_cast<uintptr_t>(d.out) | (uintptr_t)(d.q_stride * 2) | (uintptr_t)(d.k_stride * 2) |
                         (uintptr_t)(d.v_stride * 2) | (uintptr_t)(d.out_stride * os);
  const int64_t most = (int64_t)1 << 38;  // bytes from one batch entry to the next: below the map's 2^40
  return (bits & 15) == 0 && d.tq * d.q_stride < most && d.tk * d.k_stride < most && d.tk * d.v_stride < most;
}

cudaError_t launch_cross_flash(const we_cross_desc& d, uint32_t* err, int sms, cudaStream_t st) {
  return d.dim == 64 ? cross_flash<64>(d, err, sms, st) : cross_flash<128>(d, err, sms, st);
}

}  // namespace we
