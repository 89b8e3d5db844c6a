// Merging the parts of an attention whose keys are split over warps, the CTAs of a cluster, and clusters.
#pragma once
#include "common.cuh"
#include "tc_ptx.cuh"

namespace we {

// The maximum of a row that has seen no key: finite, so that a hidden score (-inf) less it is -inf, a weight of 0.
constexpr float NONE = -1e30f;

// Floats from one row to the next: D values, the maximum (in log2 units), the sum of weights, padding.
template <int D>
constexpr int MERGE_PITCH = D + 4;

// Parts of a row: values and the sum of weights, each relative to its own maximum, brought to the row's.
struct PartSum {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  __device__ __forceinline__ void add(float4 x, float m, float sum, float top) {
    const float f = ex2_ftz(m - top);
    v.x = fmaf(x.x, f, v.x);
    v.y = fmaf(x.y, f, v.y);
    v.z = fmaf(x.z, f, v.z);
    v.w = fmaf(x.w, f, v.w);
    l = fmaf(sum, f, l);
  }
};

// Called by every thread of a cluster of CLUSTER CTAs of WARPS warps, after a barrier behind the writes to `mem`:
//   mem    [WARPS][QROWS][MERGE_PITCH] of this CTA, and room for [QROWS][MERGE_PITCH] behind it
//   part   [units][all_runs][QROWS][MERGE_PITCH], done [units] (zero between calls), used when `runs` > 1 clusters share
//          a unit; `last` a word of shared memory
// finish(row, dim, 4 values, sum of weights) is called once for every 4 values of a row. The parts are added in the order
// of warps, CTAs and runs, so a call always gives the same bits.
template <int D, int QROWS, int WARPS, int CLUSTER, typename Finish>
__device__ __forceinline__ void merge_parts(float* mem, float* part_base, uint32_t* done, int* last, int unit, int all_runs,
                                            int runs, int run, int rank, Finish&& finish) {
  constexpr int PITCH = MERGE_PITCH<D>, THREADS = WARPS * 32;
  constexpr int ITEMS = QROWS * (D / 4) / CLUSTER;  // an eighth of the values for each CTA
  // the CTA's warps, into a place of its own
  float* cta = mem + WARPS * QROWS * PITCH;
  for (int x = threadIdx.x; x < QROWS * (D / 4); x += THREADS) {
    const int r = x / (D / 4), d = x % (D / 4) * 4;
    const float* from = mem + r * PITCH;
    float top = NONE;
#pragma unroll
    for (int w = 0; w < WARPS; w++) top = fmaxf(top, from[w * QROWS * PITCH + D]);
    PartSum sum;
#pragma unroll
    for (int w = 0; w < WARPS; w++, from += QROWS * PITCH)
      sum.add(*reinterpret_cast<const float4*>(from + d), from[D], from[D + 1], top);
    *reinterpret_cast<float4*>(cta + r * PITCH + d) = sum.v;
    if (d == 0) {
      cta[r * PITCH + D] = top;
      cta[r * PITCH + D + 1] = sum.l;
    }
  }
  __syncwarp();
  tc::cluster_sync_all();
  // the cluster's CTAs
  const uint32_t cta_addr = (uint32_t)__cvta_generic_to_shared(cta);
  auto remote = [](uint32_t addr, int cta_rank) { return tc::ld_cluster_f32(tc::map_rank(addr, cta_rank)); };
  float* part = runs > 1 ? part_base + (int64_t)unit * all_runs * (QROWS * PITCH) : nullptr;
  for (int x = threadIdx.x; x < ITEMS; x += THREADS) {
    const int r = (rank * ITEMS + x) / (D / 4), d = (rank * ITEMS + x) % (D / 4) * 4;
    const uint32_t at = cta_addr + 4 * (r * PITCH);
    float ms[CLUSTER], ls[CLUSTER], top = NONE;
#pragma unroll
    for (int w = 0; w < CLUSTER; w++) {
      ms[w] = remote(at + 4 * D, w);
      ls[w] = remote(at + 4 * (D + 1), w);
      top = fmaxf(top, ms[w]);
    }
    PartSum sum;
#pragma unroll
    for (int w = 0; w < CLUSTER; w++) {
      sum.add(tc::ld_cluster_f32x4(tc::map_rank(at + 4 * d, w)), ms[w], ls[w], top);
    }
    if (runs == 1) {
      finish(r, d, sum.v, sum.l);
    } else {
      float* to = part + ((int64_t)run * QROWS + r) * PITCH;
      *reinterpret_cast<float4*>(to + d) = sum.v;
      if (d == 0) {
        to[D] = top;
        to[D + 1] = sum.l;
      }
    }
  }
  if (runs > 1) __threadfence();
  __syncwarp();
  tc::cluster_sync_all();  // no CTA leaves while another reads its place; the cluster's part is written
  if (runs == 1) return;
  // the last cluster of the unit to get here merges all of its parts, in the order of the runs
  if (rank == 0 && threadIdx.x == 0) {
    __threadfence();  // behind the barrier: what the whole cluster has written is out before the count says so
    const int is_last = atomicAdd(done + unit, 1u) == (uint32_t)runs - 1u;
    if (is_last) done[unit] = 0u;
    __threadfence();
    const uint32_t flag = (uint32_t)__cvta_generic_to_shared(last);
    for (int w = 0; w < CLUSTER; w++)
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::map_rank(flag, w)), "r"(is_last) : "memory");
  }
  __syncwarp();
  tc::cluster_sync_all();
  if (!*last) return;
  __threadfence();
  // 4 neighbouring threads share the runs of one item
  for (int x = threadIdx.x / 4; x < ITEMS; x += THREADS / 4) {
    const int r = (rank * ITEMS + x) / (D / 4), d = (rank * ITEMS + x) % (D / 4) * 4, sub = threadIdx.x & 3;
    const float* from = part + (int64_t)r * PITCH;
    float top = NONE;
    for (int z = 0; z < runs; z++) top = fmaxf(top, from[(int64_t)z * (QROWS * PITCH) + D]);
    PartSum sum;
    const int z1 = runs * (sub + 1) / 4;
#pragma unroll 4
    for (int z = runs * sub / 4; z < z1; z++) {
      const float* row = from + (int64_t)z * (QROWS * PITCH);
      sum.add(*reinterpret_cast<const float4*>(row + d), row[D], row[D + 1], top);
    }
    const uint32_t quad = 0xfu << (threadIdx.x & 28);
#pragma unroll
    for (int w = 1; w < 4; w *= 2) {
      sum.v.x += __shfl_xor_sync(quad, sum.v.x, w);
      sum.v.y += __shfl_xor_sync(quad, sum.v.y, w);
      sum.v.z += __shfl_xor_sync(quad, sum.v.z, w);
      sum.v.w += __shfl_xor_sync(quad, sum.v.w, w);
      sum.l += __shfl_xor_sync(quad, sum.l, w);
    }
    if (sub == 0) finish(r, d, sum.v, sum.l);
  }
}

}  // namespace we
