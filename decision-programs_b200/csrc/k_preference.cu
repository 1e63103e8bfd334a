// Preference loss over pairs of items (paired log ratios): forward, and the
// gradient and curvature by every row's score.
//
// x = beta ((S_a - S_b) - (T_a - T_b)) with S, T an item's sums of scores and
// reference scores in fp32;  L = w ((1 - e) softplus(-x) + e softplus(x)).
// Sums run in an order that depends on the sizes alone, so that results do
// not change from run to run.
#include <string>
#include <vector>

#include "kernels.h"
#include "loss_math.cuh"

namespace dp {
namespace {

__device__ __forceinline__ float gap(const PairLoss& a, u64 r) { return a.ref ? a.score[r] - a.ref[r] : a.score[r]; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// An offset outside the rows is taken as the nearest end, so that no offset
// leads outside the arrays.
__device__ __forceinline__ u64 clamp_row(i64 b, u64 rows) { return b < 0 ? 0 : (u64(b) > rows ? rows : u64(b)); }

// One warp a pair.
__global__ void __launch_bounds__(256) k_preference(PairLoss a, u64 rows, const i64* begin, u64 pairs) {
  const u32 lane = threadIdx.x & 31;
  const u64 warps = u64(gridDim.x) * (blockDim.x >> 5);
  const u64 w0 = u64(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  for (u64 p = w0; p < pairs; p += warps) {
    const u64 b0 = begin ? clamp_row(begin[2 * p], rows) : 2 * p;
    const u64 b1 = begin ? clamp_row(begin[2 * p + 1], rows) : 2 * p + 1;
    const u64 b2 = begin ? clamp_row(begin[2 * p + 2], rows) : 2 * p + 2;
    float sa = 0.f, sb = 0.f;
    for (u64 r = b0 + lane; r < b1; r += 32) sa += gap(a, r);
    for (u64 r = b1 + lane; r < b2; r += 32) sb += gap(a, r);
    sa = warp_sum(sa);
    sb = warp_sum(sb);
    const float w = a.weight ? a.weight[p] : 1.f;
    float loss = 0.f, q = 0.f, h = 0.f;
    if (w != 0.f) {
      const PairTerms t = pair_terms(a.beta * (sa - sb), a.smoothing);
      loss = w * t.loss;
      q = w * (a.beta * t.slope);
      h = w * (a.beta * a.beta * t.bend);
    }
    h = item_hess(h);
    if (lane == 0) a.loss[p] = loss;
    for (u64 r = b0 + lane; r < b1; r += 32) {
      a.grad[r] = q;
      if (a.hess) a.hess[r] = h;
    }
    for (u64 r = b1 + lane; r < b2; r += 32) {
      a.grad[r] = -q;
      if (a.hess) a.hess[r] = h;
    }
  }
  // rows before the first item and after the last belong to no pair
  const u64 first = begin ? clamp_row(begin[0], rows) : 0, last = begin ? clamp_row(begin[2 * pairs], rows) : 2 * pairs;
  const u64 n = first + (rows - last);
  for (u64 i = u64(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += u64(gridDim.x) * blockDim.x) {
    const u64 r = i < first ? i : last + (i - first);
    a.grad[r] = 0.f;
    if (a.hess) a.hess[r] = item_hess(0.f);
  }
}

// One thread a row; a pair's loss is written by its preferred row.
__global__ void __launch_bounds__(256) k_pair_loss(PairLoss a, u64 rows, const u32* __restrict__ off,
                                                   const PairEntry* __restrict__ entry) {
  for (u64 r = u64(blockIdx.x) * blockDim.x + threadIdx.x; r < rows; r += u64(gridDim.x) * blockDim.x) {
    const float mine = gap(a, r);
    float g = 0.f, h = 0.f;
    for (u32 i = off[r]; i < off[r + 1]; ++i) {
      const PairEntry e = entry[i];
      const bool lost = e.partner >> 31;
      const float w = a.weight ? a.weight[e.pair] : 1.f;
      float loss = 0.f;
      if (w != 0.f) {
        const float other = gap(a, e.partner & 0x7fffffffu);
        const PairTerms t = pair_terms(a.beta * (lost ? other - mine : mine - other), a.smoothing);
        const float q = w * (a.beta * t.slope);
        loss = w * t.loss;
        g += lost ? -q : q;
        h += w * (a.beta * a.beta * t.bend);
      }
      if (!lost) a.loss[e.pair] = loss;
    }
    a.grad[r] = g;
    if (a.hess) a.hess[r] = item_hess(h);
  }
}

u32 blocks_for(u64 n, u64 per_block) {
  const u64 want = (n + per_block - 1) / per_block, cap = 148 * 64;
  return u32(want < 1 ? 1 : (want < cap ? want : cap));
}

}  // namespace

void launch_preference(const PairLoss& a, u64 rows, const i64* begin, u64 pairs, cudaStream_t s) {
  if (!rows && !pairs) return;
  k_preference<<<blocks_for(pairs, 8), 256, 0, s>>>(a, rows, begin, pairs);
  after_launch("preference loss");
}

void build_pair_plan(PairPlan& plan, u64 rows, const i32* pair_rows, u64 pairs, cudaStream_t s) {
  DP_CUDA(cudaGetDevice(&plan.device));
  plan.rows = rows;
  plan.pairs = pairs;
  std::vector<i32> list(2 * pairs);
  if (pairs)
    DP_CUDA(cudaMemcpyAsync(list.data(), pair_rows, list.size() * sizeof(i32), cudaMemcpyDeviceToHost, s));
  DP_CUDA(cudaStreamSynchronize(s));
  std::vector<u32> off(rows + 1, 0);
  for (u64 p = 0; p < pairs; ++p) {
    const i32 x = list[2 * p], y = list[2 * p + 1];
    if (x < 0 || y < 0 || u64(x) >= rows || u64(y) >= rows)
      fail("pair " + std::to_string(p) + " names a row outside [0, " + std::to_string(rows) + ")");
    if (x == y) fail("pair " + std::to_string(p) + " names one row twice");
    ++off[u64(x) + 1];
    ++off[u64(y) + 1];
  }
  for (u64 r = 0; r < rows; ++r) off[r + 1] += off[r];
  std::vector<PairEntry> entry(2 * pairs);
  std::vector<u32> at(off.begin(), off.end());
  for (u64 p = 0; p < pairs; ++p) {
    const u32 x = u32(list[2 * p]), y = u32(list[2 * p + 1]);
    entry[at[x]++] = PairEntry{y, u32(p)};
    entry[at[y]++] = PairEntry{x | 0x80000000u, u32(p)};
  }
  plan.off.resize(rows + 1);
  plan.entry.resize(2 * pairs);
  DP_CUDA(cudaMemcpy(plan.off.get(), off.data(), off.size() * sizeof(u32), cudaMemcpyHostToDevice));
  if (pairs)
    DP_CUDA(cudaMemcpy(plan.entry.get(), entry.data(), entry.size() * sizeof(PairEntry), cudaMemcpyHostToDevice));
}

void launch_pair_loss(const PairPlan& p, const PairLoss& a, cudaStream_t s) {
  if (!p.rows) return;
  k_pair_loss<<<blocks_for(p.rows, 256), 256, 0, s>>>(a, p.rows, p.off.get(), p.entry.get());
  after_launch("pair loss");
}

}  // namespace dp
