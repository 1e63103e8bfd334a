// Preference loss over pairs of items (paired log ratios): forward, and the
// gradient and curvature by every row's score.
//
// x = beta ((S_a - S_b) - (T_a - T_b)) with S, T an item's sums of scores and
// reference scores in fp32;  L = w ((1 - e) softplus(-x) + e softplus(x)).
// Sums run in an order that depends on the sizes alone, so that results do
// not change from run to run: no floating-point atomics.
#include <string>

#include "kernels.h"
#include "loss_math.cuh"

namespace dp {
namespace {

constexpr u32 kSMs = 148;

__device__ __forceinline__ float gap(const PairLoss& a, u64 r) { return a.ref ? a.score[r] - a.ref[r] : a.score[r]; }

// Loss, gradient by the preferred item's score, curvature of one pair.
struct PairResult {
  float loss, q, h;
};
__device__ __forceinline__ PairResult pair_result(const PairLoss& a, float difference, float w) {
  PairResult o{0.f, 0.f, 0.f};
  if (w != 0.f) {
    const PairTerms t = pair_terms(a.beta * difference, a.smoothing);
    o.loss = w * t.loss;
    o.q = w * (a.beta * t.slope);
    o.h = w * (a.beta * a.beta * t.bend);
  }
  return o;
}

// ---- consecutive items ------------------------------------------------------
// Every row an item: a thread takes pairs of rows side by side.  Bound by memory:
// 2M rows in 1M pairs, gradient and curvature, 5.5 us (28 MB, part of it from L2).
template <bool kWide>
__global__ void __launch_bounds__(256) k_preference_rows(PairLoss a, u64 rows, u64 pairs) {
  const u64 step = u64(gridDim.x) * blockDim.x, first = u64(blockIdx.x) * blockDim.x + threadIdx.x;
  for (u64 p = first; p < pairs; p += step) {
    float sa, sb;
    if constexpr (kWide) {
      const float2 s = reinterpret_cast<const float2*>(a.score)[p];
      const float2 t = a.ref ? reinterpret_cast<const float2*>(a.ref)[p] : make_float2(0.f, 0.f);
      sa = a.ref ? s.x - t.x : s.x;
      sb = a.ref ? s.y - t.y : s.y;
    } else {
      sa = gap(a, 2 * p);
      sb = gap(a, 2 * p + 1);
    }
    const PairResult o = pair_result(a, sa - sb, a.weight ? a.weight[p] : 1.f);
    a.loss[p] = o.loss;
    const float h = item_hess(o.h);
    if constexpr (kWide) {
      reinterpret_cast<float2*>(a.grad)[p] = make_float2(o.q, -o.q);
      if (a.hess) reinterpret_cast<float2*>(a.hess)[p] = make_float2(h, h);
    } else {
      a.grad[2 * p] = o.q;
      a.grad[2 * p + 1] = -o.q;
      if (a.hess) a.hess[2 * p] = a.hess[2 * p + 1] = h;
    }
  }
  for (u64 r = 2 * pairs + first; r < rows; r += step) {  // rows of no pair
    a.grad[r] = 0.f;
    if (a.hess) a.hess[r] = item_hess(0.f);
  }
}

template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int U>
__device__ __forceinline__ float span_sum(const PairLoss& a, u64 b, u64 e, u64 first, u64 step) {
  float s[U], v[U];
#pragma unroll
  for (int i = 0; i < U; ++i) s[i] = 0.f;
  u64 r = b + first;
  for (; r + (U - 1) * step < e; r += U * step) {
#pragma unroll
    for (int i = 0; i < U; ++i) v[i] = gap(a, r + i * step);
#pragma unroll
    for (int i = 0; i < U; ++i) s[i] += v[i];
  }
  for (; r < e; r += step) s[0] += gap(a, r);
#pragma unroll
  for (int d = U / 2; d > 0; d /= 2)
#pragma unroll
    for (int i = 0; i < d; ++i) s[i] += s[i + d];
  return s[0];
}
__device__ __forceinline__ void span_fill(const PairLoss& a, u64 b, u64 e, u64 first, u64 step, float q, float h) {
#pragma unroll 4
  for (u64 r = b + first; r < e; r += step) {
    a.grad[r] = q;
    if (a.hess) a.hess[r] = h;
  }
}
// An offset outside the rows is taken as the nearest end, so that no offset
// leads outside the arrays.
__device__ __forceinline__ u64 clamp_row(i64 b, u64 rows) { return b < 0 ? 0 : (u64(b) > rows ? rows : u64(b)); }
// Rows before the first item and after the last belong to no pair.
__device__ __forceinline__ void fill_outside(const PairLoss& a, u64 rows, const i64* begin, u64 pairs) {
  const u64 first = clamp_row(begin[0], rows), last = clamp_row(begin[2 * pairs], rows);
  const u64 me = u64(blockIdx.x) * blockDim.x + threadIdx.x, step = u64(gridDim.x) * blockDim.x;
  span_fill(a, 0, first, me, step, 0.f, item_hess(0.f));
  span_fill(a, last, rows, me, step, 0.f, item_hess(0.f));
}

// Sums of v over the block's threads, the same in each of them.
template <int kWarps>
__device__ __forceinline__ float2 block_sums(float2 v, float2* part) {
  v.x = lanes_sum<32>(v.x);
  v.y = lanes_sum<32>(v.y);
  __syncthreads();  // (the last call's parts have been read)
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[threadIdx.x & (kWarps - 1)];
  return make_float2(lanes_sum<kWarps>(v.x), lanes_sum<kWarps>(v.y));
}

// Pairs far longer than the others of their call, which one thread or a few
// lanes would take while the device waits, and sum in long chains: the whole
// block takes them one after another (100,000 short pairs and one item of a
// million rows: 258 us, by one thread 16.9 ms).  What only such pairs need is
// kept out of the kernels' own code, whose registers it would take.
struct LongPair {
  u64 p, b0, b1, b2;
};
// Rows that one lane of a pair takes, 64 loads of four rows one after another.
constexpr u64 kLaneRows = 256;
template <int kThreads>
__device__ __forceinline__ void take_long_pairs(const PairLoss& a, const LongPair* list, u32 n) {
  __shared__ float2 part[kThreads / 32];
  for (u32 i = 0; i < n; ++i) {
    const LongPair x = list[i];
    const float2 s = block_sums<kThreads / 32>(make_float2(span_sum<8>(a, x.b0, x.b1, threadIdx.x, kThreads),
                                                           span_sum<8>(a, x.b1, x.b2, threadIdx.x, kThreads)), part);
    const PairResult o = pair_result(a, s.x - s.y, a.weight ? a.weight[x.p] : 1.f);
    const float h = item_hess(o.h);
    if (threadIdx.x == 0) a.loss[x.p] = o.loss;
    span_fill(a, x.b0, x.b1, threadIdx.x, kThreads, o.q, h);
    span_fill(a, x.b1, x.b2, threadIdx.x, kThreads, -o.q, h);
  }
}

// Items of a few rows: a block stages the rows of 256 pairs in shared memory,
// a thread takes a pair, and the gradients go out as the scores came in, in
// whole lines.  (4M rows in 1M pairs: 118 us by 8 lanes a pair.)  Blocks whose
// rows do not fit take their pairs from memory, each by a thread, a warp or the
// block as its length asks.
constexpr u32 kPairBlock = 256, kStageRows = 4096;
__device__ __noinline__ void take_unstaged_pairs(const PairLoss& call, u64 rows, const i64* begin, u64 pairs, LongPair* list, u32* longs) {
  const PairLoss a = call;
  const u64 p = u64(blockIdx.x) * kPairBlock + threadIdx.x;
  const bool in = p < pairs;
  const u64 b0 = in ? clamp_row(begin[2 * p], rows) : 0, b1 = in ? clamp_row(begin[2 * p + 1], rows) : 0,
            b2 = in ? clamp_row(begin[2 * p + 2], rows) : 0, n = b2 - b0;
  const float w = in && a.weight ? a.weight[p] : 1.f;
  if (threadIdx.x == 0) *longs = 0;
  __syncthreads();
  // (a warp takes its longer pairs one after another; many of them, unless very
  // long, go by a thread each: 300,000 pairs of lognormal lengths in ascending
  // order 109 us, without 118)
  const bool many = __popc(__ballot_sync(0xffffffffu, n > kLaneRows)) > 12;
  const u64 alone = many ? 4 * kLaneRows : kLaneRows;
  if (in && n <= alone) {
    const PairResult o = pair_result(a, span_sum<4>(a, b0, b1, 0, 1) - span_sum<4>(a, b1, b2, 0, 1), w);
    const float h = item_hess(o.h);
    a.loss[p] = o.loss;
    span_fill(a, b0, b1, 0, 1, o.q, h);
    span_fill(a, b1, b2, 0, 1, -o.q, h);
  }
  const bool whole = n > 32 * kLaneRows;
  if (whole) list[atomicAdd(longs, 1u)] = LongPair{p, b0, b1, b2};
  const u32 lane = threadIdx.x & 31;
  for (u32 todo = __ballot_sync(0xffffffffu, n > alone && !whole); todo; todo &= todo - 1) {
    const int from = __ffs(int(todo)) - 1;
    const u64 c0 = __shfl_sync(0xffffffffu, b0, from), c1 = __shfl_sync(0xffffffffu, b1, from),
              c2 = __shfl_sync(0xffffffffu, b2, from);
    const float sa = lanes_sum<32>(span_sum<8>(a, c0, c1, lane, 32)), sb = lanes_sum<32>(span_sum<8>(a, c1, c2, lane, 32));
    const PairResult o = pair_result(a, sa - sb, __shfl_sync(0xffffffffu, w, from));
    const float h = item_hess(o.h);
    if (int(lane) == from) a.loss[p] = o.loss;
    span_fill(a, c0, c1, lane, 32, o.q, h);
    span_fill(a, c1, c2, lane, 32, -o.q, h);
  }
  __syncthreads();
  take_long_pairs<kPairBlock>(a, list, *longs);
}
__global__ void __launch_bounds__(kPairBlock, 6) k_preference_staged(const __grid_constant__ PairLoss a, u64 rows, const i64* begin, u64 pairs) {
  __shared__ __align__(16) float stage[kStageRows];
  __shared__ float stage_h[kStageRows];
  __shared__ u32 longs;
  const u64 p0 = u64(blockIdx.x) * kPairBlock, p1 = min(pairs, p0 + kPairBlock), p = p0 + threadIdx.x;
  const u64 r0 = clamp_row(begin[2 * p0], rows), r1 = clamp_row(begin[2 * p1], rows);
  const bool in = p < p1;
  const u64 b0 = in ? clamp_row(begin[2 * p], rows) : 0, b1 = in ? clamp_row(begin[2 * p + 1], rows) : 0,
            b2 = in ? clamp_row(begin[2 * p + 2], rows) : 0;
  const float w = in && a.weight ? a.weight[p] : 1.f;
  const bool room = r1 >= r0 && r1 - r0 <= kStageRows;
  const u32 n = room ? u32(r1 - r0) : 0;
  for (u32 i = threadIdx.x; i < n; i += kPairBlock) stage[i] = gap(a, r0 + i);
  // One answer for the block, since it decides on the barriers below: were the
  // offsets written while the kernel runs, the results would be of no use, but
  // every thread would still come to the same barriers.
  if (__syncthreads_and(room)) {
    // (offsets out of order lead outside a pair's own rows, not outside the stage)
    auto local = [&](u64 b) { return b <= r0 ? 0u : u32(min(u64(n), b - r0)); };
    const u32 c0 = local(b0), c1 = local(b1), c2 = local(b2);
    float sa = 0.f, sb = 0.f;
    for (u32 i = c0; i < c1; ++i) sa += stage[i];
    for (u32 i = c1; i < c2; ++i) sb += stage[i];
    const PairResult o = pair_result(a, sa - sb, w);
    const float h = item_hess(o.h);
    if (in) a.loss[p] = o.loss;
    __syncthreads();  // (every sum has been taken)
    if (in) {
      for (u32 i = c0; i < c1; ++i) { stage[i] = o.q; stage_h[i] = h; }
      for (u32 i = c1; i < c2; ++i) { stage[i] = -o.q; stage_h[i] = h; }
    }
    __syncthreads();
    for (u32 i = threadIdx.x; i < n; i += kPairBlock) {
      a.grad[r0 + i] = stage[i];
      if (a.hess) a.hess[r0 + i] = stage_h[i];
    }
  } else {
    static_assert(sizeof stage >= kPairBlock * sizeof(LongPair), "the stage holds a block's long pairs");
    take_unstaged_pairs(a, rows, begin, pairs, reinterpret_cast<LongPair*>(stage), &longs);
  }
  fill_outside(a, rows, begin, pairs);
}

// The pairs that the lanes of a block have left, looked for N at a time.
template <int N, int G>
__device__ __noinline__ void take_left_pairs(const PairLoss& call, u64 rows, const i64* begin, u64 pairs, LongPair* list, u32* longs) {
  const PairLoss a = call;
  for (u64 p0 = u64(blockIdx.x) * N; p0 < pairs; p0 += u64(gridDim.x) * N) {
    const u64 p = p0 + threadIdx.x;
    if (threadIdx.x == 0) *longs = 0;
    __syncthreads();
    if (threadIdx.x < N && p < pairs) {
      const LongPair x{p, clamp_row(begin[2 * p], rows), clamp_row(begin[2 * p + 1], rows), clamp_row(begin[2 * p + 2], rows)};
      if (x.b2 - x.b0 > G * kLaneRows) list[atomicAdd(longs, 1u)] = x;
    }
    __syncthreads();
    take_long_pairs<256>(a, list, *longs);
    __syncthreads();  // (the list has been read)
  }
}

// Short items: G lanes a pair; a pair past kLaneRows rows a lane waits for the
// block (4M rows in 20,000 even pairs 20.8 us, by lanes alone 19.8; 3000 pairs of
// 300 rows and an item of 2^20 rows 257 us, by lanes alone 1605).
template <int G>
__global__ void __launch_bounds__(256, 6) k_preference_lanes(const __grid_constant__ PairLoss a, u64 rows, const i64* begin, u64 pairs) {
  __shared__ LongPair list[256 / G];
  __shared__ u32 longs;
  const u32 lane = threadIdx.x % G;
  const u64 per_block = 256 / G, step = u64(gridDim.x) * per_block, first = u64(blockIdx.x) * per_block;
  bool left = false;
  for (u64 p0 = first; p0 < pairs; p0 += step) {
    const u64 p = p0 + threadIdx.x / G;
    const bool in = p < pairs;  // (the lanes of a warp sum together)
    const u64 b0 = in ? clamp_row(begin[2 * p], rows) : 0, b1 = in ? clamp_row(begin[2 * p + 1], rows) : 0,
              b2 = in ? clamp_row(begin[2 * p + 2], rows) : 0;
    const bool take = b2 - b0 <= G * kLaneRows;
    left |= !take;
    float sa = 0.f, sb = 0.f;
    if (take) {
      sa = span_sum<4>(a, b0, b1, lane, G);
      sb = span_sum<4>(a, b1, b2, lane, G);
    }
    sa = lanes_sum<G>(sa);
    sb = lanes_sum<G>(sb);
    if (!in || !take) continue;
    const PairResult o = pair_result(a, sa - sb, a.weight ? a.weight[p] : 1.f);
    const float h = item_hess(o.h);
    if (lane == 0) a.loss[p] = o.loss;
    span_fill(a, b0, b1, lane, G, o.q, h);
    span_fill(a, b1, b2, lane, G, -o.q, h);
  }
  fill_outside(a, rows, begin, pairs);
  if (__syncthreads_or(left)) take_left_pairs<256 / G, G>(a, rows, begin, pairs, list, &longs);
}

// Long items: a block, or a cluster of blocks, a pair.
constexpr u32 kPairCluster = 8;
template <int kBlockThreads, int U>
__global__ void __launch_bounds__(kBlockThreads) k_preference_block(PairLoss a, u64 rows, const i64* begin, u64 pairs, u32 blocks) {
  constexpr u32 kWarps = kBlockThreads / 32;
  __shared__ float2 part[2][kWarps], blocks_part[2][kPairCluster];
  u32 rank = 0, parity = 0;
  if (blocks > 1) {
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  const u64 first = rank * kBlockThreads + threadIdx.x, step = u64(blocks) * kBlockThreads;
  for (u64 p = blockIdx.x / blocks; p < pairs; p += gridDim.x / blocks) {
    const u64 b0 = clamp_row(begin[2 * p], rows), b1 = clamp_row(begin[2 * p + 1], rows),
              b2 = clamp_row(begin[2 * p + 2], rows);
    float2 s;
    s.x = lanes_sum<32>(span_sum<U>(a, b0, b1, first, step));
    s.y = lanes_sum<32>(span_sum<U>(a, b1, b2, first, step));
    if ((threadIdx.x & 31) == 0) part[parity][threadIdx.x >> 5] = s;
    __syncthreads();
    s = part[parity][threadIdx.x & (kWarps - 1)];
    s.x = lanes_sum<kWarps>(s.x);
    s.y = lanes_sum<kWarps>(s.y);
    if (blocks > 1) {
      if (threadIdx.x < blocks) {
        const u32 here = u32(__cvta_generic_to_shared(&blocks_part[parity][rank]));
        u32 there;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(threadIdx.x));
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(s.x), "f"(s.y) : "memory");
      }
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
      s = make_float2(0.f, 0.f);
      for (u32 b = 0; b < blocks; ++b) {
        s.x += blocks_part[parity][b].x;
        s.y += blocks_part[parity][b].y;
      }
    }
    parity ^= 1;  // (a pair's sums are written while slower threads read the last pair's)
    const PairResult o = pair_result(a, s.x - s.y, a.weight ? a.weight[p] : 1.f);
    const float h = item_hess(o.h);
    if (first == 0) a.loss[p] = o.loss;
    span_fill(a, b0, b1, first, step, o.q, h);
    span_fill(a, b1, b2, first, step, -o.q, h);
  }
  fill_outside(a, rows, begin, pairs);
}

// Few pairs of very many rows: every block of the device takes pieces of
// kPieceRows rows, whatever pairs they belong to, in three launches, since a
// pair's one cluster of blocks uses eight SMs alone (reference scores given, by
// pieces against by clusters: 4M rows in one pair 16.5 us against 84, one pair
// of 262,144 rows 8.8 / 9.9, of 131,072 8.3 / 7.6; eight pairs of 262,144 rows
// each 14.8 / 14.6, with the curvature 16.2 / 20.2; sixteen of them 33.9 /
// 27.5).  The pieces' sums wait in the gradient's place, which has two rows or
// more for each piece of a pair of kPiecedRows rows; shorter pairs are summed
// by the second launch.  It leaves a pair's gradient (and curvature) in its
// first row, where the third finds it for the others.
constexpr u32 kPieceRows = 8192, kPiecedRows = 4 * kPieceRows, kFewPairs = 8;
constexpr u64 kVeryLongRows = u64(1) << 18;  // a pair, on average
struct PairSpan {
  u64 b0, b1, b2;
  __device__ __forceinline__ PairSpan(const u64* offset, u64 p) : b0(offset[2 * p]), b1(offset[2 * p + 1]), b2(offset[2 * p + 2]) {}
  __device__ __forceinline__ bool pieced() const { return b2 > b0 && b2 - b0 >= kPiecedRows && b1 >= b0 && b1 <= b2; }
  // Places of a piece's two sums in the gradient.
  __device__ __forceinline__ u64 place(u64 piece) const { return b0 + 2 * (piece - b0 / kPieceRows); }
};
// The offsets, read once for the whole block.
__device__ __forceinline__ void read_offsets(u64* offset, const i64* begin, u64 pairs, u64 rows) {
  for (u64 i = threadIdx.x; i <= 2 * pairs; i += blockDim.x) offset[i] = clamp_row(begin[i], rows);
  __syncthreads();
}
__global__ void __launch_bounds__(512) k_preference_pieces(PairLoss a, u64 rows, const i64* begin, u64 pairs) {
  __shared__ float2 part[16];
  __shared__ u64 offset[2 * kFewPairs + 1];
  read_offsets(offset, begin, pairs, rows);
  const u64 piece = blockIdx.x, r0 = piece * kPieceRows, r1 = min(rows, r0 + kPieceRows);
  for (u64 p = 0; p < pairs; ++p) {
    const PairSpan x(offset, p);
    if (!x.pieced() || x.b2 <= r0 || x.b0 >= r1) continue;
    const u64 lo = max(x.b0, r0), hi = min(x.b2, r1), mid = min(max(x.b1, lo), hi);
    const float2 s = block_sums<16>(make_float2(span_sum<8>(a, lo, mid, threadIdx.x, 512),
                                                span_sum<8>(a, mid, hi, threadIdx.x, 512)), part);
    if (threadIdx.x < 2) a.grad[x.place(piece) + threadIdx.x] = threadIdx.x ? s.y : s.x;
  }
}
__global__ void __launch_bounds__(512) k_preference_settle(PairLoss a, u64 rows, const i64* begin) {
  __shared__ float2 part[16];
  __shared__ u64 offset[2 * kFewPairs + 1];
  read_offsets(offset, begin, gridDim.x, rows);
  const u64 p = blockIdx.x;
  const PairSpan x(offset, p);
  float2 s = make_float2(0.f, 0.f);
  if (x.pieced()) {
    for (u64 k = x.b0 / kPieceRows + threadIdx.x; k * kPieceRows < x.b2; k += 512) {
      const u64 at = x.place(k);
      s.x += a.grad[at];
      s.y += a.grad[at + 1];
    }
  } else {
    s.x = span_sum<8>(a, x.b0, x.b1, threadIdx.x, 512);
    s.y = span_sum<8>(a, x.b1, x.b2, threadIdx.x, 512);
  }
  s = block_sums<16>(s, part);  // (and every piece's sums have been read)
  if (threadIdx.x) return;
  const PairResult o = pair_result(a, s.x - s.y, a.weight ? a.weight[p] : 1.f);
  a.loss[p] = o.loss;
  if (x.b2 <= x.b0) return;
  a.grad[x.b0] = x.b1 > x.b0 ? o.q : -o.q;
  if (a.hess) a.hess[x.b0] = item_hess(o.h);
}
__global__ void __launch_bounds__(512) k_preference_spread(PairLoss a, u64 rows, const i64* begin, u64 pairs) {
  __shared__ u64 offset[2 * kFewPairs + 1];
  read_offsets(offset, begin, pairs, rows);
  const u64 r0 = u64(blockIdx.x) * kPieceRows, r1 = min(rows, r0 + kPieceRows);
  for (u64 p = 0; p < pairs; ++p) {
    const PairSpan x(offset, p);
    const u64 lo = max(x.b0 + 1, r0), hi = min(x.b2, r1);
    if (lo >= hi) continue;
    const float first = a.grad[x.b0], q = x.b1 > x.b0 ? first : -first, h = a.hess ? a.hess[x.b0] : 0.f;
    const u64 mid = min(max(x.b1, lo), hi);
    span_fill(a, lo, mid, threadIdx.x, 512, q, h);
    span_fill(a, mid, hi, threadIdx.x, 512, -q, h);
  }
  fill_outside(a, rows, begin, pairs);
}

// ---- any pairs --------------------------------------------------------------
// Three launches: every pair's terms once, in the pairs' order (two gathers of
// scores a pair); then the terms summed by row over the list of (row, pair)
// that the plan holds sorted by row, a warp taking kPairChunk entries whatever
// rows they belong to; then the rows that reach over several chunks, a warp
// each, which is what rows in very many pairs cost (8M pairs that share one row:
// 589 us, of strongly skewed rows 207).  Bound by
// the gathers, two of 4-byte scores and two of 8-byte terms a pair, a random
// sector a lane, of which L1 takes 0.7 to 0.8 a clock and SM: 8M pairs over 1M
// rows 170 us (82 + 83 + 5).  One thread a row, evaluating each pair from both
// of its rows, took 258.

__global__ void __launch_bounds__(256) k_gap(const float* score, const float* ref, u64 rows, float* out) {
  for (u64 r = u64(blockIdx.x) * blockDim.x + threadIdx.x; r < rows; r += u64(gridDim.x) * blockDim.x)
    out[r] = score[r] - ref[r];
}

__global__ void __launch_bounds__(256) k_pair_terms(PairLoss a, const float* score, const int2* __restrict__ pair,
                                                    u64 pairs, u64 rows, float2* terms) {
  constexpr int U = 4;
  const u64 step = u64(gridDim.x) * blockDim.x, first = u64(blockIdx.x) * blockDim.x + threadIdx.x;
  for (u64 p0 = first; p0 < pairs; p0 += U * step) {
    float d[U], w[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const u64 p = p0 + i * step;
      d[i] = w[i] = 0.f;
      if (p < pairs) {
        const int2 x = __ldcs(pair + p);
        d[i] = score[x.x] - score[x.y];
        w[i] = a.weight ? __ldcs(a.weight + p) : 1.f;
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const u64 p = p0 + i * step;
      if (p >= pairs) break;
      const PairResult o = pair_result(a, d[i], w[i]);
      __stcs(a.loss + p, o.loss);
      terms[p] = make_float2(o.q, o.h);
    }
  }
  for (u64 r = first; r < rows; r += step) {  // (rows of no pair keep these)
    a.grad[r] = 0.f;
    if (a.hess) a.hess[r] = item_hess(0.f);
  }
}

__device__ __forceinline__ void put_row(const PairLoss& a, u32 row, float2 s) {
  a.grad[row] = s.x;
  if (a.hess) a.hess[row] = item_hess(s.y);
}

// One warp a chunk of entries.  A row that begins and ends in the chunk is
// written here; of one that began before, this chunk's sum goes to head[c], of
// one that goes on after it to tail[c].  joins[c]: the row that ends in the
// chunk without having begun there, kInside where the whole chunk is part of
// one that goes on, kNoRow where there is neither.
constexpr u32 kNoRow = 0xffffffffu, kInside = 0xfffffffeu;  // past every row
__global__ void __launch_bounds__(256) k_pair_rows(PairLoss a, const PairEntry* __restrict__ entry, u64 n,
                                                   const float2* __restrict__ terms, float2* head, float2* tail,
                                                   u32* joins) {
  constexpr int kSteps = kPairChunk / 32;
  const u32 lane = threadIdx.x & 31;
  const u64 c = u64(blockIdx.x) * 8 + (threadIdx.x >> 5), base = c * kPairChunk;
  if (base >= n) return;
  u32 row[kSteps];
  float2 v[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const u64 e = base + i * 32 + lane;
    uint2 x = make_uint2(kNoRow, 0);
    if (e < n) x = __ldcs(reinterpret_cast<const uint2*>(entry) + e);  // (read once: L2 is kept for the terms)
    row[i] = x.x;
    v[i] = e < n ? terms[x.y & 0x7fffffffu] : make_float2(0.f, 0.f);
    if (x.y >> 31) v[i].x = -v[i].x;
  }
  const u32 first = __shfl_sync(0xffffffffu, row[0], 0);
  const u32 before = base ? entry[base - 1].row : kNoRow, after = base + kPairChunk < n ? entry[base + kPairChunk].row : kNoRow;
  const bool begun = before == first;
  u32 open = kNoRow;  // the row that the last step ended in, and its sum
  float2 sum = make_float2(0.f, 0.f);
  u32 join = kNoRow;
  auto close = [&](u32 r, float2 s) {
    if (r == kNoRow) return;
    if (r == first && begun) {
      head[c] = s;
      join = r;
    } else {
      put_row(a, r, s);
    }
  };
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const u32 r = row[i], up = __shfl_up_sync(0xffffffffu, r, 1);
    const u32 starts = __ballot_sync(0xffffffffu, lane == 0 ? r != open : r != up);
    // (lane 0 of a step that goes on with the open row takes its sum in)
    if (lane == 0) {
      if (starts & 1) close(open, sum);
      else v[i] = make_float2(sum.x + v[i].x, sum.y + v[i].y);
    }
    const u32 upto = starts & (0xffffffffu >> (31 - lane));
    const u32 reach = upto ? lane - (31 - __clz(upto)) : lane;
    float2 s = v[i];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float x = __shfl_up_sync(0xffffffffu, s.x, d), y = __shfl_up_sync(0xffffffffu, s.y, d);
      if (u32(d) <= reach) {
        s.x += x;
        s.y += y;
      }
    }
    if (lane < 31 && (starts >> (lane + 1) & 1)) close(r, s);
    open = __shfl_sync(0xffffffffu, r, 31);
    sum.x = __shfl_sync(0xffffffffu, s.x, 31);
    sum.y = __shfl_sync(0xffffffffu, s.y, 31);
  }
  if (lane == 0 && open != kNoRow) {
    if (open != after) {
      close(open, sum);
    } else if (open == first && begun) {  // the whole chunk is one row's
      head[c] = sum;
      join = kInside;
    } else {
      tail[c] = sum;
    }
  }
  join = __reduce_min_sync(0xffffffffu, join);  // (one lane's at most)
  if (lane == 0) joins[c] = join;
}

// The rows that end in a chunk that they did not begin in: the tail of the
// chunk where they began, then the heads of those since.
__global__ void __launch_bounds__(256) k_pair_joins(PairLoss a, const PairEntry* __restrict__ entry, u64 chunks,
                                                    const float2* head, const float2* tail, const u32* joins) {
  const u32 lane = threadIdx.x & 31;
  const u64 c = u64(blockIdx.x) * 256 + threadIdx.x;
  const u32 row = c < chunks ? joins[c] : kNoRow;
  const bool ends = row < kInside;
  u64 from = c - 1;
  if (ends && joins[c - 1] == kInside) {  // the first chunk that holds entries of the row
    u64 lo = 0, hi = c * kPairChunk - 1;  // entry[hi].row == row
    while (lo < hi) {
      const u64 mid = (lo + hi) / 2;
      if (entry[mid].row < row) lo = mid + 1;
      else hi = mid;
    }
    from = lo / kPairChunk;
  }
  const bool wide = ends && c - from > 32;
  if (ends && !wide) {
    float2 s = tail[from];
    for (u64 k = from + 1; k <= c; ++k) {
      const float2 x = head[k];
      s.x += x.x;
      s.y += x.y;
    }
    put_row(a, row, s);
  }
  for (u32 todo = __ballot_sync(0xffffffffu, wide); todo; todo &= todo - 1) {
    const int src = __ffs(int(todo)) - 1;
    const u64 f = __shfl_sync(0xffffffffu, from, src), l = __shfl_sync(0xffffffffu, c, src);
    const u32 r = __shfl_sync(0xffffffffu, row, src);
    float2 s = make_float2(0.f, 0.f);
    for (u64 k = f + lane; k <= l; k += 32) {
      const float2 x = k == f ? tail[k] : head[k];
      s.x += x.x;
      s.y += x.y;
    }
    s.x = lanes_sum<32>(s.x);
    s.y = lanes_sum<32>(s.y);
    if (lane == 0) put_row(a, r, s);
  }
}

// ---- the plan: (row, pair) entries sorted by row, by a least-significant-
// digit radix sort, which keeps the pairs of a row in their order.  8M pairs
// over 1M rows take 0.9 to 1.2 ms, as long as five to seven runs.
__global__ void __launch_bounds__(256) k_pair_entries(const int2* __restrict__ pair, u64 pairs, u64 rows, PairEntry* out,
                                                      unsigned long long* bad) {
  for (u64 p = u64(blockIdx.x) * blockDim.x + threadIdx.x; p < pairs; p += u64(gridDim.x) * blockDim.x) {
    const int2 x = pair[p];
    const bool outside = x.x < 0 || x.y < 0 || u64(x.x) >= rows || u64(x.y) >= rows;
    if (outside || x.x == x.y) atomicMin(bad, (unsigned long long)(2 * p + (outside ? 0 : 1)));
    out[2 * p] = PairEntry{u32(x.x), u32(p)};
    out[2 * p + 1] = PairEntry{u32(x.y), u32(p) | 0x80000000u};
  }
}

constexpr int kDigitBits = 8, kDigits = 1 << kDigitBits, kSortWarps = 8, kSortSteps = 16;
constexpr u32 kSortTile = kSortWarps * kSortSteps * 32;

__device__ __forceinline__ u32 digit_of(u32 row, int shift) { return (row >> shift) & (kDigits - 1); }

// Lanes of this warp with the same digit (`in`: lanes that hold an entry).
__device__ __forceinline__ u32 same_digit(u32 digit, bool in) {
  return __match_any_sync(0xffffffffu, in ? digit : kDigits);
}

__global__ void __launch_bounds__(256) k_sort_count(const PairEntry* __restrict__ in, u64 n, int shift, u32 blocks,
                                                    u32* count) {
  __shared__ u32 c[kDigits];
  c[threadIdx.x] = 0;
  __syncthreads();
  const u64 base = u64(blockIdx.x) * kSortTile;
  for (u32 i = threadIdx.x; i < kSortTile && base + i < n; i += 256) atomicAdd(&c[digit_of(in[base + i].row, shift)], 1u);
  __syncthreads();
  count[u64(threadIdx.x) * blocks + blockIdx.x] = c[threadIdx.x];
}

// One block a digit: its counts become exclusive sums over the tiles, and
// total[digit] the digit's count.
__global__ void __launch_bounds__(256) k_sort_scan(u32* count, u32 blocks, u32* total) {
  __shared__ u32 warp[8];
  u32* const row = count + u64(blockIdx.x) * blocks;
  const u32 lane = threadIdx.x & 31;
  u32 carry = 0;
  for (u32 b0 = 0; b0 < blocks; b0 += 256) {
    const u32 b = b0 + threadIdx.x, mine = b < blocks ? row[b] : 0;
    u32 s = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const u32 x = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= u32(d)) s += x;
    }
    if (lane == 31) warp[threadIdx.x >> 5] = s;
    __syncthreads();
    u32 below = 0, all = 0;
    for (u32 w = 0; w < 8; ++w) {
      if (w < threadIdx.x >> 5) below += warp[w];
      all += warp[w];
    }
    if (b < blocks) row[b] = carry + below + s - mine;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

// Moves a tile's entries to their places: digit, then tile, then the order in
// the tile (a warp holds kSortSteps * 32 consecutive entries of it).
__global__ void __launch_bounds__(256) k_sort_move(const PairEntry* __restrict__ in, u64 n, int shift, u32 blocks,
                                                   const u32* __restrict__ count, const u32* __restrict__ total,
                                                   PairEntry* out) {
  __shared__ u32 at[kSortWarps][kDigits];
  __shared__ u32 scan[kDigits];
  const u32 t = threadIdx.x, warp = t >> 5, lane = t & 31;
  for (int w = 0; w < kSortWarps; ++w) at[w][t] = 0;
  scan[t] = total[t];
  __syncthreads();
  const u64 base = u64(blockIdx.x) * kSortTile + u64(warp) * kSortSteps * 32;
  for (int i = 0; i < kSortSteps; ++i) {
    const u64 e = base + i * 32 + lane;
    const u32 d = e < n ? digit_of(in[e].row, shift) : 0;
    const u32 same = same_digit(d, e < n);
    if (e < n && (same & ((1u << lane) - 1)) == 0) at[warp][d] += __popc(same);
    __syncwarp();
  }
  // inclusive sums of the digits' totals
  for (u32 d = 1; d < kDigits; d <<= 1) {
    const u32 x = t >= d ? scan[t - d] : 0;
    __syncthreads();
    scan[t] += x;
    __syncthreads();
  }
  u32 place = scan[t] - total[t] + count[u64(t) * blocks + blockIdx.x];
  for (int w = 0; w < kSortWarps; ++w) {
    const u32 m = at[w][t];
    at[w][t] = place;
    place += m;
  }
  __syncthreads();
  for (int i = 0; i < kSortSteps; ++i) {
    const u64 e = base + i * 32 + lane;
    PairEntry x{0, 0};
    if (e < n) x = in[e];
    const u32 d = digit_of(x.row, shift), same = same_digit(d, e < n), lower = same & ((1u << lane) - 1);
    u32 to = 0;
    if (e < n) to = at[warp][d] + __popc(lower);
    __syncwarp();
    if (e < n && lower == 0) at[warp][d] += __popc(same);
    if (e < n) out[to] = x;
    __syncwarp();
  }
}

u32 blocks_for(u64 n, u64 per_block, u64 cap = u64(kSMs) * 16) {
  const u64 want = (n + per_block - 1) / per_block;
  return u32(want < 1 ? 1 : (want < cap ? want : cap));
}

}  // namespace

void launch_preference(const PairLoss& a, u64 rows, const i64* begin, u64 pairs, cudaStream_t s) {
  if (!rows && !pairs) return;
  const u64 average = pairs ? rows / pairs : rows;  // rows of a pair
  if (!begin) {
    const auto odd = [](const float* p) { return reinterpret_cast<std::uintptr_t>(p) & 7; };
    if (odd(a.score) || odd(a.ref) || odd(a.grad) || odd(a.hess))
      k_preference_rows<false><<<blocks_for(rows / 2 + 1, 256), 256, 0, s>>>(a, rows, pairs);
    else
      k_preference_rows<true><<<blocks_for(rows / 2 + 1, 256), 256, 0, s>>>(a, rows, pairs);
  } else if (average <= 12 && pairs >= 1024) {
    need(pairs <= (u64(kPairBlock) << 31), "too many pairs for one launch");
    k_preference_staged<<<u32((pairs + kPairBlock - 1) / kPairBlock), kPairBlock, 0, s>>>(a, rows, begin, pairs);
  } else if (average < 64 && pairs >= 64) {
    k_preference_lanes<8><<<blocks_for(pairs, 32), 256, 0, s>>>(a, rows, begin, pairs);
  } else if (average < 1024 && pairs >= 4 * kSMs) {
    k_preference_lanes<32><<<blocks_for(pairs, 8), 256, 0, s>>>(a, rows, begin, pairs);
  } else if (pairs >= 1 && pairs <= kFewPairs && average >= kVeryLongRows && rows < (u64(kPieceRows) << 31)) {
    const u32 pieces = u32((rows + kPieceRows - 1) / kPieceRows);
    k_preference_pieces<<<pieces, 512, 0, s>>>(a, rows, begin, pairs);
    after_launch("preference loss");
    k_preference_settle<<<u32(pairs), 512, 0, s>>>(a, rows, begin);
    after_launch("preference loss");
    k_preference_spread<<<pieces, 512, 0, s>>>(a, rows, begin, pairs);
  } else {
    // A block a pair; few pairs of many rows: a cluster of larger blocks
    // each, with more loads under way (a cluster's 4M rows of one pair: 184 us
    // by eight blocks of 512 threads, 84 by eight of 1024; 1000 pairs of 4000:
    // 19 and 41).
    u32 blocks = 1;
    while (blocks < kPairCluster && pairs * blocks * 2 <= kSMs && average > 4096u * blocks) blocks *= 2;
    const bool large = average >= 32768;
    const u64 most = kSMs * (large ? 2 : 4), clusters = pairs < 1 ? 1 : (pairs < most ? pairs : most);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(u32(clusters * blocks));
    cfg.blockDim = dim3(large ? 1024 : 512);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = blocks;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = blocks > 1 ? 1 : 0;
    auto* const kernel = large ? k_preference_block<1024, 8> : k_preference_block<512, 4>;
    DP_CUDA((cudaLaunchKernelEx(&cfg, kernel, a, rows, begin, pairs, blocks)));
  }
  after_launch("preference loss");
}

void build_pair_plan(PairPlan& plan, u64 rows, const i32* pair_rows, u64 pairs, cudaStream_t s) {
  DP_CUDA(cudaGetDevice(&plan.device));
  plan.rows = rows;
  plan.pairs = pairs;
  if (!pairs) return;
  const u64 n = 2 * pairs, chunks = (n + kPairChunk - 1) / kPairChunk;
  SlabPlan slab;
  slab.want(plan.pair, pairs);
  slab.want(plan.entry, n);
  slab.want(plan.terms, pairs);
  slab.want(plan.head, chunks);
  slab.want(plan.tail, chunks);
  slab.want(plan.joins, chunks);
  slab.want(plan.gap, rows);
  slab.commit(plan.slabs, plan.device);
  const u32 tiles = u32((n + kSortTile - 1) / kSortTile);
  DevBuf<PairEntry> other;
  DevBuf<u32> count, total;
  DevBuf<unsigned long long> bad;
  SlabPlan work;
  work.want(other, n);
  work.want(count, u64(kDigits) * tiles);
  work.want(total, kDigits);
  work.want(bad, 1);
  std::vector<DevBuf<unsigned char>> scratch;
  work.commit(scratch, plan.device);
  DP_CUDA(cudaMemcpyAsync(plan.pair.get(), pair_rows, pairs * sizeof(int2), cudaMemcpyDeviceToDevice, s));
  DP_CUDA(cudaMemsetAsync(bad.get(), 0xff, sizeof(unsigned long long), s));
  int passes = 0;
  while (passes * kDigitBits < 32 && (rows - 1) >> (passes * kDigitBits)) ++passes;
  // an even number of passes ends where it began
  PairEntry *from = passes % 2 ? other.get() : plan.entry.get(), *to = passes % 2 ? plan.entry.get() : other.get();
  k_pair_entries<<<blocks_for(pairs, 256), 256, 0, s>>>(plan.pair.get(), pairs, rows, from, bad.get());
  after_launch("pair entries");
  unsigned long long worst = 0;
  DP_CUDA(cudaMemcpyAsync(&worst, bad.get(), sizeof worst, cudaMemcpyDeviceToHost, s));
  DP_CUDA(cudaStreamSynchronize(s));
  if (worst != ~0ull)
    fail("pair " + std::to_string(worst / 2) +
         (worst % 2 ? std::string(" names one row twice") : " names a row outside [0, " + std::to_string(rows) + ")"));
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * kDigitBits;
    k_sort_count<<<tiles, 256, 0, s>>>(from, n, shift, tiles, count.get());
    after_launch("pair sort");
    k_sort_scan<<<kDigits, 256, 0, s>>>(count.get(), tiles, total.get());
    after_launch("pair sort");
    k_sort_move<<<tiles, 256, 0, s>>>(from, n, shift, tiles, count.get(), total.get(), to);
    after_launch("pair sort");
    std::swap(from, to);
  }
  DP_CUDA(cudaStreamSynchronize(s));
  for (auto& b : scratch) SlabCache::give(plan.device, std::move(b));
}

PairPlan::~PairPlan() {
  if (slabs.empty()) return;
  cudaDeviceSynchronize();  // no run of the plan is under way when its memory goes to the next one
  for (auto& b : slabs) SlabCache::give(device, std::move(b));
}

void launch_pair_loss(const PairPlan& p, const PairLoss& a, cudaStream_t s) {
  if (!p.rows) return;
  const float* score = a.score;
  if (a.ref && p.pairs) {
    k_gap<<<blocks_for(p.rows, 256), 256, 0, s>>>(a.score, a.ref, p.rows, p.gap.get());
    after_launch("pair loss");
    score = p.gap.get();
  }
  const u64 most = p.pairs > p.rows ? p.pairs : p.rows;
  k_pair_terms<<<blocks_for(most, 256), 256, 0, s>>>(a, score, p.pair.get(), p.pairs, p.rows, p.terms.get());
  after_launch("pair loss");
  if (!p.pairs) return;
  const u64 n = 2 * p.pairs, chunks = (n + kPairChunk - 1) / kPairChunk;
  k_pair_rows<<<u32((chunks + 7) / 8), 256, 0, s>>>(a, p.entry.get(), n, p.terms.get(), p.head.get(), p.tail.get(),
                                                    p.joins.get());
  after_launch("pair loss");
  if (chunks > 1) {
    k_pair_joins<<<u32((chunks + 255) / 256), 256, 0, s>>>(a, p.entry.get(), chunks, p.head.get(), p.tail.get(),
                                                        p.joins.get());
    after_launch("pair loss");
  }
}

}  // namespace dp
