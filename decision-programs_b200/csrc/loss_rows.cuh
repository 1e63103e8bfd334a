// Row kernels of the choice losses (included by one source file a margin type).
//
// A row of K margins is read once and kept in registers: maximum, sum of
// exponentials and gradient are all taken from there, so that the traffic is
// the margins in and the gradient out, which bounds these kernels (a gradient
// element costs two exponentials and about ten instructions for the two to
// four bytes in and out that it moves).
//
// Rows start at any multiple of their element size.  A row is cut on 16-byte
// boundaries of its own address: whole 16-byte vectors are moved as such, the
// ragged first and last ones element by element, so that nothing outside the
// row is read or written.
#pragma once
#include <atomic>
#include <cstring>
#include <type_traits>

#include "kernels.h"
#include "loss_math.cuh"

namespace dp {
namespace {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
// e^x.  The difference z - m is taken before the scaling by log2 e: margins of
// the type's lowest value would overflow if they were scaled first.
__device__ __forceinline__ float exp_fast(float x) { return ex2(x * kLog2e); }

// 16 bytes of margins.
template <class T>
struct Vec {
  static constexpr int N = 16 / int(sizeof(T));
  uint4 raw;
  __device__ __forceinline__ void unpack(float (&f)[N]) const {
    const u32 w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        __half2 h;
        memcpy(&h, &w[i], 4);
        const float2 v = __half22float2(h);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      } else {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  __device__ __forceinline__ void pack(const float (&f)[N]) {
    u32 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(f[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        memcpy(&w[i], &h, 4);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        memcpy(&w[i], &h, 4);
      }
    }
    raw = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void fill(float v) {
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = v;
    pack(f);
  }
};

// A row cut into 16-byte vectors: vector j holds elements
// [j N - shift, (j + 1) N - shift), of which those in [0, K) are the row's.
template <class T>
struct RowCut {
  static constexpr int N = Vec<T>::N;
  const T* z;
  u32 K, shift;
  __device__ RowCut(const T* row, u32 classes)
      : z(row), K(classes), shift(u32(reinterpret_cast<std::uintptr_t>(row) & 15) / u32(sizeof(T))) {}
  __device__ u32 vectors() const { return (K + shift + N - 1) / N; }
  __device__ i64 first(u32 j) const { return i64(j) * N - shift; }
  __device__ bool whole(u32 j) const { return (j > 0 || shift == 0) && u64(j + 1) * N <= u64(K) + shift; }
  __device__ __forceinline__ Vec<T> load(u32 j, float outside) const {
    Vec<T> v;
    const i64 k0 = first(j);
    if (whole(j)) {
      v.raw = *reinterpret_cast<const uint4*>(z + k0);
    } else {
      float f[N];
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = k0 + i >= 0 && k0 + i < i64(K) ? to_f32(z[k0 + i]) : outside;
      v.pack(f);
    }
    return v;
  }
  // N values of this row's vector j into a row of another array.
  template <class U>
  __device__ __forceinline__ void store(U* row, u32 j, const float (&f)[N]) const {
    const i64 k0 = first(j);
    U* const at = row + k0;
    if (whole(j) && (reinterpret_cast<std::uintptr_t>(at) & 15) == 0) {
      constexpr int M = Vec<U>::N;
#pragma unroll
      for (int b = 0; b < N / M; ++b) {
        float part[M];
#pragma unroll
        for (int i = 0; i < M; ++i) part[i] = f[b * M + i];
        Vec<U> v;
        v.pack(part);
        reinterpret_cast<uint4*>(at)[b] = v.raw;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (k0 + i >= 0 && k0 + i < i64(K)) at[i] = from_f32<U>(f[i]);
    }
  }
};

template <int G, class Op>
__device__ __forceinline__ float lanes_reduce(float v, Op op) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
struct MaxOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct SumOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
__device__ __forceinline__ u32 cluster_rank() {
  u32 r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Stores a pair at the same shared-memory place in block `rank` of the cluster.
__device__ __forceinline__ void cluster_put(float2* at, u32 rank, float2 v) {
  const u32 here = u32(__cvta_generic_to_shared(at));
  u32 there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(v.x), "f"(v.y) : "memory");
}
constexpr u32 kMaxCluster = 8;

// A sum of exponentials relative to `from`, made relative to `to` >= from.  A
// part that is masked throughout has from = -inf and the sum 0 (or NaN).
__device__ __forceinline__ float rebase(float s, float from, float to) {
  return from == neg_inf() ? s : s * exp_fast(from - to);
}

// The maximum and the sum over the blocks of a cluster, in the order of their
// ranks: every block gets the same two numbers.
__device__ __forceinline__ void cluster_join(float2* parts, u32 blocks, float& m, float& s) {
  if (threadIdx.x < blocks) cluster_put(parts + cluster_rank(), threadIdx.x, make_float2(m, s));
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  float top = neg_inf();
  for (u32 b = 0; b < blocks; ++b) top = fmaxf(top, parts[b].x);
  float sum = 0.f;
  for (u32 b = 0; b < blocks; ++b) sum += rebase(parts[b].y, parts[b].x, top);
  m = top;
  s = sum;
}

// What a row's losses read, loaded while its margins are on their way.
template <bool kPolicy>
__device__ __forceinline__ RowScalars policy_scalars(const RowArgs& a, u64 r) {
  RowScalars x;
  if constexpr (kPolicy) {
    x.old = a.policy.old_log_prob[r];
    x.adv = a.policy.advantage[r];
    if (a.policy.ref_log_prob) x.ref = a.policy.ref_log_prob[r];
    if (a.policy.weight) x.w = a.policy.weight[r];
  }
  return x;
}

// Results of one row from its maximum and sum; returns the loss's derivative
// by the log-probability.  `writer`: one thread of the row.
template <bool kPolicy>
__device__ __forceinline__ float finish_row(const RowArgs& a, u64 r, const RowScalars& x, float m, float s, bool writer) {
  float2 norm;
  float loss = 0.f, c = 0.f;
  const float l = row_log_prob(m, s, x.zy, norm);
  if (kPolicy && s != 0.f) c = policy_row(a.policy, x, l, loss);
  if (writer) {
    a.log_prob[r] = l;
    if constexpr (kPolicy) a.loss[r] = loss;
    else a.norm[r] = norm;
  }
  return c;
}
template <bool kPolicy>
__device__ __forceinline__ void skip_row(const RowArgs& a, u64 r, bool writer) {
  if (!writer) return;
  a.log_prob[r] = 0.f;
  if constexpr (kPolicy) a.loss[r] = 0.f;
  else a.norm[r] = make_float2(0.f, 0.f);
}

// Gradient and curvature of one vector of margins, p = exp((z - base) - low) * scale.
template <class T>
__device__ __forceinline__ void grad_vector(const RowCut<T>& cut, u32 j, const Vec<T>& v, i32 y, float c, float base,
                                            float low, float scale, T* g, float* h) {
  constexpr int N = Vec<T>::N;
  float p[N], e[N];
  v.unpack(p);
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = exp_fast((p[i] - base) - low);
  const float down = -c * scale;
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = down * p[i];
  const i64 at = i64(y) - cut.first(j);  // the label's place in this vector, if it is there
  if (at >= 0 && at < N) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (int(at) == i) e[i] = c * (1.f - p[i] * scale);
  }
  cut.store(g, j, e);
  if (h) {
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = margin_hess(c, p[i] * scale);
    cut.store(h, j, e);
  }
}
template <class T>
__device__ __forceinline__ void zero_vector(const RowCut<T>& cut, u32 j, T* g, float* h) {
  constexpr int N = Vec<T>::N;
  float e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = 0.f;
  cut.store(g, j, e);
  if (h) cut.store(h, j, e);
}

// G lanes of a warp a row, V vectors a lane, kept in registers.
template <class T, bool kPolicy, int G, int V>
__global__ void __launch_bounds__(256, 4) k_row_loss(RowArgs a) {
  constexpr int N = Vec<T>::N;
  const u32 lane = threadIdx.x % G;
  const u64 r = u64(blockIdx.x) * (256 / G) + threadIdx.x / G;
  const bool in = r < a.m.rows;
  const i32 y = in ? a.label[r] : -1;
  const bool live = u32(y) < a.m.classes;
  const RowCut<T> cut(static_cast<const T*>(a.m.z) + (in ? r : 0) * a.m.stride, a.m.classes);
  const u32 nvec = cut.vectors();
  float c = 0.f, base = 0.f, scale = 0.f, m = neg_inf(), s = 0.f;
  Vec<T> v[V];
  RowScalars x;
  if (live) {
    x = policy_scalars<kPolicy>(a, r);
    x.zy = to_f32(cut.z[y]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const u32 j = lane + i * G;
      if (j < nvec) v[i] = cut.load(j, neg_inf());
      else v[i].fill(neg_inf());
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float f[N];
      v[i].unpack(f);
#pragma unroll
      for (int k = 0; k < N; ++k) m = fmaxf(m, f[k]);
    }
  }
  m = lanes_reduce<G>(m, MaxOp());  // (the lanes of a warp reduce together, whatever their rows)
  base = exp_base(m);
  if (live) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float f[N];
      v[i].unpack(f);
#pragma unroll
      for (int k = 0; k < N; ++k) s += exp_fast(f[k] - base);
    }
  }
  s = lanes_reduce<G>(s, SumOp());
  if (live) {
    c = finish_row<kPolicy>(a, r, x, m, s, lane == 0);
    scale = 1.f / s;
  } else if (in) {
    skip_row<kPolicy>(a, r, lane == 0);
  }
  __syncwarp();  // (a gradient in the margins' place: every lane has read its label's margin)
  if constexpr (kPolicy) {
    if (!a.out.grad || !in) return;
    T* const g = static_cast<T*>(a.out.grad) + r * a.out.grad_stride;
    float* const h = a.out.hess ? a.out.hess + r * a.out.hess_stride : nullptr;
    if (c == 0.f) {
      for (u32 j = lane; j < nvec; j += G) zero_vector(cut, j, g, h);
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const u32 j = lane + i * G;
      if (j < nvec) grad_vector(cut, j, v[i], y, c, base, 0.f, scale, g, h);
    }
  }
}

// ---- long rows --------------------------------------------------------------
// `blocks` blocks of a cluster share a row, and each cluster walks its rows
// (r, r + clusters, ...).  Every thread streams its own vectors through its
// own places of a ring in shared memory, by asynchronous copies that run
// ahead of it into the following rows, so that margins keep arriving while
// sums are joined and gradients are written; nothing in the ring is shared,
// so it needs no barrier.  A row that fits in the ring stays there between
// its sum and its gradient (one read of the margins); a longer one is
// streamed twice.
__device__ __forceinline__ void copy_async(void* shared, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(u32(__cvta_generic_to_shared(shared))), "l"(global)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most n (below S) of this thread's latest groups are under way.
template <int S>
__device__ __forceinline__ void copy_wait(u32 n) {
  if constexpr (S > 1) {
    if (n == S - 1) asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
    else copy_wait<S - 1>(n);
  } else {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
}

// The rows of one cluster in order, their labels read 32 at a time.
struct RowWalk {
  const i32* label;
  u64 rows, step, r;
  u32 classes, at = 32;
  i32 batch = -1;
  __device__ RowWalk(const RowArgs& a, u64 first, u64 clusters)
      : label(a.label), rows(a.m.rows), step(clusters), r(first), classes(a.m.classes) {}
  __device__ bool done() const { return r >= rows; }
  __device__ i32 here() {
    if (at == 32) {
      const u64 mine = r + (threadIdx.x & 31) * step;
      batch = mine < rows ? label[mine] : -1;
      at = 0;
    }
    return __shfl_sync(0xffffffffu, batch, at);
  }
  __device__ void next() {
    r += step;
    ++at;
  }
};

// One block's share [j0, j1) of a row's vectors, in groups of NT * U.
template <class T, int NT, int U>
struct RowShare {
  u32 j0 = 0, j1 = 0;
  RowShare() = default;
  __device__ RowShare(const RowCut<T>& cut, u32 rank, u32 blocks) {
    const u32 nvec = cut.vectors(), per = (nvec + blocks - 1) / blocks;
    j0 = min(nvec, rank * per);
    j1 = min(nvec, j0 + per);
  }
  __device__ u32 groups() const { return (j1 - j0 + NT * U - 1) / (NT * U); }
};

template <class T, bool kPolicy, int NT, int U, int S>
__global__ void __launch_bounds__(NT) k_row_loss_ring(RowArgs a, u32 blocks, u32 clusters) {
  constexpr int N = Vec<T>::N, kWarps = NT / 32;
  extern __shared__ uint4 ring[];  // [S][U][NT]
  __shared__ float2 warp_part[2][kWarps];
  __shared__ float2 block_part[2][kMaxCluster];
  const u32 t = threadIdx.x, rank = blocks > 1 ? cluster_rank() : 0;
  const u64 first = blockIdx.x / blocks;
  const T* const z = static_cast<const T*>(a.m.z);
  if (blocks > 1) {  // every block runs before another one writes to its memory
    cluster_arrive();
    cluster_wait();
  }
  const bool backward = kPolicy && a.out.grad != nullptr;

  // the copies' place: row, share, next group, and which pass over the row
  RowWalk in_rows(a, first, clusters);
  RowCut<T> in_cut(z, a.m.classes);
  RowShare<T, NT, U> in_share;
  u32 in_group = 0, in_groups = 0, in_slot = 0;
  bool again = false;
  auto issue = [&]() {
    while (in_group == in_groups && !(in_groups && again) && !in_rows.done()) {
      const bool live = u32(in_rows.here()) < a.m.classes;
      if (live) {
        in_cut = RowCut<T>(z + in_rows.r * a.m.stride, a.m.classes);
        in_share = RowShare<T, NT, U>(in_cut, rank, blocks);
        in_group = 0;
        in_groups = in_share.groups();
        again = backward && in_groups > S;
      }
      in_rows.next();
    }
    if (in_group == in_groups && again) {  // the second pass over a row that the ring does not hold
      in_group = 0;
      again = false;
    }
    if (in_group < in_groups) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const u32 j = in_share.j0 + (in_group * U + u) * NT + t;
        uint4* const at = ring + (in_slot * U + u) * NT + t;
        if (j < in_share.j1) {
          if (in_cut.whole(j)) copy_async(at, in_cut.z + in_cut.first(j));
          else *at = in_cut.load(j, neg_inf()).raw;
        }
      }
      ++in_group;
    }
    copy_commit();  // (empty groups too: the count of groups under way stays S)
    in_slot = in_slot + 1 == S ? 0 : in_slot + 1;
  };
  for (int i = 0; i < S; ++i) issue();

  u32 slot = 0, parity = 0;
  auto advance = [&](u32 x) { return x + 1 == S ? 0 : x + 1; };
  for (RowWalk rows(a, first, clusters); !rows.done(); rows.next()) {
    const u64 r = rows.r;
    const i32 y = rows.here();
    const RowCut<T> cut(z + r * a.m.stride, a.m.classes);
    const RowShare<T, NT, U> share(cut, rank, blocks);
    const u32 groups = share.groups();
    const bool live = u32(y) < a.m.classes, stays = backward && groups <= S;
    float c = 0.f, base = 0.f, scale = 0.f, zy = 0.f;
    if (live) {
      RowScalars x = policy_scalars<kPolicy>(a, r);
      x.zy = zy = to_f32(cut.z[y]);
      float m = neg_inf(), s = 0.f;
      u32 at = slot;
      for (u32 q = 0; q < groups; ++q) {
        copy_wait<S>(stays ? S - 1 - q : S - 1);
        float top = m;
        Vec<T> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (share.j0 + (q * U + u) * NT + t < share.j1) v[u].raw = ring[(at * U + u) * NT + t];
          else v[u].fill(neg_inf());
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[N];
          v[u].unpack(f);
#pragma unroll
          for (int k = 0; k < N; ++k) top = fmaxf(top, f[k]);
        }
        s = rebase(s, m, top);
        m = top;
        const float b = exp_base(m);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[N];
          v[u].unpack(f);
#pragma unroll
          for (int k = 0; k < N; ++k) s += exp_fast(f[k] - b);
        }
        at = advance(at);
        if (!stays) {
          issue();
          slot = at;
        }
      }
      // the pairs of the threads, then of the warps (every warp alike), then of the blocks
      const float wm = lanes_reduce<32>(m, MaxOp());
      s = lanes_reduce<32>(rebase(s, m, wm), SumOp());
      if ((t & 31) == 0) warp_part[parity][t >> 5] = make_float2(wm, s);
      __syncthreads();
      const float2 p = warp_part[parity][t & (kWarps - 1)];
      m = lanes_reduce<kWarps>(p.x, MaxOp());
      s = lanes_reduce<kWarps>(rebase(p.y, p.x, m), SumOp());
      if (blocks > 1) cluster_join(block_part[parity], blocks, m, s);
      parity ^= 1;  // (a row's parts are written while slower threads read the last row's)
      base = exp_base(m);
      scale = 1.f / s;
      c = finish_row<kPolicy>(a, r, x, m, s, rank == 0 && t == 0);
    } else {
      skip_row<kPolicy>(a, r, rank == 0 && t == 0);
    }
    if constexpr (kPolicy) {
      if (!backward) continue;
      T* const g = static_cast<T*>(a.out.grad) + r * a.out.grad_stride;
      float* const h = a.out.hess ? a.out.hess + r * a.out.hess_stride : nullptr;
      const u32 mine = share.j0 + t;
      if (!live) {
        for (u32 j = mine; j < share.j1; j += NT) zero_vector(cut, j, g, h);
        continue;
      }
      const float down = -c * scale;
      for (u32 q = 0; q < groups; ++q) {
        if (!stays) copy_wait<S>(S - 1);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const u32 j = mine + (q * U + u) * NT;
          if (j < share.j1) {
            if (c == 0.f) {
              zero_vector(cut, j, g, h);
            } else {
              Vec<T> v;
              v.raw = ring[(slot * U + u) * NT + t];
              float f[N], e[N];
              v.unpack(f);
#pragma unroll
              for (int k = 0; k < N; ++k) f[k] = exp_fast(f[k] - base);
#pragma unroll
              for (int k = 0; k < N; ++k) e[k] = down * f[k];
              cut.store(g, j, e);
              if (h) {
#pragma unroll
                for (int k = 0; k < N; ++k) e[k] = margin_hess(c, f[k] * scale);
                cut.store(h, j, e);
              }
            }
          }
        }
        slot = advance(slot);
        issue();
      }
      // the label's element, by the thread that has written its vector
      const u32 jy = (u32(y) + cut.shift) / N;
      if (c != 0.f && jy >= share.j0 && jy < share.j1 && (jy - share.j0) % NT == t)
        g[y] = from_f32<T>(c * (1.f - exp_fast(zy - base) * scale));
    }
  }
}

// Few classes: a block stages kTileRows whole rows in shared memory (adjacent
// threads read adjacent elements, whatever the row length), each thread then
// takes one row, and the block writes the gradients as it read the margins.
// Rows lie an odd number of words apart, so that the 32 rows of a warp use
// the 32 banks.
constexpr u32 kTileRows = 256, kTileClasses = 32;
template <class T, bool kPolicy>
__global__ void __launch_bounds__(kTileRows) k_row_loss_tile(RowArgs a) {
  extern __shared__ float tile[];
  __shared__ float4 row_data[kPolicy ? kTileRows : 1];  // c, 1 / s, label
  const u32 K = a.m.classes, Kp = K | 1u;
  const u64 r0 = u64(blockIdx.x) * kTileRows;
  const u32 rows = u32(min(u64(kTileRows), a.m.rows - r0)), n = rows * K;
  const u32 step_row = kTileRows / K, step_col = kTileRows % K;
  {
    const T* z = static_cast<const T*>(a.m.z) + r0 * a.m.stride;
    u32 row = threadIdx.x / K, col = threadIdx.x % K;
#pragma unroll 4
    for (u32 e = threadIdx.x; e < n; e += kTileRows) {
      tile[row * Kp + col] = to_f32(z[row * a.m.stride + col]);
      row += step_row;
      col += step_col;
      if (col >= K) { col -= K; ++row; }
    }
  }
  __syncthreads();
  if (threadIdx.x < rows) {
    const u64 r = r0 + threadIdx.x;
    float* const z = tile + threadIdx.x * Kp;
    const i32 y = a.label[r];
    float c = 0.f, s = 1.f;
    if (u32(y) < K) {
      RowScalars x = policy_scalars<kPolicy>(a, r);
      x.zy = z[y];
      float m = neg_inf();
      for (u32 k = 0; k < K; ++k) m = fmaxf(m, z[k]);
      const float base = exp_base(m);
      s = 0.f;
      for (u32 k = 0; k < K; ++k) {
        const float e = exp_fast(z[k] - base);
        s += e;
        if constexpr (kPolicy) z[k] = e;
      }
      c = finish_row<kPolicy>(a, r, x, m, s, true);
    } else {
      skip_row<kPolicy>(a, r, true);
    }
    if constexpr (kPolicy) row_data[threadIdx.x] = make_float4(c, 1.f / s, __int_as_float(y), 0.f);
  }
  if constexpr (kPolicy) {
    if (!a.out.grad) return;
    __syncthreads();
    T* const g = static_cast<T*>(a.out.grad) + r0 * a.out.grad_stride;
    float* const h = a.out.hess ? a.out.hess + r0 * a.out.hess_stride : nullptr;
    u32 row = threadIdx.x / K, col = threadIdx.x % K;
#pragma unroll 4
    for (u32 e = threadIdx.x; e < n; e += kTileRows) {
      const float4 d = row_data[row];
      const float p = tile[row * Kp + col] * d.y;
      const bool none = d.x == 0.f;
      g[row * a.out.grad_stride + col] = from_f32<T>(none ? 0.f : margin_grad(d.x, p, col == u32(__float_as_int(d.z))));
      if (h) h[row * a.out.hess_stride + col] = none ? 0.f : margin_hess(d.x, p);
      row += step_row;
      col += step_col;
      if (col >= K) { col -= K; ++row; }
    }
  }
}

// ---- the backward pass alone: the row's norm is given, so every element is
// on its own.
// The row's coefficient, 0 where the row has no label or no class.
__device__ __forceinline__ float grad_weight(const GradArgs& a, u64 r, i32 y, float2 n) {
  return u32(y) < a.m.classes && !(n.x == neg_inf() && n.y == 0.f) ? a.weight[r] : 0.f;
}

// G threads take a piece of G * U vectors of a row.
template <class T, int G, int U>
__global__ void __launch_bounds__(256) k_log_prob_grad(GradArgs a, u32 pieces) {
  const u64 id = u64(blockIdx.x) * (256 / G) + threadIdx.x / G;
  const u64 r = id / pieces;
  if (r >= a.m.rows) return;
  const u32 j0 = u32(id - r * pieces) * (G * U) + threadIdx.x % G;
  const i32 y = a.label[r];
  const float2 n = a.norm[r];
  const float c = grad_weight(a, r, y, n);
  const RowCut<T> cut(static_cast<const T*>(a.m.z) + r * a.m.stride, a.m.classes);
  const u32 nvec = cut.vectors();
  T* const g = static_cast<T*>(a.out.grad) + r * a.out.grad_stride;
  float* const h = a.out.hess ? a.out.hess + r * a.out.hess_stride : nullptr;
  if (c == 0.f) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (j0 + i * G < nvec) zero_vector(cut, j0 + i * G, g, h);
    return;
  }
  Vec<T> v[U];
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (j0 + i * G < nvec) v[i] = cut.load(j0 + i * G, neg_inf());
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (j0 + i * G < nvec) grad_vector(cut, j0 + i * G, v[i], y, c, n.x, n.y, 1.f, g, h);
}

// Few classes: a block takes kTileRows rows, adjacent threads adjacent elements.
template <class T>
__global__ void __launch_bounds__(kTileRows) k_log_prob_grad_tile(GradArgs a) {
  __shared__ float4 row_data[kTileRows];  // c, norm, label
  const u32 K = a.m.classes;
  const u64 r0 = u64(blockIdx.x) * kTileRows;
  const u32 rows = u32(min(u64(kTileRows), a.m.rows - r0)), n = rows * K;
  if (threadIdx.x < rows) {
    const u64 r = r0 + threadIdx.x;
    const i32 y = a.label[r];
    const float2 nm = a.norm[r];
    row_data[threadIdx.x] = make_float4(grad_weight(a, r, y, nm), nm.x, nm.y, __int_as_float(y));
  }
  __syncthreads();
  const T* const z = static_cast<const T*>(a.m.z) + r0 * a.m.stride;
  T* const g = static_cast<T*>(a.out.grad) + r0 * a.out.grad_stride;
  float* const h = a.out.hess ? a.out.hess + r0 * a.out.hess_stride : nullptr;
  const u32 step_row = kTileRows / K, step_col = kTileRows % K;
  u32 row = threadIdx.x / K, col = threadIdx.x % K;
#pragma unroll 4
  for (u32 e = threadIdx.x; e < n; e += kTileRows) {
    const float4 d = row_data[row];
    float gv = 0.f, hv = 0.f;
    if (d.x != 0.f) {
      const float p = exp_fast((to_f32(z[row * a.m.stride + col]) - d.y) - d.z);
      gv = margin_grad(d.x, p, col == u32(__float_as_int(d.w)));
      hv = margin_hess(d.x, p);
    }
    g[row * a.out.grad_stride + col] = from_f32<T>(gv);
    if (h) h[row * a.out.hess_stride + col] = hv;
    row += step_row;
    col += step_col;
    if (col >= K) { col -= K; ++row; }
  }
}

// ---- launches ---------------------------------------------------------------
constexpr u32 kSMs = 148;
constexpr int kMaxDevices = 16;
inline u32 grid_of(u64 blocks) {
  need(blocks < (u64(1) << 31), "too many rows for one launch");
  return u32(blocks);
}
// Vectors of the longest row: one more than its elements fill when rows start
// off the 16-byte boundaries.
template <class T>
u32 row_vectors(const Margins& m) {
  constexpr u64 N = 16 / sizeof(T);
  const bool even = (reinterpret_cast<std::uintptr_t>(m.z) % 16 == 0) && (m.rows <= 1 || m.stride % N == 0);
  return u32((u64(m.classes) + (even ? 0 : N - 1) + N - 1) / N);
}

template <class T, bool kPolicy, int G>
void launch_lanes(const RowArgs& a, u32 per_lane, cudaStream_t s) {
  const u32 grid = grid_of((a.m.rows + 256 / G - 1) / (256 / G));
  if (per_lane <= 1) k_row_loss<T, kPolicy, G, 1><<<grid, 256, 0, s>>>(a);
  else if (per_lane <= 2) k_row_loss<T, kPolicy, G, 2><<<grid, 256, 0, s>>>(a);
  else if (per_lane <= 3) k_row_loss<T, kPolicy, G, 3><<<grid, 256, 0, s>>>(a);
  else if (per_lane <= 4) k_row_loss<T, kPolicy, G, 4><<<grid, 256, 0, s>>>(a);
  else if (per_lane <= 6) k_row_loss<T, kPolicy, G, 6><<<grid, 256, 0, s>>>(a);
  else k_row_loss<T, kPolicy, G, 8><<<grid, 256, 0, s>>>(a);
}

template <class T, bool kPolicy, int NT, int U, int S, int kPerSM>
void launch_ring(const RowArgs& a, u32 blocks, cudaStream_t s) {
  constexpr u32 kShared = u32(NT) * U * S * 16;
  static_assert(kShared * kPerSM <= 220 * 1024, "the rings of an SM's blocks exceed its shared memory");
  auto* const kernel = k_row_loss_ring<T, kPolicy, NT, U, S>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = kShared;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = blocks > 1 ? 1 : 0;
  // one cluster for every place that the device has for one (clusters do not
  // fill it evenly), asked for once a device and cluster size
  static std::atomic<int> places[kMaxDevices][kMaxCluster + 1];
  int dev = 0;
  DP_CUDA(cudaGetDevice(&dev));
  int fit = dev < kMaxDevices ? places[dev][blocks].load(std::memory_order_relaxed) : 0;
  if (fit == 0) {
    DP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kShared)));
    if (blocks > 1) {
      DP_CUDA(cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg));
    } else {
      DP_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, NT, kShared));
      fit *= int(kSMs);
    }
    need(fit > 0, "the device has no place for a row's blocks");
    if (dev < kMaxDevices) places[dev][blocks].store(fit, std::memory_order_relaxed);
  }
  const u32 clusters = u32(a.m.rows < u64(fit) ? a.m.rows : u64(fit));
  cfg.gridDim = dim3(clusters * blocks);
  DP_CUDA((cudaLaunchKernelEx(&cfg, kernel, a, blocks, clusters)));
}

template <class T, bool kPolicy>
void launch_rows_of(const RowArgs& a, cudaStream_t s) {
  if (!a.m.rows) return;
  constexpr u32 V = 8;  // most vectors a lane holds
  const u32 K = a.m.classes, nvec = row_vectors<T>(a.m);
  if (K <= kTileClasses) {
    const size_t shared = size_t(kTileRows) * (K | 1u) * sizeof(float);
    k_row_loss_tile<T, kPolicy><<<grid_of((a.m.rows + kTileRows - 1) / kTileRows), kTileRows, shared, s>>>(a);
  } else if (nvec <= 8 * V) {
    launch_lanes<T, kPolicy, 8>(a, (nvec + 7) / 8, s);
  } else if (nvec <= 32 * V) {
    launch_lanes<T, kPolicy, 32>(a, (nvec + 31) / 32, s);
  } else if (nvec <= 1536 && a.m.rows >= 2 * kSMs) {
    launch_ring<T, kPolicy, 128, 2, 6, 8>(a, 1, s);
  } else {
    // a row over as few blocks as keep most of it in their rings, or, with
    // few rows, over more of them so that the device is filled
    u32 blocks = 1;
    while (blocks < kMaxCluster &&
           ((kPolicy && nvec > blocks * 4096u) || (a.m.rows * blocks * 2 <= kSMs && nvec > blocks * 512u)))
      blocks *= 2;
    launch_ring<T, kPolicy, 512, 2, 6, 2>(a, blocks, s);
  }
  after_launch("row loss");
}

template <class T>
void launch_grad_of(const GradArgs& a, cudaStream_t s) {
  if (!a.m.rows) return;
  const u64 rows = a.m.rows;
  const u32 nvec = row_vectors<T>(a.m);
  constexpr u32 U = 4;
  if (a.m.classes <= kTileClasses) {
    k_log_prob_grad_tile<T><<<grid_of((rows + kTileRows - 1) / kTileRows), kTileRows, 0, s>>>(a);
  } else if (nvec <= 8 * U) {
    k_log_prob_grad<T, 8, U><<<grid_of((rows + 31) / 32), 256, 0, s>>>(a, 1u);
  } else if (nvec <= 32 * U * 2) {
    const u32 pieces = (nvec + 32 * U - 1) / (32 * U);
    k_log_prob_grad<T, 32, U><<<grid_of((rows * pieces + 7) / 8), 256, 0, s>>>(a, pieces);
  } else {
    const u32 pieces = (nvec + 256 * U - 1) / (256 * U);
    k_log_prob_grad<T, 256, U><<<grid_of(rows * pieces), 256, 0, s>>>(a, pieces);
  }
  after_launch("log_prob_grad");
}

}  // namespace
}  // namespace dp
