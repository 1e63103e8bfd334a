// Row kernels of the choice losses (included by one source file a margin type).
//
// The traffic is the margins in and the gradient out; a gradient element also
// costs two exponentials (one for the sum, one for itself: a kept one would
// take the room of two margins), which at 16 a clock and SM is three quarters
// of the time that a 16-bit margin and its gradient take to move.  Everything
// else is kept to few instructions: fp32 arithmetic is done on pairs (add, mul
// and fma .f32x2), maxima of 16-bit margins on packed pairs.
//
// Rows start at any multiple of their element size.  A row is cut on the
// 16-byte boundaries of its own address: whole 16-byte vectors are moved as
// such, the few elements before the first and after the last one by one, so
// that nothing outside the row is read or written.
#pragma once
#include <cstring>
#include <type_traits>

#include "kernels.h"
#include "loss_math.cuh"

namespace dp {
namespace {

// Two fp32 numbers in a register pair.
struct Two {
  u64 v;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two ex2_both(Two x) {
  float a, b;
  x.get(a, b);
  return Two(ex2(a), ex2(b));
}

// 16 bytes of margins as pairs.
template <class T>
struct Vec {
  static constexpr int N = 16 / int(sizeof(T)), P = N / 2;
  static __device__ __forceinline__ void unpack(const uint4& raw, Two (&f)[P]) {
    const u32 w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (sizeof(T) == 4) {
      f[0] = Two(__uint_as_float(w[0]), __uint_as_float(w[1]));
      f[1] = Two(__uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          __half2 h;
          memcpy(&h, &w[i], 4);
          const float2 v = __half22float2(h);
          f[i] = Two(v.x, v.y);
        } else {
          f[i] = Two(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        }
      }
    }
  }
  static __device__ __forceinline__ uint4 pack(const Two (&f)[P]) {
    u32 w[4];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float a, b;
      f[i].get(a, b);
      if constexpr (sizeof(T) == 4) {
        w[2 * i] = __float_as_uint(a);
        w[2 * i + 1] = __float_as_uint(b);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        memcpy(&w[i], &h, 4);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        memcpy(&w[i], &h, 4);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // A vector of -inf, which changes no maximum and no sum.
  static __device__ __forceinline__ uint4 none() {
    const u32 w = sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u);
    return make_uint4(w, w, w, w);
  }
  // The larger of each place of two vectors (a NaN counts as nothing).
  static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
    return make_uint4(larger(a.x, b.x), larger(a.y, b.y), larger(a.z, b.z), larger(a.w, b.w));
  }
  static __device__ __forceinline__ u32 larger(u32 a, u32 b) {
    if constexpr (sizeof(T) == 4) {
      return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    } else {
      typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type x, y;
      memcpy(&x, &a, 4);
      memcpy(&y, &b, 4);
      x = __hmax2(x, y);
      u32 r;
      memcpy(&r, &x, 4);
      return r;
    }
  }
  static __device__ __forceinline__ float largest(const uint4& v) {
    const u32 w = larger(larger(v.x, v.y), larger(v.z, v.w));
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w);
    } else {
      T lo, hi;
      const u16 a = u16(w), b = u16(w >> 16);
      memcpy(&lo, &a, 2);
      memcpy(&hi, &b, 2);
      return fmaxf(to_f32(lo), to_f32(hi));
    }
  }
};

// A row cut on 16-byte boundaries: whole vectors [j0, j1) counted from `base`,
// and the elements [0, head) and [tail, K) outside them.
template <class T>
struct RowCut {
  static constexpr int N = Vec<T>::N;
  const T* z;
  const T* base;
  u32 K, shift, j0, j1, head, tail;
  __device__ __forceinline__ RowCut(const T* row, u32 classes) : z(row), K(classes) {
    shift = u32(reinterpret_cast<std::uintptr_t>(row) & 15) / u32(sizeof(T));
    base = row - shift;
    j0 = shift ? 1 : 0;
    j1 = max(j0, (K + shift) / N);
    head = shift ? min(K, N - shift) : 0;
    tail = min(K, j1 * N - shift);
  }
  // The row's elements outside the whole vectors, dealt to `G` threads.
  template <int G, class F>
  __device__ __forceinline__ void edges(u32 lane, F&& f) const {
#pragma unroll
    for (u32 e = lane; e < 2 * N; e += G) {
      const u32 k = e < N ? e : tail + e - N;
      if (e < N ? e < head : k < K) f(k);
    }
  }
  // The place of element k among the vectors (an edge's is outside [j0, j1)).
  __device__ __forceinline__ u32 vector_of(u32 k) const { return (k + shift) / N; }
};

// Where a row's gradient and curvature go: rows of other arrays addressed by
// the margins' vectors; without a common 16-byte boundary, element by element.
template <class T>
struct RowOut {
  static constexpr int N = Vec<T>::N, P = N / 2;
  T* g;
  float* h;
  bool g16, h16;
  __device__ __forceinline__ RowOut(const MarginGrad& o, u64 r, u32 shift)
      : g(static_cast<T*>(o.grad) + r * o.grad_stride - shift), h(o.hess ? o.hess + r * o.hess_stride - shift : nullptr) {
    g16 = (reinterpret_cast<std::uintptr_t>(g) & 15) == 0;
    h16 = (reinterpret_cast<std::uintptr_t>(h) & 15) == 0;
  }
  __device__ __forceinline__ void store(u32 j, const uint4& v) const {
    T* const at = g + u64(j) * N;
    if (g16) {
      *reinterpret_cast<uint4*>(at) = v;
    } else {
      T part[N];
      memcpy(part, &v, 16);
#pragma unroll
      for (int i = 0; i < N; ++i) at[i] = part[i];
    }
  }
  __device__ __forceinline__ void store_hess(u32 j, const Two (&f)[P]) const {
    float* const at = h + u64(j) * N;
    float v[N];
#pragma unroll
    for (int i = 0; i < P; ++i) f[i].get(v[2 * i], v[2 * i + 1]);
    if (h16) {
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(at + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) at[i] = v[i];
    }
  }
  __device__ __forceinline__ void zero(u32 j) const {
    store(j, make_uint4(0, 0, 0, 0));
    if (h) {
      Two f[P];
#pragma unroll
      for (int i = 0; i < P; ++i) f[i] = Two(0.f);
      store_hess(j, f);
    }
  }
  // An element k of the row, off the vectors.
  __device__ __forceinline__ void put(u32 shift, u32 k, float gv, float hv) const {
    g[u64(shift) + k] = from_f32<T>(gv);
    if (h) h[u64(shift) + k] = hv;
  }
};

// How p_k comes from a margin: 2^((z - base) log2 e + low) * scale, c being
// the derivative by the row's log-probability.
struct RowCoef {
  float c, base, low, scale;
  __device__ __forceinline__ float p(float z) const { return ex2(fmaf(z - base, kLog2e, low)) * scale; }
};
template <class T>
__device__ __forceinline__ void grad_vector(const RowOut<T>& out, u32 j, const uint4& raw, const RowCoef& q) {
  constexpr int P = Vec<T>::P;
  Two f[P], e[P];
  Vec<T>::unpack(raw, f);
#pragma unroll
  for (int i = 0; i < P; ++i) f[i] = ex2_both(fma(f[i] + Two(-q.base), Two(kLog2e), Two(q.low)));
#pragma unroll
  for (int i = 0; i < P; ++i) e[i] = f[i] * Two(-q.c * q.scale);
  out.store(j, Vec<T>::pack(e));
  if (out.h) {
    const float size = fabsf(q.c), least = size * 1e-16f;  // (margin_hess on pairs)
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const Two p = f[i] * Two(q.scale);
      float a, b;
      (fma(p, Two(-1.f), Two(1.f)) * p * Two(2.f * size)).get(a, b);
      e[i] = Two(a < least ? least : a, b < least ? least : b);
    }
    out.store_hess(j, e);
  }
}
// The same of U vectors D apart, of those below j1: without a curvature all are
// computed before the first is stored, so that their exponentials overlap.
template <class T, int U, int D>
__device__ __forceinline__ void grad_vectors(const RowOut<T>& out, u32 j, u32 j1, uint4 (&v)[U], const RowCoef& q) {
  if (out.h) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u * D < j1) grad_vector(out, j + u * D, v[u], q);
    return;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    constexpr int P = Vec<T>::P;
    Two f[P];
    Vec<T>::unpack(v[u], f);
#pragma unroll
    for (int i = 0; i < P; ++i)
      f[i] = ex2_both(fma(f[i] + Two(-q.base), Two(kLog2e), Two(q.low))) * Two(-q.c * q.scale);
    v[u] = Vec<T>::pack(f);
  }
  if (out.g16) {
    uint4* const at = reinterpret_cast<uint4*>(out.g) + j;
    if (j + (U - 1) * D < j1) {
#pragma unroll
      for (int u = 0; u < U; ++u) at[u * D] = v[u];
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j + u * D < j1) at[u * D] = v[u];
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j + u * D < j1) out.store(j + u * D, v[u]);
  }
}
// Element k of the row by itself.
template <class T>
__device__ __forceinline__ void grad_element(const RowOut<T>& out, const RowCut<T>& cut, u32 k, i32 y, const RowCoef& q) {
  float gv = 0.f, hv = 0.f;
  if (q.c != 0.f) {
    const float p = q.p(to_f32(cut.z[k]));
    gv = margin_grad(q.c, p, k == u32(y));
    hv = margin_hess(fabsf(q.c), p);
  }
  out.put(cut.shift, k, gv, hv);
}
// The label's element once more, by the thread that has written its vector.
template <class T>
__device__ __forceinline__ void grad_label(const RowOut<T>& out, const RowCut<T>& cut, i32 y, float zy, const RowCoef& q) {
  out.g[u64(cut.shift) + u32(y)] = from_f32<T>(margin_grad(q.c, q.p(zy), true));
}

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

// A sum of exponentials relative to `from`, made relative to `to` >= from.  A
// part that is masked throughout has from = -inf and the sum 0 (or NaN).
__device__ __forceinline__ float rebase(float s, float from, float to) {
  return from == neg_inf() ? s : s * exp_fast(from - to);
}
// A thread's running maximum and sum, joined with U more vectors.
template <class T, int U>
__device__ __forceinline__ void join_vectors(const uint4 (&v)[U], float& m, float& s) {
  uint4 w = v[0];
#pragma unroll
  for (int u = 1; u < U; ++u) w = Vec<T>::larger(w, v[u]);
  const float top = fmaxf(m, Vec<T>::largest(w));
  s = rebase(s, m, top);
  m = top;
  const Two b(-exp_base(top));
  Two sum[2] = {Two(s, 0.f), Two(0.f)};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    Two f[Vec<T>::P];
    Vec<T>::unpack(v[u], f);
#pragma unroll
    for (int i = 0; i < Vec<T>::P; ++i) sum[i & 1] = sum[i & 1] + ex2_both((f[i] + b) * Two(kLog2e));
  }
  float x, y;
  (sum[0] + sum[1]).get(x, y);
  s = x + y;
}
__device__ __forceinline__ void join_element(float z, float& m, float& s) {
  const float top = fmaxf(m, z);
  s = rebase(s, m, top) + exp_fast(z - exp_base(top));
  m = top;
}

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
__device__ __forceinline__ void cluster_put(i32* at, u32 rank, i32 v) {
  const u32 here = u32(__cvta_generic_to_shared(at));
  u32 there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(rank));
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(there), "r"(v) : "memory");
}
constexpr u32 kMaxCluster = 8;

// The maximum and the sum over the blocks of a cluster, in the order of their
// ranks: every block gets the same two numbers.
__device__ __forceinline__ void cluster_join(float2* parts, u32 blocks, float& m, float& s) {
  // Only the warp that has written to the other blocks arrives with release:
  // it would make the others wait for their last row's gradients to arrive.
  if (threadIdx.x < 32) {
    if (threadIdx.x < blocks) cluster_put(parts + cluster_rank(), threadIdx.x, make_float2(m, s));
    __syncwarp();
    cluster_arrive();
  } else {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  }
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

// G lanes of a warp a row, V vectors a lane, kept in registers (with eight, the
// policy loss has 56 to 84 bytes a thread of a 16-bit row in local memory, of an
// fp32 row 4 to 20: four blocks an SM leave 64 registers): one read, no
// barrier, and enough warps for memory to stay busy.  134M fp32 margins in rows
// of 1000: forward and backward 157 us, 6.9 TB/s (bound by DRAM); bf16 in rows
// of 2048: 95 us, 5.7 TB/s (DRAM and the exponential unit).
template <class T, bool kPolicy, int G, int V>
__global__ void __launch_bounds__(256, 4) k_row_loss(RowArgs a) {
  const u32 lane = threadIdx.x % G;
  const u64 r = u64(blockIdx.x) * (256 / G) + threadIdx.x / G;
  const bool in = r < a.m.rows;
  const i32 y = in ? a.label[r] : -1;
  const bool live = u32(y) < a.m.classes;
  const RowCut<T> cut(static_cast<const T*>(a.m.z) + (in ? r : 0) * a.m.stride, a.m.classes);
  const uint4* const z16 = reinterpret_cast<const uint4*>(cut.base);
  float m = neg_inf(), s = 0.f;
  uint4 v[V];
  RowScalars x;
  if (live) {
    x = policy_scalars<kPolicy>(a, r);
    x.zy = to_f32(cut.z[y]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const u32 j = cut.j0 + lane + i * G;
      v[i] = j < cut.j1 ? z16[j] : Vec<T>::none();
    }
    if (cut.head || cut.tail < cut.K) cut.template edges<G>(lane, [&](u32 k) { join_element(to_f32(cut.z[k]), m, s); });
    join_vectors<T, V>(v, m, s);
  }
  const float top = lanes_reduce<G>(m, MaxOp());  // (the lanes of a warp reduce together, whatever their rows)
  s = lanes_reduce<G>(rebase(s, m, top), SumOp());
  float c = 0.f;
  if (live) c = finish_row<kPolicy>(a, r, x, top, s, lane == 0);
  else if (in) skip_row<kPolicy>(a, r, lane == 0);
  __syncwarp();  // (a gradient in the margins' place: every lane has read its label's margin)
  if constexpr (kPolicy) {
    if (!a.out.grad || !in) return;
    const RowOut<T> out(a.out, r, cut.shift);
    const RowCoef q{c, exp_base(top), 0.f, inverse(s)};
    if (c == 0.f) {
      for (u32 j = cut.j0 + lane; j < cut.j1; j += G) out.zero(j);
    } else {
      constexpr int U = V == 6 ? 3 : (V == 8 ? 4 : V);  // (V is a multiple of it)
#pragma unroll
      for (int i = 0; i < V; i += U) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = v[i + u];
        grad_vectors<T, U, G>(out, cut.j0 + lane + i * G, cut.j1, w, q);
      }
    }
    if (cut.head || cut.tail < cut.K)
      cut.template edges<G>(lane, [&](u32 k) { grad_element(out, cut, k, y, q); });
    if (c != 0.f) {
      const u32 jy = cut.vector_of(u32(y));
      if (jy >= cut.j0 && jy < cut.j1 && (jy - cut.j0) % G == lane) grad_label(out, cut, y, x.zy, q);
    }
  }
}

// ---- long rows --------------------------------------------------------------
// A block, or a cluster of `blocks` blocks, a row.  Every thread streams its
// own vectors through its own places of a ring in shared memory, by
// asynchronous copies that run ahead of it; nothing in the ring is shared, so
// it needs no barrier.  A row that fits in the rings stays there between its
// sum and its gradient (one read of the margins); a longer one is streamed
// twice, the second time mostly from L2.  Blocks come and go with their rows:
// several on an SM, in different places of theirs, keep memory and arithmetic
// busy, and rows without a label, which cost half of the others or less, do
// not leave some blocks with more work than others (8192 x 65,536 bf16, a
// quarter without a label: 336 us, 5.6 TB/s; by resident blocks that take every
// n-th row and copy ahead into the next one 448).  16-bit rows are bound by the
// exponential unit (72 % busy) and DRAM (82 %) together, fp32 rows by DRAM
// (134M margins in rows of 4096: 159 us, 6.8 TB/s); the log-probability alone
// reads 4096 x 65,537 bf16 in 77 us, 6.3 TB/s.
__device__ __forceinline__ void copy_async(u32 shared, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared), "l"(global) : "memory");
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

// One block's share [j0, j1) of a row's whole vectors, in groups of NT * U.
template <class T, int NT, int U>
struct RowShare {
  u32 j0 = 0, j1 = 0;
  RowShare() = default;
  // (the blocks of a cluster are a power of two)
  __device__ __forceinline__ RowShare(const RowCut<T>& cut, u32 rank, u32 blocks) {
    const u32 n = cut.j1 - cut.j0, per = (n + blocks - 1) >> (31 - __clz(blocks));
    j0 = cut.j0 + min(n, rank * per);
    j1 = min(cut.j1, j0 + per);
  }
  __device__ __forceinline__ u32 groups() const { return (j1 - j0 + NT * U - 1) / (NT * U); }
};

template <class T, bool kPolicy, int NT, int U, int S, int kPerSM>
__global__ void __launch_bounds__(NT, kPerSM) k_row_loss_ring(RowArgs a, u32 blocks) {
  constexpr int kWarps = NT / 32;
  extern __shared__ uint4 ring[];  // [S][U][NT]
  __shared__ float2 warp_part[kWarps];
  __shared__ float2 block_part[kMaxCluster];
  __shared__ float row_c;
  __shared__ i32 row_label;
  const u32 t = threadIdx.x, rank = blocks > 1 ? cluster_rank() : 0;
  const u64 r = blocks > 1 ? blockIdx.x / blocks : blockIdx.x;
  // Whether the row has a label decides which barriers its threads meet at, so
  // one thread reads it for all of them: were the labels written while the
  // kernel runs, the results would be of no use, but every thread would still
  // come to the same barriers.
  i32 y;
  if (blocks > 1) {
    cluster_arrive();  // (every block runs before another one writes to its memory)
    cluster_wait();
    if (rank == 0 && t < 32) {
      const i32 mine = __shfl_sync(0xffffffffu, a.label[r], 0);
      if (t < blocks) cluster_put(&row_label, t, mine);
      __syncwarp();
    }
    cluster_arrive();
    cluster_wait();
    y = row_label;
  } else if (kWarps > 1) {
    if (t == 0) row_label = a.label[r];
    __syncthreads();
    y = row_label;
  } else {
    y = __shfl_sync(0xffffffffu, a.label[r], 0);
  }
  const bool live = u32(y) < a.m.classes, backward = kPolicy && a.out.grad != nullptr;
  const RowCut<T> cut(static_cast<const T*>(a.m.z) + r * a.m.stride, a.m.classes);
  const RowShare<T, NT, U> share(cut, rank, blocks);
  const u32 n = share.j1 - share.j0, groups = share.groups();
  const bool ragged = rank == 0 && (cut.head || cut.tail < cut.K);
  if (!live) {
    skip_row<kPolicy>(a, r, rank == 0 && t == 0);
    if constexpr (kPolicy) {
      if (!backward) return;
      const RowOut<T> out(a.out, r, cut.shift);
      const RowCoef none{0.f, 0.f, 0.f, 0.f};
      if (ragged) cut.template edges<NT>(t, [&](u32 k) { grad_element(out, cut, k, y, none); });
      for (u32 j = share.j0 + t; j < share.j1; j += NT) out.zero(j);
    }
    return;
  }
  const bool again = backward && groups > S;  // the ring does not hold the share
  const uint4* const from = reinterpret_cast<const uint4*>(cut.base) + share.j0 + t;
  const u32 ring_at = u32(__cvta_generic_to_shared(ring + t));
  u32 in_group = 0, in_slot = 0, in_left = again ? 2 * groups : groups;
  auto issue = [&]() {
    if (in_left) {
      const uint4* const src = from + u64(in_group) * (U * NT);
      const u32 to = ring_at + in_slot * (U * NT * 16), left = n - in_group * (U * NT);
      if (left >= U * NT) {
#pragma unroll
        for (int u = 0; u < U; ++u) copy_async(to + u * (NT * 16), src + u * NT);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (t + u * NT < left) copy_async(to + u * (NT * 16), src + u * NT);
      }
      in_group = in_group + 1 == groups ? 0 : in_group + 1;
      in_slot = in_slot + 1 == S ? 0 : in_slot + 1;
      --in_left;
    }
    copy_commit();  // (empty groups too: the count of groups under way stays S)
  };
#pragma unroll
  for (int i = 0; i < S; ++i) issue();

  RowScalars x;
  const float zy = to_f32(cut.z[y]);
  if (t < 32) {
    x = policy_scalars<kPolicy>(a, r);
    x.zy = zy;
  }
  float m = neg_inf(), s = 0.f;
  if (ragged) cut.template edges<NT>(t, [&](u32 k) { join_element(to_f32(cut.z[k]), m, s); });
  const bool stays = backward && !again;
  u32 slot = 0;
#pragma unroll 1
  for (u32 i = 0; i < groups; ++i) {
    copy_wait<S>(stays ? S - 1 - i : S - 1);
    const uint4* const at = ring + slot * (U * NT) + t;
    const u32 left = n - i * (U * NT);
    if (left >= U * NT) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = at[u * NT];
      join_vectors<T, U>(v, m, s);
    } else {  // the last, short group: only as many vectors as there are
#pragma unroll 1
      for (u32 k = t; k - t < left; k += NT) {
        const uint4 v[1] = {k < left ? at[k - t] : Vec<T>::none()};
        join_vectors<T, 1>(v, m, s);
      }
    }
    slot = slot + 1 == S ? 0 : slot + 1;
    if (!stays) issue();
  }
  // the pairs of the threads, then of the warps (every warp alike), then of the blocks
  const float wm = lanes_reduce<32>(m, MaxOp());
  s = lanes_reduce<32>(rebase(s, m, wm), SumOp());
  m = wm;
  if constexpr (kWarps > 1) {
    if ((t & 31) == 0) warp_part[t >> 5] = make_float2(m, s);
    __syncthreads();
    const float2 p = warp_part[t & (kWarps - 1)];
    m = lanes_reduce<kWarps>(p.x, MaxOp());
    s = lanes_reduce<kWarps>(rebase(p.y, p.x, m), SumOp());
  }
  if (blocks > 1) cluster_join(block_part, blocks, m, s);
  // the loss and its derivative are one warp's work
  RowCoef q{0.f, exp_base(m), 0.f, inverse(s)};
  if (t < 32) {
    q.c = finish_row<kPolicy>(a, r, x, m, s, rank == 0 && t == 0);
    if (kWarps > 1 && t == 0) row_c = q.c;
  }
  if constexpr (kPolicy) {
    if (!backward) return;
    if constexpr (kWarps > 1) {
      __syncthreads();
      q.c = row_c;
    } else {
      __syncwarp();  // (in place: the label's margin has been read)
    }
    const RowOut<T> out(a.out, r, cut.shift);
    if (ragged) cut.template edges<NT>(t, [&](u32 k) { grad_element(out, cut, k, y, q); });
    u32 j = share.j0 + t;
    if (q.c == 0.f) {
      copy_wait<1>(0);  // (a block does not end with copies under way)
      for (; j < share.j1; j += NT) out.zero(j);
      return;
    }
    if (stays) slot = 0;
#pragma unroll 1
    for (u32 i = 0; i < groups; ++i) {
      if (again) copy_wait<S>(S - 1);
      const uint4* const at = ring + slot * (U * NT) + t;
      if (share.j1 - (j - t) >= U * NT) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = at[u * NT];
        grad_vectors<T, U, NT>(out, j, share.j1, v, q);
      } else {
#pragma unroll 1
        for (u32 k = j; k < share.j1; k += NT) {
          uint4 v[1] = {at[k - j]};
          grad_vectors<T, 1, NT>(out, k, share.j1, v, q);
        }
      }
      j += U * NT;
      slot = slot + 1 == S ? 0 : slot + 1;
      if (again) issue();
    }
    const u32 jy = cut.vector_of(u32(y));
    if (jy >= share.j0 && jy < share.j1 && (jy - share.j0) % NT == t) grad_label(out, cut, y, zy, q);
  }
}

// ---- the backward pass alone: the row's norm is given, so every element is
// on its own.

// The row's coefficient, 0 where the row has no label or no class.
__device__ __forceinline__ float grad_weight(const GradArgs& a, u64 r, i32 y, float2 n) {
  return u32(y) < a.m.classes && !(n.x == neg_inf() && n.y == 0.f) ? a.weight[r] : 0.f;
}

// G threads take a piece of G * U vectors of a row (the first one its edges
// too).  Bound by DRAM: 4096 x 65,536 bf16, a quarter without a label, 153 us,
// 6.1 TB/s; 134M fp32 margins 162 us, 6.6 TB/s.
template <class T, int G, int U>
__global__ void __launch_bounds__(256) k_log_prob_grad(GradArgs a, u32 pieces) {
  const u64 id = u64(blockIdx.x) * (256 / G) + threadIdx.x / G;
  const u64 r = pieces > 1 ? id / pieces : id;
  if (r >= a.m.rows) return;
  const u32 piece = u32(id - r * pieces), lane = threadIdx.x % G;
  const i32 y = a.label[r];
  const float2 n = a.norm[r];
  const RowCoef q{grad_weight(a, r, y, n), n.x, -n.y * kLog2e, 1.f};
  const RowCut<T> cut(static_cast<const T*>(a.m.z) + r * a.m.stride, a.m.classes);
  const RowOut<T> out(a.out, r, cut.shift);
  const uint4* const z16 = reinterpret_cast<const uint4*>(cut.base);
  const u32 j0 = cut.j0 + piece * (G * U), j = j0 + lane;
  if (piece == 0 && (cut.head || cut.tail < cut.K))
    cut.template edges<G>(lane, [&](u32 k) { grad_element(out, cut, k, y, q); });
  if (q.c == 0.f) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (j + i * G < cut.j1) out.zero(j + i * G);
    return;
  }
  // (read before this thread overwrites its vector in place)
  const u32 jy = cut.vector_of(u32(y));
  const bool labels = jy >= j0 && jy < cut.j1 && jy < j0 + G * U && (jy - j0) % G == lane;
  const float zy = labels ? to_f32(cut.z[y]) : 0.f;
  uint4 v[U];
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (j + i * G < cut.j1) v[i] = z16[j + i * G];
  grad_vectors<T, U, G>(out, j, cut.j1, v, q);
  if (labels) grad_label(out, cut, y, zy, q);
}

// ---- few classes: one thread a row, the row in its registers.  Rows that are
// a power of two of bytes, up to 64, and lie on its boundaries are moved by
// the thread itself; others go through shared memory, where a block stages
// them as they lie in memory, each thread puts its gradient back in its row's
// place, and the block copies the gradients out: memory is read and written in
// whole lines whatever the row length.  A row costs one thread about a hundred
// instructions and ten to twenty a class.
struct TileArgs {
  RowArgs row;
  const float2* norm;    // the backward pass alone: the rows' norms
  const float* weight;   // and the loss's derivatives
};
enum TileMode { kTileLogProb, kTilePolicy, kTileGrad };
constexpr u32 kTileClasses = 64;  // the most that its registers hold

// Copies `rows` rows of K (at most KT) elements between memory (`stride`
// apart) and a tile of NT rows without gaps; whole vectors when the rows have
// no gaps either.
template <class U, bool kIn, int KT, int NT>
__device__ __forceinline__ void copy_rows(U* tile, U* mem, u32 rows, u32 K, u64 stride) {
  const u32 n = rows * K, t = threadIdx.x;
  if (stride == K && (reinterpret_cast<std::uintptr_t>(mem) & 15) == 0) {
    constexpr u32 N = 16 / sizeof(U);
    constexpr int kMost = (KT * int(sizeof(U)) + 15) / 16;
    uint4 *const a = reinterpret_cast<uint4*>(tile) + t, *const b = reinterpret_cast<uint4*>(mem) + t;
    const u32 nv = n / N;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      if (t + i * NT < nv) {
        if (kIn) copy_async(u32(__cvta_generic_to_shared(a + i * NT)), b + i * NT);
        else b[i * NT] = a[i * NT];
      }
    }
    const u32 e = nv * N + t;  // (fewer elements than threads are left)
    if (e < n) {
      if (kIn) tile[e] = mem[e];
      else mem[e] = tile[e];
    }
    if (kIn) {
      copy_commit();
      copy_wait<1>(0);
    }
  } else {
    const u32 step_row = NT / K, step_col = NT % K;
    u32 row = t / K, col = t % K;
#pragma unroll 4
    for (u32 e = t; e < n; e += NT) {
      if (kIn) tile[e] = mem[row * stride + col];
      else mem[row * stride + col] = tile[e];
      row += step_row;
      col += step_col;
      if (col >= K) { col -= K; ++row; }
    }
  }
}

// Turns a row's margins (-inf past its K classes) into probabilities and
// writes the row's results; c: in, the loss's derivative where it is given;
// out, the one to go by, 0 for a row without gradient.
template <TileMode kMode, int KT>
__device__ __forceinline__ void tile_row(const TileArgs& t, u64 r, u32 K, bool live, RowScalars& x, float2 norm, float& c,
                                         float (&z)[KT]) {
  if (!live) {
    if constexpr (kMode != kTileGrad) skip_row<kMode == kTilePolicy>(t.row, r, true);
    c = 0.f;
    return;
  }
  float m = norm.x, low = -norm.y * kLog2e;
  if constexpr (kMode != kTileGrad) {
    m = z[0];
#pragma unroll
    for (int k = 1; k < KT; ++k) m = fmaxf(m, z[k]);
    low = 0.f;
  }
  const Two base(-exp_base(m));
  Two sum(0.f);
#pragma unroll
  for (int k4 = 0; k4 < KT; k4 += 4) {
    if (KT <= 16 || u32(k4) < K) {
#pragma unroll
      for (int k = k4; k < (k4 + 4 < KT ? k4 + 4 : KT); k += 2) {
        const Two e = ex2_both(fma(Two(z[k], k + 1 < KT ? z[k + 1 < KT ? k + 1 : k] : neg_inf()) + base, Two(kLog2e), Two(low)));
        sum = sum + e;
        float past;
        e.get(z[k], k + 1 < KT ? z[k + 1 < KT ? k + 1 : k] : past);
      }
    }
  }
  if constexpr (kMode != kTileGrad) {
    float s, odd;
    sum.get(s, odd);
    s += odd;
    c = finish_row<kMode == kTilePolicy>(t.row, r, x, m, s, true);
    const float scale = inverse(s);
#pragma unroll
    for (int k = 0; k < KT; ++k) z[k] *= scale;
  }
}
// Threads of a warp that read the same place of rows `words` words long meet
// in a bank when they are this far apart.
__host__ __device__ constexpr u32 bank_spread(u32 words) {
  u32 spread = 32;
  while (spread > 1 && words % (64 / spread) == 0) spread /= 2;
  return spread;
}
template <class T>
__host__ __device__ constexpr u32 row_words(u32 K) {
  return K * sizeof(T) % 4 ? 1 : u32(K * sizeof(T) / 4);
}
// Rows so long that four threads or fewer apart meet: each thread begins its
// row at a place of its own and goes round.
constexpr u32 kTurnSpread = 4;

// NT rows a block; KT: the row length (kExact) or the most that it may be.  fp32
// rows are bound by DRAM (6.7M x 10, forward and backward: 107 us, 6.5 TB/s),
// 16-bit ones by instructions (the same in bf16: 93 us, 4.6 TB/s).
template <class T, TileMode kMode, int KT, int NT, bool kExact, bool kTurn>
__global__ void __launch_bounds__(NT) k_row_tile(TileArgs t, u32 spread_given) {
  extern __shared__ uint4 tile16[];
  const RowArgs& a = t.row;
  const u32 K = kExact ? u32(KT) : a.m.classes, spread = kExact ? bank_spread(row_words<T>(KT)) : spread_given;
  T* const tile = reinterpret_cast<T*>(tile16);
  float* const htile = reinterpret_cast<float*>(tile16 + (NT * K * u32(sizeof(T)) + 15) / 16);
  const u64 r0 = u64(blockIdx.x) * NT, r = r0 + threadIdx.x;
  const u32 rows = u32(min(u64(NT), a.m.rows - r0));
  const bool in = threadIdx.x < rows;
  const i32 y = in ? a.label[r] : -1;
  const bool live = u32(y) < K;
  RowScalars x;
  float2 norm = make_float2(0.f, 0.f);
  float c = 0.f;
  if (live) {
    x = policy_scalars<kMode == kTilePolicy>(a, r);
    if constexpr (kMode == kTileGrad) {
      norm = t.norm[r];
      if (!(norm.x == neg_inf() && norm.y == 0.f)) c = t.weight[r];
    }
  }
  copy_rows<T, true, KT, NT>(tile, const_cast<T*>(static_cast<const T*>(a.m.z)) + r0 * a.m.stride, rows, K, a.m.stride);
  __syncthreads();
  const bool backward = kMode == kTileGrad || (kMode == kTilePolicy && a.out.grad != nullptr);
  if (in) {
    T* const mine = tile + threadIdx.x * K;
    const u32 turn = kTurn ? (threadIdx.x & 31) / spread * (4 / u32(sizeof(T))) : 0;
    auto place = [&](u32 k) {  // the class that register k holds
      const u32 at = turn + k;
      return kTurn && at >= K ? at - K : at;
    };
    float z[KT];
#pragma unroll
    for (int k = 0; k < KT; ++k) z[k] = u32(k) < K ? to_f32(mine[place(k)]) : neg_inf();
    if (kMode != kTileGrad && live) x.zy = to_f32(mine[y]);
    tile_row<kMode, KT>(t, r, K, live, x, norm, c, z);
    if (backward) {
      float* const mine_h = htile + threadIdx.x * K;
      const bool none = c == 0.f, hess = a.out.hess != nullptr;
      const float size = fabsf(c), down = -c;
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        if (u32(k) < K) {
          const u32 at = place(k);
          mine[at] = from_f32<T>(none ? 0.f : down * z[k]);
          if (hess) mine_h[at] = none ? 0.f : margin_hess(size, z[k]);
          if (at == u32(y)) c = none ? 0.f : c - c * z[k];
        }
      }
      if (!none) mine[y] = from_f32<T>(c);
    }
  }
  if (!backward) return;
  __syncthreads();
  copy_rows<T, false, KT, NT>(tile, static_cast<T*>(a.out.grad) + r0 * a.out.grad_stride, rows, K, a.out.grad_stride);
  if (a.out.hess) copy_rows<float, false, KT, NT>(htile, a.out.hess + r0 * a.out.hess_stride, rows, K, a.out.hess_stride);
}

// A row of B bytes between registers and memory on its boundaries.
template <int B>
struct RowBytes {
  static constexpr int kWord = B < 16 ? B : 16;
  using Word = typename std::conditional<B == 4, u32, typename std::conditional<B == 8, uint2, uint4>::type>::type;
  Word w[B / kWord];
  __device__ __forceinline__ void load(const void* p) {
#pragma unroll
    for (int i = 0; i < B / kWord; ++i) w[i] = static_cast<const Word*>(p)[i];
  }
  __device__ __forceinline__ void store(void* p) const {
#pragma unroll
    for (int i = 0; i < B / kWord; ++i) static_cast<Word*>(p)[i] = w[i];
  }
};
// 10M x 4 fp32, forward and backward with curvature: 107 us, 6.7 TB/s, bound by
// DRAM.
template <class T, TileMode kMode, int K>
__global__ void __launch_bounds__(256) k_row_thread(TileArgs t) {
  const RowArgs& a = t.row;
  const u64 r = u64(blockIdx.x) * 256 + threadIdx.x;
  if (r >= a.m.rows) return;
  const i32 y = a.label[r];
  const bool live = u32(y) < u32(K);
  RowBytes<K * int(sizeof(T))> raw;
  T v[K];
  float z[K];
  RowScalars x;
  float2 norm = make_float2(0.f, 0.f);
  float c = 0.f;
  raw.load(static_cast<const T*>(a.m.z) + r * a.m.stride);
  x = policy_scalars<kMode == kTilePolicy>(a, r);
  if constexpr (kMode == kTileGrad) {
    norm = t.norm[r];
    if (!(norm.x == neg_inf() && norm.y == 0.f)) c = t.weight[r];
  }
  memcpy(v, &raw, sizeof v);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    z[k] = to_f32(v[k]);
    if (k == y) x.zy = z[k];
  }
  tile_row<kMode, K>(t, r, K, live, x, norm, c, z);
  if (kMode == kTileLogProb || (kMode == kTilePolicy && !a.out.grad)) return;
  const bool none = c == 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = from_f32<T>(none ? 0.f : margin_grad(c, z[k], k == y));
  memcpy(&raw, v, sizeof v);
  raw.store(static_cast<T*>(a.out.grad) + r * a.out.grad_stride);
  if (a.out.hess) {
    const float size = fabsf(c);
    RowBytes<K * 4> h;
#pragma unroll
    for (int k = 0; k < K; ++k) z[k] = none ? 0.f : margin_hess(size, z[k]);
    memcpy(&h, z, sizeof z);
    h.store(a.out.hess + r * a.out.hess_stride);
  }
}

// ---- launches ---------------------------------------------------------------
constexpr u32 kSMs = 148;
inline u32 grid_of(u64 blocks) {
  need(blocks < (u64(1) << 31), "too many rows for one launch");
  return u32(blocks);
}
// Whole vectors of the longest row.
template <class T>
u32 row_vectors(const Margins& m) {
  return m.classes / u32(16 / sizeof(T));
}

template <class T, TileMode kMode, int KT, int NT, bool kExact>
void launch_tile_of(const TileArgs& t, cudaStream_t s) {
  const u64 K = t.row.m.classes, size = (NT * K * sizeof(T) + 15) / 16 * 16 + (t.row.out.hess ? NT * K * 4 : 0);
  const u32 spread = bank_spread(row_words<T>(u32(K)));
  // (of the up to eight classes that end at KT none but KT itself can meet so often)
  constexpr bool kMayTurn = bank_spread(row_words<T>(KT)) <= kTurnSpread;
  auto* kernel = k_row_tile<T, kMode, KT, NT, kExact, kExact && kMayTurn>;
  if constexpr (!kExact && kMayTurn)
    if (spread <= kTurnSpread) kernel = k_row_tile<T, kMode, KT, NT, kExact, true>;
  constexpr int kMost = NT * KT * (int(sizeof(T)) + 4) + 16;  // (one value for every call: other threads launch too)
  if constexpr (kMost > 48 * 1024)
    if (size > 48 * 1024) DP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
  kernel<<<grid_of((t.row.m.rows + NT - 1) / NT), NT, size, s>>>(t, spread);
}
// Up to 16 classes by their number, so that nothing is spent on classes that
// are not there (6.7M rows of 10 fp32 classes, forward and backward: 107 us; with
// one variant for 9 to 12 classes, and copies in loops, 161).
template <class T, TileMode kMode, int KT>
void launch_tile_exact(const TileArgs& t, cudaStream_t s) {
  if (int(t.row.m.classes) == KT) launch_tile_of<T, kMode, KT, 256, true>(t, s);
  else if constexpr (KT < 16) launch_tile_exact<T, kMode, KT + 1>(t, s);
}
// Whether every row of an array lies on the boundaries of its B bytes.
inline bool on_boundaries(const void* p, u64 rows, u64 stride, u64 size, u64 B) {
  const u64 unit = B < 16 ? B : 16;
  return !p || (reinterpret_cast<std::uintptr_t>(p) % unit == 0 && (rows <= 1 || stride * size % unit == 0));
}
template <class T, TileMode kMode>
void launch_tile(const TileArgs& t, cudaStream_t s) {
  const RowArgs& a = t.row;
  const u32 K = a.m.classes;
  const u64 B = K * sizeof(T);
  if ((B & (B - 1)) == 0 && B >= 4 && B <= 64 && K <= 16 && on_boundaries(a.m.z, a.m.rows, a.m.stride, sizeof(T), B) &&
      on_boundaries(a.out.grad, a.m.rows, a.out.grad_stride, sizeof(T), B) &&
      on_boundaries(a.out.hess, a.m.rows, a.out.hess_stride, 4, K * 4)) {
    const u32 grid = grid_of((a.m.rows + 255) / 256);
    if constexpr (sizeof(T) == 4)
      if (K == 1) k_row_thread<T, kMode, 1><<<grid, 256, 0, s>>>(t);
    if (K == 2) k_row_thread<T, kMode, 2><<<grid, 256, 0, s>>>(t);
    if (K == 4) k_row_thread<T, kMode, 4><<<grid, 256, 0, s>>>(t);
    if (K == 8) k_row_thread<T, kMode, 8><<<grid, 256, 0, s>>>(t);
    if (K == 16) k_row_thread<T, kMode, 16><<<grid, 256, 0, s>>>(t);
  } else if (K <= 16) {
    launch_tile_exact<T, kMode, (sizeof(T) == 4 ? 2 : 1)>(t, s);  // (one fp32 class is always on its boundaries)
  } else if (K <= 20) {
    launch_tile_of<T, kMode, 20, 128, false>(t, s);
  } else if (K <= 24) {
    launch_tile_of<T, kMode, 24, 128, false>(t, s);
  } else if (K <= 28) {
    launch_tile_of<T, kMode, 28, 128, false>(t, s);
  } else if (K <= 32) {
    launch_tile_of<T, kMode, 32, 128, false>(t, s);
  } else if (K <= 40) {
    launch_tile_of<T, kMode, 40, 128, false>(t, s);
  } else if (K <= 48) {
    launch_tile_of<T, kMode, 48, 128, false>(t, s);
  } else if (K <= 56) {
    launch_tile_of<T, kMode, 56, 128, false>(t, s);
  } else {
    launch_tile_of<T, kMode, 64, 128, false>(t, s);
  }
}

// One thread a row up to 36 fp32 or 24 16-bit classes (67M margins, one thread
// and lanes: 36 fp32 classes 101 and 117 us forward and backward, 40 104 and
// 96; 24 bf16 classes 86 and 105, 32 103 and 82); up to 64 where rows lie off
// the 16-byte boundaries, which lanes would take element by element at both
// ends (33 bf16 classes 84 and 145 us, fp32 98 and 150).
template <class T>
bool use_tile(const Margins& m) {
  const bool even = m.classes * sizeof(T) % 16 == 0 && on_boundaries(m.z, m.rows, m.stride, sizeof(T), 16);
  return m.classes <= (!even ? kTileClasses : sizeof(T) == 4 ? 36 : 24);
}

// (between 2 and 32 lanes, up to four vectors a lane are the next smaller G's)
template <class T, bool kPolicy, int G>
void launch_lanes(const RowArgs& a, u32 nvec, cudaStream_t s) {
  const u32 grid = grid_of((a.m.rows + 256 / G - 1) / (256 / G)), per_lane = (nvec + G - 1) / G;
  // (fp32 rows for two lanes have nine vectors at least, shorter ones a thread)
  constexpr bool kShort = G == 32 || (G == 2 && sizeof(T) == 2);
  if constexpr (kShort) {
    if (per_lane <= 2) k_row_loss<T, kPolicy, G, 2><<<grid, 256, 0, s>>>(a);
    else if (per_lane <= 3) k_row_loss<T, kPolicy, G, 3><<<grid, 256, 0, s>>>(a);
    else if (per_lane <= 4) k_row_loss<T, kPolicy, G, 4><<<grid, 256, 0, s>>>(a);
  }
  if (!kShort || per_lane > 4) {
    if (per_lane <= 5) k_row_loss<T, kPolicy, G, 5><<<grid, 256, 0, s>>>(a);
    else if (per_lane <= 6) k_row_loss<T, kPolicy, G, 6><<<grid, 256, 0, s>>>(a);
    else k_row_loss<T, kPolicy, G, 8><<<grid, 256, 0, s>>>(a);
  }
}

template <class T, bool kPolicy, int NT, int U, int S, int kPerSM>
void launch_ring(const RowArgs& a, u32 blocks, cudaStream_t s) {
  constexpr u32 kShared = u32(NT) * U * S * 16;
  static_assert(kShared * kPerSM <= 220 * 1024, "the rings of an SM's blocks exceed its shared memory");
  auto* const kernel = k_row_loss_ring<T, kPolicy, NT, U, S, kPerSM>;
  if (kShared > 40 * 1024)  // (with the static arrays above the 48 KB that need no leave)
    DP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kShared)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid_of(a.m.rows * blocks));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = kShared;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = blocks > 1 ? 1 : 0;
  DP_CUDA((cudaLaunchKernelEx(&cfg, kernel, a, blocks)));
}

// Blocks of 256 threads a row, at least `blocks`: with few rows, as many as
// the device has room for and the row gives each of them two vectors a thread.
inline u32 few_rows_cluster(u64 rows, u32 nvec, u32 blocks) {
  while (blocks < kMaxCluster && rows * blocks * 2 <= kSMs && nvec > blocks * 512u) blocks *= 2;
  return blocks;
}

// The ring kernel's shapes: threads a row and groups of four vectors a thread
// that their ring holds; as many blocks are resident as the rings leave room
// for, about 24 warps an SM.
enum RingShape { kRing32x3, kRing64x2, kRing64x3, kRing64x4, kRing128x4, kRing256x3, kRing256x4 };
// As few threads as a row keeps busy, for joining their sums costs what about
// four vectors of each take, but as many as half fill the device.  For the
// policy loss the smallest ring that holds the row (134M margins of 4096 bf16
// classes: 92 us by 32 threads x 4 groups and 64 x 3, 103 by 64 x 4; of 3000
// 94 by 32 x 3, 100 by 32 x 4, 110 by 64 x 3; of 16,384 92 by 128 x 4, 99 by
// 64 x 4, 104 by 256 x 3); for the log-probability, which only streams, less
// ring and more rows under way (4096: 43 us by 64 x 2, 48 by 64 x 3, 53 by
// 64 x 4; 8192 43 by 64 x 3, 49 by 32 x 4; 65,536 45 by 256 x 3, 46 by
// 128 x 4, 50 by 64 x 3).
inline RingShape ring_shape(u64 rows, u32 nvec, bool policy) {
  u32 least = 32;
  while (least < 256 && rows * least < u64(kSMs) * 384) least *= 2;
  if (least <= 32 && nvec <= 384) return kRing32x3;
  if (!policy) {
    if (least <= 64 && nvec <= 512) return kRing64x2;
    if (least <= 64 && nvec <= 3072) return kRing64x3;
    if (least <= 128 && nvec <= 6144) return kRing128x4;
    return kRing256x3;
  }
  if (least <= 64 && nvec <= 768) return kRing64x3;
  if (least <= 64 && nvec <= 1024) return kRing64x4;
  if (least <= 128 && nvec <= 2048) return kRing128x4;
  return nvec <= 3072 ? kRing256x3 : kRing256x4;
}

template <class T, bool kPolicy>
void launch_rows_of(const RowArgs& a, cudaStream_t s) {
  if (!a.m.rows) return;
  constexpr u32 V = 8;  // most vectors a lane holds
  const u32 nvec = row_vectors<T>(a.m);
  if (use_tile<T>(a.m)) {
    launch_tile<T, kPolicy ? kTilePolicy : kTileLogProb>(TileArgs{a, nullptr, nullptr}, s);
  } else if (nvec <= 32 * V && a.m.rows <= 16 * kSMs) {
    // few rows: a warp each (64 rows of 1000 fp16 classes: 3.1 us, by 16 lanes 4.6)
    launch_lanes<T, kPolicy, 32>(a, nvec, s);
  } else if (nvec <= 2 * V) {
    // As few lanes as hold the row with up to eight vectors each, for a row's
    // scalars are every lane's work (67M bf16 margins, with up to eight and up
    // to four: rows of 80 56 and 75 us, of 128 63 and 57, of 256 54 and 55, of
    // 300 63 and 84).
    launch_lanes<T, kPolicy, 2>(a, nvec, s);
  } else if (nvec <= 4 * V) {
    launch_lanes<T, kPolicy, 4>(a, nvec, s);
  } else if (nvec <= 8 * V) {
    launch_lanes<T, kPolicy, 8>(a, nvec, s);
  } else if (nvec <= 16 * V) {
    launch_lanes<T, kPolicy, 16>(a, nvec, s);
  } else if (nvec <= 32 * V) {
    launch_lanes<T, kPolicy, 32>(a, nvec, s);
  } else {
    // (whether a gradient is asked for changes nothing: the loss keeps its bits)
    // A row past two rings, the second read coming from L2, is cut over a
    // cluster of blocks (134M margins, past one ring and past two: bf16 65,536
    // classes 119 and 104 us, 131,072 126 and 113; fp32 32,768 202 and 188,
    // 65,536 213 and 200; past four 65,536 fp32 classes take 276).
    u32 blocks = 1;
    while (kPolicy && blocks < kMaxCluster && nvec > blocks * (2u * 256 * 4 * 4)) blocks *= 2;
    switch (ring_shape(a.m.rows, nvec, kPolicy)) {
      case kRing32x3: launch_ring<T, kPolicy, 32, 4, 3, 28>(a, 1, s); break;
      case kRing64x2:
        if constexpr (!kPolicy) launch_ring<T, kPolicy, 64, 4, 2, 24>(a, 1, s);
        break;
      case kRing64x3: launch_ring<T, kPolicy, 64, 4, 3, 16>(a, 1, s); break;
      case kRing64x4:
        if constexpr (kPolicy) launch_ring<T, kPolicy, 64, 4, 4, 12>(a, 1, s);
        break;
      case kRing128x4: launch_ring<T, kPolicy, 128, 4, 4, 6>(a, 1, s); break;
      case kRing256x3: launch_ring<T, kPolicy, 256, 4, 3, 4>(a, few_rows_cluster(a.m.rows, nvec, blocks), s); break;
      case kRing256x4:
        if constexpr (kPolicy) launch_ring<T, kPolicy, 256, 4, 4, 3>(a, few_rows_cluster(a.m.rows, nvec, blocks), s);
        break;
    }
  }
  after_launch("row loss");
}

// G threads a piece of a row, U vectors each.
template <class T, int G>
void launch_grad_pieces(const GradArgs& a, u32 nvec, cudaStream_t s) {
  constexpr u32 U = 4, per_block = 256 / G;
  const u32 pieces = (nvec + G * U - 1) / (G * U);
  k_log_prob_grad<T, G, U><<<grid_of((a.m.rows * pieces + per_block - 1) / per_block), 256, 0, s>>>(a, pieces);
}

template <class T>
void launch_grad_of(const GradArgs& a, cudaStream_t s) {
  if (!a.m.rows) return;
  const u32 nvec = row_vectors<T>(a.m);
  if (use_tile<T>(a.m)) {
    RowArgs row{};
    row.m = a.m;
    row.label = a.label;
    row.out = a.out;
    launch_tile<T, kTileGrad>(TileArgs{row, a.norm, a.weight}, s);
  } else if (sizeof(T) == 2 && nvec <= 8) {  // (fp32 rows this short take a thread)
    if constexpr (sizeof(T) == 2) launch_grad_pieces<T, 2>(a, nvec, s);
  } else if (nvec <= 16) {
    launch_grad_pieces<T, 4>(a, nvec, s);
  } else if (nvec <= 32) {
    launch_grad_pieces<T, 8>(a, nvec, s);
  } else if (nvec <= 64) {
    launch_grad_pieces<T, 16>(a, nvec, s);
  } else if (nvec <= 1024) {
    launch_grad_pieces<T, 32>(a, nvec, s);
  } else {
    launch_grad_pieces<T, 256>(a, nvec, s);
  }
  after_launch("log_prob_grad");
}

}  // namespace
}  // namespace dp
