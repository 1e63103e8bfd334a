// Row losses over class margins: log-probability of the label and the clipped
// policy loss (forward and backward), and the backward pass of the
// log-probability alone.
//
// p_k = exp(z_k - m) / s with m = max z, s = sum exp(z - m), both in fp32;
// a gradient is rounded once, to the margins' type, when it is stored.
#include "kernels.h"
#include "loss_math.cuh"

namespace dp {
namespace {

struct RowArgs {
  Margins m;
  const i32* label;
  PolicyRows policy;
  float* loss;
  float* log_prob;
  float2* norm;
  MarginGrad out;
};

template <class Op>
__device__ __forceinline__ float warp_reduce(float v, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
struct MaxOp {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct SumOp {
  __device__ float operator()(float a, float b) const { return a + b; }
};

template <class Op>
__device__ float block_reduce(float v, float init, Op op) {
  __shared__ float part[32];
  v = warp_reduce(v, op);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x < (blockDim.x >> 5) ? part[threadIdx.x] : init;
  if (threadIdx.x < 32) {
    v = warp_reduce(v, op);
    if (threadIdx.x == 0) part[0] = v;
  }
  __syncthreads();
  return part[0];
}

// One block a row; the row is read once for its maximum, once for its sum and
// once for its gradient.
template <class T, bool kPolicy>
__global__ void __launch_bounds__(256) k_row_loss(RowArgs a) {
  const u32 K = a.m.classes;
  for (u64 r = blockIdx.x; r < a.m.rows; r += gridDim.x) {
    const T* z = static_cast<const T*>(a.m.z) + r * a.m.stride;
    const i32 y = a.label[r];
    const bool live = u32(y) < K;
    float m = neg_inf(), s = 0.f, c = 0.f, l = 0.f, loss = 0.f;
    float2 norm = make_float2(0.f, 0.f);
    if (live) {
      for (u32 k = threadIdx.x; k < K; k += blockDim.x) m = fmaxf(m, to_f32(z[k]));
      m = block_reduce(m, neg_inf(), MaxOp());
      for (u32 k = threadIdx.x; k < K; k += blockDim.x) s += expf(to_f32(z[k]) - exp_base(m));
      s = block_reduce(s, 0.f, SumOp());
      l = row_log_prob(m, s, to_f32(z[y]), norm);
      if (kPolicy && s != 0.f) c = policy_row(a.policy, r, l, loss);
    }
    __syncthreads();  // the label's margin is read before a gradient in place overwrites it
    if (threadIdx.x == 0) {
      if (kPolicy) a.loss[r] = loss;
      a.log_prob[r] = l;
      if (!kPolicy) a.norm[r] = norm;
    }
    if (kPolicy && a.out.grad) {
      T* g = static_cast<T*>(a.out.grad) + r * a.out.grad_stride;
      float* h = a.out.hess ? a.out.hess + r * a.out.hess_stride : nullptr;
      for (u32 k = threadIdx.x; k < K; k += blockDim.x) {
        const float p = c != 0.f ? expf(to_f32(z[k]) - m) / s : 0.f;
        g[k] = from_f32<T>(c != 0.f ? margin_grad(c, p, k == u32(y)) : 0.f);
        if (h) h[k] = c != 0.f ? margin_hess(c, p) : 0.f;
      }
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256) k_log_prob_grad(Margins m, const i32* label, const float2* norm,
                                                       const float* weight, MarginGrad out) {
  const u32 K = m.classes;
  for (u64 r = blockIdx.x; r < m.rows; r += gridDim.x) {
    const T* z = static_cast<const T*>(m.z) + r * m.stride;
    T* g = static_cast<T*>(out.grad) + r * out.grad_stride;
    float* h = out.hess ? out.hess + r * out.hess_stride : nullptr;
    const i32 y = label[r];
    const float2 n = norm[r];
    const bool none = n.x == neg_inf() && n.y == 0.f;
    const float c = u32(y) < K && !none ? weight[r] : 0.f;
    for (u32 k = threadIdx.x; k < K; k += blockDim.x) {
      const float p = c != 0.f ? expf((to_f32(z[k]) - n.x) - n.y) : 0.f;
      g[k] = from_f32<T>(c != 0.f ? margin_grad(c, p, k == u32(y)) : 0.f);
      if (h) h[k] = c != 0.f ? margin_hess(c, p) : 0.f;
    }
  }
}

u32 row_blocks(u64 rows) { return u32(rows < (u64(1) << 30) ? rows : u64(1) << 30); }

template <bool kPolicy>
void launch_rows(const RowArgs& a, cudaStream_t s) {
  if (!a.m.rows) return;
  const u32 grid = row_blocks(a.m.rows);
  if (a.m.dtype == kF32) k_row_loss<float, kPolicy><<<grid, 256, 0, s>>>(a);
  else if (a.m.dtype == kF16) k_row_loss<__half, kPolicy><<<grid, 256, 0, s>>>(a);
  else k_row_loss<__nv_bfloat16, kPolicy><<<grid, 256, 0, s>>>(a);
  after_launch("row loss");
}

}  // namespace

void launch_log_prob(const Margins& m, const i32* label, float* log_prob, float2* norm, cudaStream_t s) {
  RowArgs a{};
  a.m = m;
  a.label = label;
  a.log_prob = log_prob;
  a.norm = norm;
  launch_rows<false>(a, s);
}

void launch_policy_loss(const Margins& m, const i32* label, const PolicyRows& p, float* loss, float* log_prob,
                        const MarginGrad& out, cudaStream_t s) {
  RowArgs a{};
  a.m = m;
  a.label = label;
  a.policy = p;
  a.loss = loss;
  a.log_prob = log_prob;
  a.out = out;
  launch_rows<true>(a, s);
}

void launch_log_prob_grad(const Margins& m, const i32* label, const float2* norm, const float* weight,
                          const MarginGrad& out, cudaStream_t s) {
  if (!m.rows) return;
  const u32 grid = row_blocks(m.rows);
  if (m.dtype == kF32) k_log_prob_grad<float><<<grid, 256, 0, s>>>(m, label, norm, weight, out);
  else if (m.dtype == kF16) k_log_prob_grad<__half><<<grid, 256, 0, s>>>(m, label, norm, weight, out);
  else k_log_prob_grad<__nv_bfloat16><<<grid, 256, 0, s>>>(m, label, norm, weight, out);
  after_launch("log_prob_grad");
}

}  // namespace dp
