// Scalar parts of the choice losses, shared by their kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "loss.h"

namespace dp {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
// e^x.  The difference z - m is taken before the scaling by log2 e: margins of
// the type's lowest value would overflow if they were scaled first.
__device__ __forceinline__ float exp_fast(float x) { return ex2(x * kLog2e); }
// 1 / s to a last place or so.
__device__ __forceinline__ float inverse(float s) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
  return y;
}

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// A row whose classes are all masked (every margin -inf) has m = -inf and no
// sum; exponents are then taken relative to 0, so that the sum is 0 and not
// NaN, and a NaN margin still makes it NaN.
__device__ __forceinline__ float exp_base(float m) { return m == neg_inf() ? 0.f : m; }

// Log-probability and its two-part norm of a row from its maximum m, the sum
// s of exp(z - exp_base(m)) and the label's margin.  The norm stays in two
// parts because exp((z - m) - log s) keeps its precision at margins far from
// zero, where m + log s would round away what log s says.
__device__ __forceinline__ float row_log_prob(float m, float s, float zy, float2& norm) {
  if (s == 0.f) {  // no class left
    norm = make_float2(neg_inf(), 0.f);
    return neg_inf();
  }
  const float ls = logf(s);
  norm = make_float2(m, ls);
  return (zy - m) - ls;
}

// What a row's loss reads beside its margins; zy: the label's margin.
struct RowScalars {
  float zy = 0.f, old = 0.f, ref = 0.f, adv = 0.f, w = 1.f;
};

// The lesser of two numbers, a NaN where there is one.
__device__ __forceinline__ float least_of(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
constexpr float kMostSlope = 0x1p126f;

// Clipped policy loss of a row and its derivative by the log-probability:
// L = w (-min(r A, clamp(r, 1 - lo, 1 + hi) A) + kl (e^d - d - 1)),
// r = exp(l - old), d = ref - l.  Comparisons keep a NaN ratio NaN.  A masked
// class that was chosen has l = -inf, so that r = 0 and d is infinite.  Ratios
// past fp32's range are held to its largest number (no advantage makes nothing
// of them), and the derivative to kMostSlope in size: an infinite one would make
// NaN of the classes of probability 0, and twice kMostSlope is still finite.
__device__ __forceinline__ float policy_row(const PolicyRows& p, const RowScalars& x, float l, float& loss) {
  if (x.w == 0.f) {
    loss = 0.f;
    return 0.f;
  }
  const float ratio = least_of(exp_fast(l - x.old), FLT_MAX), adv = x.adv;
  const float low = 1.f - p.clip_low, high = 1.f + p.clip_high;
  const float held = ratio < low ? low : (ratio > high ? high : ratio);
  const float s1 = ratio * adv, s2 = held * adv;
  const bool clipped = s1 > s2;
  float v = clipped ? -s2 : -s1;
  float c = clipped ? 0.f : -s1;
  if (p.ref_log_prob) {
    // e^d - d - 1 by its series where the difference would lose it (the first
    // term left out is below 2^-24 of the sum for |d| < 1/2)
    const float d = x.ref - l;
    float t = 1.f / 40320.f;
    t = fmaf(t, d, 1.f / 5040.f);
    t = fmaf(t, d, 1.f / 720.f);
    t = fmaf(t, d, 1.f / 120.f);
    t = fmaf(t, d, 1.f / 24.f);
    t = fmaf(t, d, 1.f / 6.f);
    t = fmaf(t, d, 0.5f);
    const bool near = fabsf(d) < 0.5f;
    // (an infinite d: e^d - d is e^d)
    const float e = exp_fast(d), over = near ? t * d * d : (e - fminf(d, FLT_MAX)) - 1.f;
    v = v + p.kl * over;
    c = c - least_of(p.kl * (near ? over + d : e - 1.f), kMostSlope);
  }
  loss = x.w * v;
  return -least_of(-least_of(x.w * c, kMostSlope), kMostSlope);
}

// Gradient and curvature of c * log p(label) by one margin of probability p.
__device__ __forceinline__ float margin_grad(float c, float p, bool chosen) { return c * ((chosen ? 1.f : 0.f) - p); }
// The softmax objective's diagonal form, |c| max(2 p (1 - p), 1e-16), for
// size = |c|; the comparison lets a NaN through.
__device__ __forceinline__ float margin_hess(float size, float p) {
  const float least = size * 1e-16f, h = (1.f - p) * p * (size + size);
  return h < least ? least : h;
}

// Preference loss of a pair at x = beta * (gap of scores): the loss, its
// derivative and its second derivative by x.  Both sigmoids come from
// e = exp(-|x|), which never overflows and keeps a saturated pair's small one.
struct PairTerms {
  float loss, slope, bend;
};
__device__ __forceinline__ PairTerms pair_terms(float x, float smoothing) {
  const float e = expf(-fabsf(x)), small = log1pf(e), inv = 1.f / (1.f + e);
  const float up = x >= 0.f ? inv : e * inv, down = x >= 0.f ? e * inv : inv;  // sigma(x), sigma(-x)
  const float keep = 1.f - smoothing;
  PairTerms t;
  t.loss = keep * (fmaxf(-x, 0.f) + small);
  if (smoothing != 0.f) t.loss += smoothing * (fmaxf(x, 0.f) + small);  // an infinite x would make 0 * inf of it
  t.slope = smoothing * up - keep * down;
  t.bend = up * down;
  return t;
}
// Curvature of an item over its pairs, with the objectives' floor.
__device__ __forceinline__ float item_hess(float h) { return h < 1e-16f ? 1e-16f : h; }

}  // namespace dp
