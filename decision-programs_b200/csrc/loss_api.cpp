// extern "C" entry points of the choice losses (declared in
// include/dp_gbdt.h): argument checks on the host, then asynchronous launches
// on the caller's stream.
#include <cmath>
#include <initializer_list>
#include <memory>

#include "../../include/dp_gbdt.h"
#include "loss.h"

namespace {

using dp::need;
using dp::u64;

// The C boundary: no exception leaves it, not even one of building a message.
template <class F>
int guarded(F&& body) noexcept {
  try {
    body();
    return 0;
  } catch (const std::exception& e) {
    try {
      dp::set_last_error(e.what());
    } catch (...) {
    }
  } catch (...) {
    try {
      dp::set_last_error("unknown error");
    } catch (...) {
    }
  }
  return -1;
}

// Byte range [lo, hi) that rows of `width` elements, `stride` apart, cover.
struct Span {
  u64 lo = 0, hi = 0;
};
Span span_of(const void* p, u64 rows, u64 width, u64 stride, u64 size) {
  const u64 lo = reinterpret_cast<std::uintptr_t>(p);
  return rows && p ? Span{lo, lo + ((rows - 1) * stride + width) * size} : Span{};
}
bool overlap(const Span& a, const Span& b) { return a.lo < b.hi && b.lo < a.hi; }
Span vector_of(const void* p, u64 n, u64 size = 4) { return span_of(p, n, 1, 1, size); }
// Whether a vector touches an element of such rows (the gaps between rows are
// no elements).
bool touches_rows(const Span& v, const void* p, u64 rows, u64 width, u64 stride, u64 size) {
  const Span all = span_of(p, rows, width, stride, size);
  if (!overlap(v, all)) return false;
  if (v.lo <= all.lo) return true;
  const u64 row = (v.lo - all.lo) / (stride * size), at = (v.lo - all.lo) % (stride * size);
  return at < width * size || (row + 1 < rows && all.lo + (row + 1) * stride * size < v.hi);
}

// A check whose message names an argument; it is put together only on failure.
void need_of(bool ok, const char* what, const char* rule) {
  if (!ok) dp::fail(std::string(what) + " " + rule);
}
void check_rows(u64 rows, u64 width, u64 stride, u64 size, const void* p, const char* what) {
  need_of(stride >= width, what, "row stride must cover the classes");
  need_of(stride <= (u64(1) << 40), what, "row stride out of range");
  need_of(rows <= (u64(1) << 62) / 8 / (stride ? stride : 1), what, "size overflows 64-bit byte offsets");
  need_of(rows == 0 || p != nullptr, what, "pointer is null");
  need_of(reinterpret_cast<std::uintptr_t>(p) % size == 0, what, "pointer is not aligned to its type");
}
// Vectors: an address off its type's boundary would fault on the device.
template <class... P>
void check_aligned(const P*... p) {
  need(((reinterpret_cast<std::uintptr_t>(p) % sizeof(P) == 0) && ...), "a vector's pointer is not aligned to its type");
}

dp::Margins margins_of(int32_t dtype, const void* margin, u64 rows, uint32_t classes, u64 stride) {
  need(dtype >= 0 && dtype <= 2, "margin type must be 0 (fp32), 1 (fp16) or 2 (bf16)");
  need(classes >= 1 && classes <= 0x7fffffffu, "the number of classes must be in [1, 2^31)");
  check_rows(rows, classes, stride, dp::margin_bytes(dtype), margin, "margin");
  return dp::Margins{margin, dtype, rows, classes, stride};
}

dp::MarginGrad grad_of(const dp::Margins& m, void* grad, u64 grad_stride, float* hess, u64 hess_stride) {
  dp::MarginGrad g{};
  if (!grad) {
    need(!hess, "the curvature is written with a gradient: the gradient pointer is null");
    return g;
  }
  const u64 size = dp::margin_bytes(m.dtype);
  check_rows(m.rows, m.classes, grad_stride, size, grad, "gradient");
  const Span z = span_of(m.z, m.rows, m.classes, m.stride, size),
             o = span_of(grad, m.rows, m.classes, grad_stride, size);
  need(!overlap(z, o) || (grad == m.z && grad_stride == m.stride),
       "the gradient may take the margins' place (same pointer and row stride) but not overlap them otherwise");
  if (hess) {
    check_rows(m.rows, m.classes, hess_stride, sizeof(float), hess, "curvature");
    const Span h = span_of(hess, m.rows, m.classes, hess_stride, sizeof(float));
    need(!overlap(h, z) && !overlap(h, o), "the curvature overlaps the margins or the gradient");
  }
  g.grad = grad;
  g.grad_stride = grad_stride;
  g.hess = hess;
  g.hess_stride = hess_stride;
  return g;
}

// The vectors that a row call writes beside its gradient touch neither its
// matrices nor each other, and the vectors that it reads only where they are
// the same vector: a row is then read before it is written.
void check_row_outputs(const dp::Margins& m, const dp::MarginGrad& g, std::initializer_list<Span> written,
                       std::initializer_list<Span> read) {
  const u64 size = dp::margin_bytes(m.dtype);
  for (const Span* o = written.begin(); o != written.end(); ++o) {
    need(!touches_rows(*o, m.z, m.rows, m.classes, m.stride, size), "an output vector overlaps the margins");
    need(!touches_rows(*o, g.grad, m.rows, m.classes, g.grad_stride, size) &&
             !touches_rows(*o, g.hess, m.rows, m.classes, g.hess_stride, sizeof(float)),
         "an output vector overlaps the gradient or the curvature");
    for (const Span* p = written.begin(); p != o; ++p) need(!overlap(*o, *p), "two output vectors overlap");
    for (const Span& in : read)
      need(!overlap(*o, in) || (o->lo == in.lo && o->hi == in.hi), "an output vector overlaps an input vector");
  }
  for (const Span& in : read)
    need(!touches_rows(in, g.grad, m.rows, m.classes, g.grad_stride, size) &&
             !touches_rows(in, g.hess, m.rows, m.classes, g.hess_stride, sizeof(float)),
         "the gradient or the curvature overlaps an input vector");
}

dp::PairLoss pair_args(const float* score, const float* ref, const float* weight, float beta, float smoothing,
                       float* loss, float* grad, float* hess, u64 rows, u64 pairs, const Span& offsets = Span{}) {
  need(std::isfinite(beta) && beta > 0.f, "beta must be positive and finite");
  need(smoothing >= 0.f && smoothing <= 0.5f, "label smoothing must be in [0, 0.5]");
  need(rows == 0 || (score != nullptr && grad != nullptr), "score or gradient pointer is null");
  need(pairs == 0 || loss != nullptr, "loss pointer is null");
  check_aligned(score, ref, weight, loss, grad, hess);
  // The outputs' places are written (partial sums too) while scores, weights
  // and offsets are read.
  const Span z = vector_of(score, rows), t = vector_of(ref, rows), o = vector_of(grad, rows), h = vector_of(hess, rows),
             l = vector_of(loss, pairs), w = vector_of(weight, pairs);
  need(!overlap(o, z) && !overlap(o, t), "the gradient overlaps the scores");
  need(!overlap(h, z) && !overlap(h, t) && !overlap(h, o), "the curvature overlaps the scores or the gradient");
  need(!overlap(l, z) && !overlap(l, t) && !overlap(l, o) && !overlap(l, h),
       "the loss overlaps the scores, the gradient or the curvature");
  for (const Span& out : {o, h, l})
    need(!overlap(out, w) && !overlap(out, offsets), "an output overlaps the weights or the item offsets");
  dp::PairLoss a{};
  a.score = score;
  a.ref = ref;
  a.weight = weight;
  a.beta = beta;
  a.smoothing = smoothing;
  a.loss = loss;
  a.grad = grad;
  a.hess = hess;
  return a;
}

}  // namespace

extern "C" {

int dp_log_prob(int32_t dtype, const void* margin, uint64_t rows, uint32_t classes, uint64_t row_stride,
                const int32_t* label, float* log_prob, float* norm, void* stream) {
  return guarded([&] {
    const dp::Margins m = margins_of(dtype, margin, rows, classes, row_stride);
    need(rows == 0 || (label != nullptr && log_prob != nullptr && norm != nullptr),
         "label, log-probability or norm pointer is null");
    need(reinterpret_cast<std::uintptr_t>(norm) % sizeof(float2) == 0, "norm pointer is not aligned to 8 bytes");
    check_aligned(label, log_prob);
    dp::RowArgs a{};
    a.m = m;
    a.label = label;
    a.log_prob = log_prob;
    a.norm = reinterpret_cast<float2*>(norm);
    check_row_outputs(m, a.out, {vector_of(log_prob, rows), vector_of(norm, rows, sizeof(float2))},
                      {vector_of(label, rows)});
    dp::launch_rows(a, false, static_cast<cudaStream_t>(stream));
  });
}

int dp_log_prob_grad(int32_t dtype, const void* margin, uint64_t rows, uint32_t classes, uint64_t row_stride,
                     const int32_t* label, const float* norm, const float* weight, void* grad, uint64_t grad_stride,
                     float* hess, uint64_t hess_stride, void* stream) {
  return guarded([&] {
    const dp::Margins m = margins_of(dtype, margin, rows, classes, row_stride);
    need(rows == 0 || (label != nullptr && norm != nullptr && weight != nullptr && grad != nullptr),
         "label, norm, weight or gradient pointer is null");
    need(reinterpret_cast<std::uintptr_t>(norm) % sizeof(float2) == 0, "norm pointer is not aligned to 8 bytes");
    check_aligned(label, weight);
    const dp::MarginGrad g = grad_of(m, grad, grad_stride, hess, hess_stride);
    check_row_outputs(m, g, {},
                      {vector_of(label, rows), vector_of(norm, rows, sizeof(float2)), vector_of(weight, rows)});
    dp::launch_grad(dp::GradArgs{m, label, reinterpret_cast<const float2*>(norm), weight, g},
                    static_cast<cudaStream_t>(stream));
  });
}

int dp_policy_loss(int32_t dtype, const void* margin, uint64_t rows, uint32_t classes, uint64_t row_stride,
                   const int32_t* label, const float* old_log_prob, const float* ref_log_prob,
                   const float* advantage, const float* weight, float clip_low, float clip_high, float kl,
                   float* loss, float* log_prob, void* grad, uint64_t grad_stride, float* hess,
                   uint64_t hess_stride, void* stream) {
  return guarded([&] {
    const dp::Margins m = margins_of(dtype, margin, rows, classes, row_stride);
    need(rows == 0 || (label != nullptr && old_log_prob != nullptr && advantage != nullptr),
         "label, old log-probability or advantage pointer is null");
    need(rows == 0 || (loss != nullptr && log_prob != nullptr), "loss or log-probability pointer is null");
    check_aligned(label, old_log_prob, ref_log_prob, advantage, weight, loss, log_prob);
    need(clip_low >= 0.f && clip_low <= 1.f, "clip_low must be in [0, 1]");
    need(std::isfinite(clip_high) && clip_high >= 0.f, "clip_high must be finite and not negative");
    need(std::isfinite(kl) && kl >= 0.f, "the KL coefficient must be finite and not negative");
    dp::RowArgs a{};
    a.m = m;
    a.label = label;
    a.loss = loss;
    a.log_prob = log_prob;
    a.out = grad_of(m, grad, grad_stride, hess, hess_stride);
    check_row_outputs(m, a.out, {vector_of(loss, rows), vector_of(log_prob, rows)},
                      {vector_of(label, rows), vector_of(old_log_prob, rows), vector_of(ref_log_prob, rows),
                       vector_of(advantage, rows), vector_of(weight, rows)});
    dp::PolicyRows& p = a.policy;
    p.old_log_prob = old_log_prob;
    p.ref_log_prob = kl != 0.f ? ref_log_prob : nullptr;  // (0 times an infinite term would be NaN)
    p.advantage = advantage;
    p.weight = weight;
    p.clip_low = clip_low;
    p.clip_high = clip_high;
    p.kl = kl;
    dp::launch_rows(a, true, static_cast<cudaStream_t>(stream));
  });
}

int dp_preference_loss(uint64_t rows, const int64_t* item_begin, uint64_t pairs, const float* score,
                       const float* ref_score, const float* weight, float beta, float smoothing, float* loss,
                       float* grad, float* hess, void* stream) {
  return guarded([&] {
    need(rows < (u64(1) << 60) && pairs < (u64(1) << 40), "rows or pairs out of range");
    check_aligned(item_begin);
    need(item_begin != nullptr || rows >= 2 * pairs, "without item offsets every pair needs two rows");
    const dp::PairLoss a =
        pair_args(score, ref_score, weight, beta, smoothing, loss, grad, hess, rows, pairs,
                  item_begin ? vector_of(item_begin, 2 * pairs + 1, sizeof(int64_t)) : Span{});
    dp::launch_preference(a, rows, item_begin, pairs, static_cast<cudaStream_t>(stream));
  });
}

int dp_preference_prepare(uint64_t rows, const int32_t* pair_rows, uint64_t pairs, void* stream, void** out_plan) {
  return guarded([&] {
    need(out_plan != nullptr, "output pointer is null");
    need(rows < (u64(1) << 31) && pairs < (u64(1) << 31), "rows and pairs must be below 2^31");
    need(pairs == 0 || pair_rows != nullptr, "pair pointer is null");
    check_aligned(pair_rows);
    auto plan = std::make_unique<dp::PairPlan>();
    dp::build_pair_plan(*plan, rows, pair_rows, pairs, static_cast<cudaStream_t>(stream));
    *out_plan = plan.release();
  });
}

int dp_preference_run(void* plan, const float* score, const float* ref_score, const float* weight, float beta,
                      float smoothing, float* loss, float* grad, float* hess, void* stream) {
  return guarded([&] {
    need(plan != nullptr, "plan is null");
    const dp::PairPlan& p = *static_cast<dp::PairPlan*>(plan);
    const dp::PairLoss a =
        pair_args(score, ref_score, weight, beta, smoothing, loss, grad, hess, p.rows, p.pairs);
    dp::DeviceGuard g(p.device);
    dp::launch_pair_loss(p, a, static_cast<cudaStream_t>(stream));
  });
}

int dp_preference_free(void* plan) {
  return guarded([&] {
    if (!plan) return;
    dp::PairPlan* p = static_cast<dp::PairPlan*>(plan);
    dp::DeviceGuard g(p->device);
    delete p;
  });
}

}  // extern "C"
