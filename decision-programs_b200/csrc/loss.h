// Losses that learn from choices: log-probabilities of a chosen class and
// their backward pass, the clipped policy loss, and the preference loss over
// pairs (dp_log_prob, dp_log_prob_grad, dp_policy_loss, dp_preference_* in
// include/dp_gbdt.h).  Launchers take device pointers, enqueue on `s` and
// never synchronise or allocate.
#pragma once
#include <cuda_runtime.h>

#include "common.h"

namespace dp {

enum MarginType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };
inline u64 margin_bytes(int dtype) { return dtype == kF32 ? 4 : 2; }

// Margins [rows][classes], rows `stride` elements apart.
struct Margins {
  const void* z = nullptr;
  int dtype = kF32;
  u64 rows = 0;
  u32 classes = 0;
  u64 stride = 0;
};
// Gradient in the margins' type and curvature in fp32; null when not wanted.
struct MarginGrad {
  void* grad = nullptr;
  u64 grad_stride = 0;
  float* hess = nullptr;
  u64 hess_stride = 0;
};
struct PolicyRows {
  const float* old_log_prob = nullptr;
  const float* ref_log_prob = nullptr;  // null: no KL term
  const float* advantage = nullptr;
  const float* weight = nullptr;  // null: 1
  float clip_low = 0.f, clip_high = 0.f, kl = 0.f;
};

// Forward (and, for the policy loss, backward) pass over rows: log_prob and
// norm, or loss, log_prob and the gradient.
struct RowArgs {
  Margins m;
  const i32* label = nullptr;
  PolicyRows policy;
  float* loss = nullptr;
  float* log_prob = nullptr;
  float2* norm = nullptr;
  MarginGrad out;
};
// The log-probability's backward pass.
struct GradArgs {
  Margins m;
  const i32* label = nullptr;
  const float2* norm = nullptr;
  const float* weight = nullptr;
  MarginGrad out;
};
// One source file a margin type.
void launch_rows_f32(const RowArgs& a, bool policy, cudaStream_t s);
void launch_rows_f16(const RowArgs& a, bool policy, cudaStream_t s);
void launch_rows_bf16(const RowArgs& a, bool policy, cudaStream_t s);
void launch_grad_f32(const GradArgs& a, cudaStream_t s);
void launch_grad_f16(const GradArgs& a, cudaStream_t s);
void launch_grad_bf16(const GradArgs& a, cudaStream_t s);
inline void launch_rows(const RowArgs& a, bool policy, cudaStream_t s) {
  (a.m.dtype == kF32 ? launch_rows_f32 : a.m.dtype == kF16 ? launch_rows_f16 : launch_rows_bf16)(a, policy, s);
}
inline void launch_grad(const GradArgs& a, cudaStream_t s) {
  (a.m.dtype == kF32 ? launch_grad_f32 : a.m.dtype == kF16 ? launch_grad_f16 : launch_grad_bf16)(a, s);
}

// Scores of items: item i is rows [begin[i], begin[i + 1]) of score (begin
// null: row i); pair p is items 2p (preferred) and 2p + 1.
struct PairLoss {
  const float* score = nullptr;
  const float* ref = nullptr;     // null: no reference model
  const float* weight = nullptr;  // per pair; null: 1
  float beta = 1.f, smoothing = 0.f;
  float* loss = nullptr;  // [pairs]
  float* grad = nullptr;  // [rows]
  float* hess = nullptr;  // [rows] or null
};
void launch_preference(const PairLoss& a, u64 rows, const i64* begin, u64 pairs, cudaStream_t s);

// Any pairs over rows, laid out once: a copy of the pairs, and an entry for
// each row of each pair, sorted by row and within a row by pair; workspace of
// a run (one at a time).
struct PairEntry {
  u32 row;
  u32 pair;  // bit 31 set: the row is the one not preferred
};
// Entries that one warp sums: all their gathers are under way at once, and more
// of them take the registers of other warps (8M pairs over 1M rows: 170 us at
// 128, 178 at 256, 195 at 512).
constexpr u32 kPairChunk = 128;
struct PairPlan {
  u64 rows = 0, pairs = 0;
  int device = 0;
  std::vector<DevBuf<unsigned char>> slabs;  // memory of the views below
  DevBuf<int2> pair;
  DevBuf<PairEntry> entry;
  DevBuf<float2> terms;        // [pairs] derivative by the preferred score, curvature
  DevBuf<float2> head, tail;   // [chunks] sums of rows that reach over chunks
  DevBuf<u32> joins;           // [chunks] which of them end there
  DevBuf<float> gap;           // [rows] score - ref
  PairPlan() = default;
  ~PairPlan();  // the plan's device is current
  PairPlan(const PairPlan&) = delete;
  PairPlan& operator=(const PairPlan&) = delete;
};
// Checks the pairs (device, [pairs][2]: preferred row, other row) and lays
// them out; waits for `s`.  Throws when a pair names a row outside
// [0, rows) or one row twice.
void build_pair_plan(PairPlan& plan, u64 rows, const i32* pair_rows, u64 pairs, cudaStream_t s);
void launch_pair_loss(const PairPlan& p, const PairLoss& a, cudaStream_t s);

}  // namespace dp
