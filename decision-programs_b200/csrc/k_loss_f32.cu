// Row losses over fp32 margins.
#include "loss_rows.cuh"

namespace dp {

void launch_rows_f32(const RowArgs& a, bool policy, cudaStream_t s) {
  if (policy) launch_rows_of<float, true>(a, s);
  else launch_rows_of<float, false>(a, s);
}
void launch_grad_f32(const GradArgs& a, cudaStream_t s) { launch_grad_of<float>(a, s); }

}  // namespace dp
