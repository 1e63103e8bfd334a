// Row losses over bf16 margins.
#include "loss_rows.cuh"

namespace dp {

void launch_rows_bf16(const RowArgs& a, bool policy, cudaStream_t s) {
  if (policy) launch_rows_of<__nv_bfloat16, true>(a, s);
  else launch_rows_of<__nv_bfloat16, false>(a, s);
}
void launch_grad_bf16(const GradArgs& a, cudaStream_t s) { launch_grad_of<__nv_bfloat16>(a, s); }

}  // namespace dp
