// Row losses over fp16 margins.
#include "loss_rows.cuh"

namespace dp {

void launch_rows_f16(const RowArgs& a, bool policy, cudaStream_t s) {
  if (policy) launch_rows_of<__half, true>(a, s);
  else launch_rows_of<__half, false>(a, s);
}
void launch_grad_f16(const GradArgs& a, cudaStream_t s) { launch_grad_of<__half>(a, s); }

}  // namespace dp
