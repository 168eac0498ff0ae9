// The symbol log-probability kernels for f32 logits.
#include "symbol_logprob.cuh"

namespace ntcb {
cudaError_t symbol_rows_f32(const RowArgs& a, cudaStream_t s, int sms) { return launch_rows<float>(a, s, sms); }
cudaError_t symbol_grad_f32(const GradArgs& a, cudaStream_t s, int sms) { return launch_grad<float>(a, s, sms); }
}  // namespace ntcb
