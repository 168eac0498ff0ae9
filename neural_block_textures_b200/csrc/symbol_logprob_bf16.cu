// The symbol log-probability kernels for bf16 logits.
#include "symbol_logprob.cuh"

namespace ntcb {
cudaError_t symbol_rows_bf16(const RowArgs& a, cudaStream_t s, int sms) { return launch_rows<__nv_bfloat16>(a, s, sms); }
cudaError_t symbol_grad_bf16(const GradArgs& a, cudaStream_t s, int sms) { return launch_grad<__nv_bfloat16>(a, s, sms); }
}  // namespace ntcb
