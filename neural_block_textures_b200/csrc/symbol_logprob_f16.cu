// The symbol log-probability kernels for f16 logits.
#include "symbol_logprob.cuh"

namespace ntcb {
cudaError_t symbol_rows_f16(const RowArgs& a, cudaStream_t s, int sms) { return launch_rows<__half>(a, s, sms); }
cudaError_t symbol_grad_f16(const GradArgs& a, cudaStream_t s, int sms) { return launch_grad<__half>(a, s, sms); }
}  // namespace ntcb
