// The arguments of the symbol log-probability kernels and their launchers, one per type of the logits (each in a source of
// its own, because the sorted variants take long to compile).
#pragma once
#include <cuda_runtime.h>

namespace ntcb {

struct RowArgs {
    const void* x;
    const void* sym;
    long long rows, stride, sym_stride;
    int V, topk, sym_type;
    float *logp, *entropy, *lse, *top_logp;
    int* top_ids;
};

struct GradArgs {
    const void* x;
    const void* sym;
    const float *lse, *entropy, *dlogp, *dentropy;
    void* dx;
    long long rows, stride, sym_stride, dx_stride, dlogp_stride, dentropy_stride;
    int V, sym_type, chunks, far_parts;
};

cudaError_t symbol_rows_f32(const RowArgs& a, cudaStream_t s, int sms);
cudaError_t symbol_rows_f16(const RowArgs& a, cudaStream_t s, int sms);
cudaError_t symbol_rows_bf16(const RowArgs& a, cudaStream_t s, int sms);
cudaError_t symbol_grad_f32(const GradArgs& a, cudaStream_t s, int sms);
cudaError_t symbol_grad_f16(const GradArgs& a, cudaStream_t s, int sms);
cudaError_t symbol_grad_bf16(const GradArgs& a, cudaStream_t s, int sms);

}  // namespace ntcb
