// ntcb_symbol_logprobs / ntcb_symbol_logprobs_grad: the checks and the calls (the kernels: symbol_logprob.cuh).
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/ntc_b200.h"
#include "device_scope.h"
#include "symbol_logprob.h"

namespace ntcb {
namespace {

const char* check_desc(const ntcb_symbol_desc* d) {
    if (!d) return "null description";
    if (d->dtype < NTCB_F32 || d->dtype > NTCB_BF16) return "unknown type of the logits";
    if (d->symbol_type < NTCB_SYM_U8 || d->symbol_type > NTCB_SYM_I64) return "unknown type of the symbols";
    if (d->rows < 0) return "negative row count";
    if (d->vocab < 1 || d->vocab > (1ll << 28)) return "vocab outside 1 .. 2^28";
    if (d->row_stride < 0 || (d->row_stride > 0 && d->row_stride < d->vocab)) return "row_stride between 0 and vocab: rows overlap";
    if (d->symbol_stride < 0) return "negative symbol_stride";
    // the largest grids: one CTA per row, and one per 4096 logits of a row (gradient, 32 bits), below 2^31 CTAs in all
    if (d->rows > 0x7fffffffll / 8 || d->rows * ((d->vocab + 2047) / 2048 + 1) > 0x7fffffffll) return "more than 2^31 blocks of 2048 logits";
    return nullptr;
}
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
size_t dtype_size(int t) { return t == NTCB_F32 ? 4 : 2; }
// Whether rows of V elements written at `out` (stride os) may share memory with the rows read at `in` (stride is): the same
// rows, rows that lie between one another, or no common range at all.
bool may_write(const void* in, long long is, const void* out, long long os, long long rows, long long V, size_t size) {
    const long long a = (long long)(reinterpret_cast<uintptr_t>(in) / size), b = (long long)(reinterpret_cast<uintptr_t>(out) / size);
    if (a + (rows - 1) * is + V <= b || b + (rows - 1) * os + V <= a) return true;
    if (rows == 1) return a == b;
    if (is != os) return false;
    const long long off = ((b - a) % is + is) % is;
    return a == b || (off >= V && off <= is - V);
}
size_t symbol_size(int t) { return t == NTCB_SYM_U8 ? 1 : t == NTCB_SYM_I16 ? 2 : t == NTCB_SYM_I32 ? 4 : 8; }

}  // namespace
}  // namespace ntcb

extern "C" int ntcb_symbol_logprobs(const ntcb_symbol_desc* d, const void* logits, const void* symbols, int topk, float* logp,
                                    float* entropy, float* lse, int* top_ids, float* top_logp, void* stream, char* why, size_t why_cap) {
    using namespace ntcb;
    const auto refuse = [&](const char* m) { set_why(why, why_cap, m); return 0; };
    if (const char* m = check_desc(d)) return refuse(m);
    if (topk < 0 || topk > NTCB_MAX_TOPK) return refuse("topk outside 0 .. 32");
    if (topk > d->vocab) return refuse("topk above vocab");
    if (d->rows == 0) return 1;
    if (!logits || !symbols || !logp || !entropy || !lse || (topk && (!top_ids || !top_logp))) return refuse("null buffer");
    if (!aligned(logits, dtype_size(d->dtype)) || !aligned(symbols, symbol_size(d->symbol_type)) || !aligned(logp, 4) || !aligned(entropy, 4) ||
        !aligned(lse, 4) || (topk && (!aligned(top_ids, 4) || !aligned(top_logp, 4))))
        return refuse("a buffer is not aligned to its type");
    DeviceScope scope(d->device, why, why_cap);
    if (!scope.ok) return 0;
    const RowArgs a{logits, symbols, d->rows, d->row_stride, d->symbol_stride, (int)d->vocab, topk, d->symbol_type,
                    logp, entropy, lse, top_logp, top_ids};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = d->dtype == NTCB_F32 ? symbol_rows_f32(a, s, scope.sms)
                          : d->dtype == NTCB_F16 ? symbol_rows_f16(a, s, scope.sms)
                                                 : symbol_rows_bf16(a, s, scope.sms);
    return scope.launched(e, why, why_cap);
}

extern "C" int ntcb_symbol_logprobs_grad(const ntcb_symbol_desc* d, const void* logits, const void* symbols, const float* lse,
                                         const float* entropy, const float* dlogp, long long dlogp_stride, const float* dentropy,
                                         long long dentropy_stride, void* dlogits, long long dlogits_stride, void* stream, char* why,
                                         size_t why_cap) {
    using namespace ntcb;
    const auto refuse = [&](const char* m) { set_why(why, why_cap, m); return 0; };
    if (const char* m = check_desc(d)) return refuse(m);
    if (dlogp_stride < 0 || dentropy_stride < 0) return refuse("negative stride of an incoming gradient");
    if (dlogits_stride < d->vocab) return refuse("dlogits_stride below vocab: rows overlap");
    if (d->rows == 0) return 1;
    if (!logits || !symbols || !lse || !dlogp || !dlogits || (dentropy && !entropy)) return refuse("null buffer");
    const size_t sz = dtype_size(d->dtype);
    if (!aligned(logits, sz) || !aligned(dlogits, sz) || !aligned(symbols, symbol_size(d->symbol_type)) || !aligned(lse, 4) || !aligned(dlogp, 4) ||
        (dentropy && (!aligned(dentropy, 4) || !aligned(entropy, 4))))
        return refuse("a buffer is not aligned to its type");
    if (!may_write(logits, d->row_stride, dlogits, dlogits_stride, d->rows, d->vocab, sz)) return refuse("dlogits overlaps the logits without being them");
    DeviceScope scope(d->device, why, why_cap);
    if (!scope.ok) return 0;
    const GradArgs a{logits, symbols, lse, entropy, dlogp, dentropy, dlogits, d->rows, d->row_stride, d->symbol_stride, dlogits_stride,
                     dlogp_stride, dentropy_stride, (int)d->vocab, d->symbol_type, 1, 1};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = d->dtype == NTCB_F32 ? symbol_grad_f32(a, s, scope.sms)
                          : d->dtype == NTCB_F16 ? symbol_grad_f16(a, s, scope.sms)
                                                 : symbol_grad_bf16(a, s, scope.sms);
    return scope.launched(e, why, why_cap);
}
