// The host side of the operators on torch tensors (symbols.py, optim.py) for calls that are all host work: a Python call per
// tensor or argument costs 40 ns to 2 us, which is 15 us for one small rating and 130 us for an AdamW step over 300
// tensors. These functions look at the same things and make the same calls of the C ABI (include/ntc_b200.h). Anything
// but the plain case is left to the Python code, which names what is wrong: they return None (or an index) then.
// Called through ctypes.PyDLL, so with the interpreter's lock held (and let go while they allocate and launch); a Python exception that is set is raised there. A C++
// exception must not leave an entry (it would end the process): torch throws them from as little as a size() of a tensor
// subclass or a nested tensor, so everything is done inside torch's own translation to Python's exceptions.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <vector>

#include "../../include/ntc_b200.h"

namespace {

int dtype_code(at::ScalarType t) {
    return t == at::kFloat ? NTCB_F32 : t == at::kHalf ? NTCB_F16 : t == at::kBFloat16 ? NTCB_BF16 : -1;
}
int symbol_code(at::ScalarType t) {
    return t == at::kByte ? NTCB_SYM_U8 : t == at::kShort ? NTCB_SYM_I16 : t == at::kInt ? NTCB_SYM_I32 : t == at::kLong ? NTCB_SYM_I64 : -1;
}
// A tensor whose memory holds its values as they are: a negated view (the imaginary part of a conjugate) holds their negatives.
bool plain(PyObject* o) {
    if (!THPVariable_Check(o)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.layout() == at::kStrided && !t.is_nested() && !t.is_neg();
}

// The description of plain logits [n, V] and symbols [n] on one CUDA device; false for anything else.
bool describe(PyObject* logits, PyObject* symbols, ntcb_symbol_desc& d) {
    if (!plain(logits) || !plain(symbols)) return false;
    const at::Tensor &x = THPVariable_Unpack(logits), &s = THPVariable_Unpack(symbols);
    if (!x.is_cuda() || x.dim() != 2 || s.dim() != 1 || s.device() != x.device() || s.size(0) != x.size(0)) return false;
    const int64_t n = x.size(0), v = x.size(1);
    d = ntcb_symbol_desc{x.get_device(), dtype_code(x.scalar_type()), symbol_code(s.scalar_type()), 0, n, v, n > 1 ? x.stride(0) : v, s.stride(0)};
    return d.dtype >= 0 && d.symbol_type >= 0 && v >= 1 && (v == 1 || x.stride(1) == 1);
}
// A float tensor [n] on the logits' device.
bool per_row(PyObject* o, const ntcb_symbol_desc& d) {
    if (!plain(o)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.get_device() == d.device && t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == d.rows;
}
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// The interpreter's lock let go: an allocation may wait for the device and a launch for a place in its queue, and what is
// queued there may be a host function that needs the lock.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

// Raises a tensor's version, as torch's own in-place operations do: a backward pass over values saved before then fails
// instead of using the new ones. Inference tensors have no version.
void written(const at::Tensor& t) { if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); }

PyObject* failed(const char* name, const char* why) {
    PyErr_Format(PyExc_RuntimeError, "%s: %s", name, why);
    return nullptr;
}

}  // namespace

extern "C" {

// (logp, entropy, lse, top_ids, top_logp), or None.
PyObject* ntcb_host_logprobs(PyObject* logits, PyObject* symbols, int topk) {
    HANDLE_TH_ERRORS
        ntcb_symbol_desc d;
        if (!describe(logits, symbols, d) || topk < 0 || topk > NTCB_MAX_TOPK || topk > d.vocab) Py_RETURN_NONE;
        const at::Tensor x = THPVariable_Unpack(logits), s = THPVariable_Unpack(symbols);
        if (((at::GradMode::is_enabled() && x.requires_grad()) || x._fw_grad(0).defined()) &&
            PyErr_WarnEx(PyExc_UserWarning, "symbol_logprobs: the logits require a gradient, but autograd records nothing of this call: "
                         "take it from symbol_logprobs_grad, and pass logits.detach() here", 2) < 0)   // 2: the caller's line
            return nullptr;
        at::Tensor out[5];
        char why[256];
        bool ok;
        {
            const Unlocked unlocked;
            const auto f = at::TensorOptions().dtype(at::kFloat).device(x.device());
            for (int i = 0; i < 3; i++) out[i] = at::empty({d.rows}, f);
            out[3] = at::empty({d.rows, topk}, f.dtype(at::kInt));
            out[4] = at::empty({d.rows, topk}, f);
            ok = ntcb_symbol_logprobs(&d, x.data_ptr(), s.data_ptr(), topk, out[0].data_ptr<float>(), out[1].data_ptr<float>(),
                                      out[2].data_ptr<float>(), out[3].data_ptr<int>(), out[4].data_ptr<float>(), stream_of(d.device), why, sizeof(why));
        }
        if (!ok) return failed("symbol_logprobs", why);
        PyObject* r = PyTuple_New(5);
        if (!r) return nullptr;
        for (int i = 0; i < 5; i++) {
            PyObject* t = THPVariable_Wrap(out[i]);
            if (!t) { Py_DECREF(r); return nullptr; }
            PyTuple_SET_ITEM(r, i, t);
        }
        return r;
    END_HANDLE_TH_ERRORS
}

// The gradient in a new tensor, or None. entropy and dentropy may be None.
PyObject* ntcb_host_logprobs_grad(PyObject* logits, PyObject* symbols, PyObject* lse, PyObject* entropy, PyObject* dlogp, PyObject* dentropy) {
    HANDLE_TH_ERRORS
        ntcb_symbol_desc d;
        if (!describe(logits, symbols, d) || !per_row(lse, d) || !per_row(dlogp, d)) Py_RETURN_NONE;
        const bool with = dentropy != Py_None;
        if (with && (!per_row(dentropy, d) || !per_row(entropy, d) || !THPVariable_Unpack(entropy).is_contiguous())) Py_RETURN_NONE;
        if (!THPVariable_Unpack(lse).is_contiguous()) Py_RETURN_NONE;
        const at::Tensor x = THPVariable_Unpack(logits), s = THPVariable_Unpack(symbols), sum = THPVariable_Unpack(lse), l = THPVariable_Unpack(dlogp);
        const at::Tensor h = with ? THPVariable_Unpack(entropy) : at::Tensor(), e = with ? THPVariable_Unpack(dentropy) : at::Tensor();
        at::Tensor out;
        char why[256];
        bool ok;
        {
            const Unlocked unlocked;
            out = at::empty({d.rows, d.vocab}, at::TensorOptions().dtype(x.scalar_type()).device(x.device()));
            ok = ntcb_symbol_logprobs_grad(&d, x.data_ptr(), s.data_ptr(), sum.data_ptr<float>(), with ? h.data_ptr<float>() : nullptr,
                                           l.data_ptr<float>(), l.stride(0), with ? e.data_ptr<float>() : nullptr, with ? e.stride(0) : 0,
                                           out.data_ptr(), d.vocab, stream_of(d.device), why, sizeof(why));
        }
        if (!ok) return failed("symbol_logprobs_grad", why);
        return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// A step of plan `a` over n parameters and gradients (lists; a gradient may be None) after checking sizes, types, layout and
// device. Returns -1, or the index of the first tensor that does not fit (with the Python exception that it raised, if it
// did), -2 when the lists do not, or -3 with a reason in why.
int ntcb_host_adamw_step(const ntcb_adamw* a, PyObject* params, PyObject* grads, int n, const long long* sizes, const int* param_types,
                         const int* grad_types, int device, void* state, const ntcb_adamw_args* args, char* why, size_t why_cap) {
    if (!PyList_Check(params) || !PyList_Check(grads) || PyList_GET_SIZE(params) != n || PyList_GET_SIZE(grads) != n) return -2;
    const auto fits = [&](PyObject* o, long long size, int type) {
        if (!plain(o)) return false;
        const at::Tensor& t = THPVariable_Unpack(o);
        return t.numel() == size && dtype_code(t.scalar_type()) == type && t.is_contiguous() && t.is_cuda() && t.get_device() == device;
    };
    int i = 0;
    try {
        std::vector<void*> at((size_t)n * 2, nullptr);
        for (; i < n; i++) {
            PyObject *p = PyList_GET_ITEM(params, i), *g = PyList_GET_ITEM(grads, i);
            if (g == Py_None) continue;
            if (!fits(p, sizes[i], param_types[i]) || !fits(g, sizes[i], grad_types[i])) return i;
            at[i] = THPVariable_Unpack(p).data_ptr();
            at[n + i] = THPVariable_Unpack(g).data_ptr();
        }
        void* stream = stream_of(device);
        bool ok;
        {
            const Unlocked unlocked;
            ok = ntcb_adamw_step(a, at.data(), at.data() + n, state, args, stream, why, why_cap);
        }
        if (!ok) return -3;
        for (int k = 0; k < n && k < PyList_GET_SIZE(params); k++)
            if (at[n + k] && THPVariable_Check(PyList_GET_ITEM(params, k))) written(THPVariable_Unpack(PyList_GET_ITEM(params, k)));
        return -1;
    } catch (python_error& e) {
        e.restore();
    } catch (...) {   // a tensor that does not say what it is, or has no memory
    }
    return i;
}

// Raises the version of a tensor that a call wrote.
PyObject* ntcb_host_written(PyObject* tensor) {
    HANDLE_TH_ERRORS
        if (THPVariable_Check(tensor)) written(THPVariable_Unpack(tensor));
        Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

}  // extern "C"
