"""AdamW over many tensors in one launch (ntcb_adamw_*), with the moments in 32 bits or in 8: the optimiser for tensors
that a host holds and differentiates itself (many texture models' levels and layers, a symbol model's tables), beside
the Adam that runs inside the trainer's own steps. With weight_decay 0 it is that Adam.

    opt = AdamW(params, state_bits=8, weight_decay=0.01)
    for it in range(1, iters + 1):
        ...                                   # gradients, in p.grad or in a list
        opt.step(it, lr)

A step runs on torch's current stream of the parameters' device, without synchronising, and writes the parameters in
place; autograd does not record that, but a backward pass over values saved before the step fails, as after torch's own
in-place operations (a graph's replays are not seen). In a captured CUDA graph the step number comes from the device: pass `it` as an
int64 tensor and advance it there. The graph has the addresses of the parameters, the gradients and the state: keep those
tensors as long as it is replayed (the state stays by itself until close()).
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import abi
from .symbols import DTYPES, _call, _host, _raw_stream

_T = torch.Tensor
_outlived = []   # (plan, state) of collected optimisers that a graph may still step
_pack_args = struct.Struct("6dqQ3Q").pack   # ntcb_adamw_args


class AdamW:
    """params: contiguous float32, float16 or bfloat16 CUDA tensors on one device; kept, and written by step().
    grad_dtype: the gradients' type where it is not the parameter's. The state (`state`, one uint8 tensor) starts at
    zero, set on the stream that is current here, which another stream's first step waits for as for any tensor's
    contents; it can be saved and restored with state_dict() / load_state_dict()."""

    def __init__(self, params, state_bits: int = 32, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, seed: int = 0, grad_dtype: torch.dtype | None = None) -> None:
        self.h = None
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW: no parameters")
        if state_bits not in (8, 32):
            raise ValueError("AdamW: state_bits must be 8 or 32")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("AdamW: betas must be in [0, 1)")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("AdamW: eps and weight_decay must not be negative")
        if 0.0 < eps < torch.finfo(torch.float32).tiny:
            raise ValueError("AdamW: eps must be 0 or at least 1.18e-38 (a normal 32-bit number)")
        if grad_dtype is not None and grad_dtype not in DTYPES:
            raise TypeError(f"AdamW: gradients must be float32, float16 or bfloat16, not {grad_dtype}")
        for p in self.params:
            if not isinstance(p, torch.Tensor) or p.dtype not in DTYPES:
                raise TypeError("AdamW: parameters must be float32, float16 or bfloat16 tensors")
            if not p.is_cuda or p.device != self.params[0].device:
                raise ValueError("AdamW: parameters must be on one CUDA device")
            if not p.is_contiguous() or p.is_neg():
                raise ValueError("AdamW: parameters must be contiguous, and no negated views")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self.params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("AdamW: two parameters share memory")
        self.device = self.params[0].device
        self.state_bits, self.betas, self.eps, self.weight_decay, self.seed = state_bits, tuple(betas), eps, weight_decay, seed
        n = len(self.params)
        self._index = self.device.index
        self._sizes = [p.numel() for p in self.params]
        self._grad_dtypes = [grad_dtype or p.dtype for p in self.params]
        self.lib = abi.load_library()
        why = C.create_string_buffer(256)
        self._keep = ((C.c_longlong * n)(*self._sizes), (C.c_int * n)(*[DTYPES[p.dtype] for p in self.params]),
                      (C.c_int * n)(*[DTYPES[t] for t in self._grad_dtypes]))
        self._plan = tuple(C.addressof(a) for a in self._keep)
        self.h = self.lib.ntcb_adamw_create(self._index, n, *self._keep, state_bits, why, 256)
        if not self.h:
            raise RuntimeError("AdamW: " + why.value.decode())
        self.offsets = [int(self.lib.ntcb_adamw_offset(self.h, i)) for i in range(n + 1)]   # elements; the last is the total
        self.state = torch.zeros(self.lib.ntcb_adamw_state_bytes(self.h), dtype=torch.uint8, device=self.device)
        if state_bits == 32:
            self._mv = self.state.view(torch.float32).split(self.offsets[-1]) if self.offsets[-1] else (self.state.view(torch.float32),) * 2

    def close(self) -> None:
        """Frees the plan. No graph that captured a call may be replayed after this; an optimiser that is merely collected
        leaves the plan and the state of captured calls in place."""
        if getattr(self, "h", None):
            self.lib.ntcb_adamw_destroy(self.h)
            self.h = None

    def __del__(self) -> None:
        try:
            if getattr(self, "h", None) and self.lib.ntcb_adamw_captured(self.h):
                _outlived.append((self.h, self.state))
                self.h = None
            self.close()
        except Exception:
            pass

    def __reduce_ex__(self, protocol):
        raise TypeError("AdamW: a plan cannot be copied or pickled; use state_dict() and load_state_dict()")

    def _open(self) -> None:
        if not self.h:
            raise RuntimeError("AdamW: closed")

    def _scalar(self, x: torch.Tensor, dtype: torch.dtype, name: str) -> tuple[int, int]:
        """(the host value's place holder, the device address) of a one-element device tensor."""
        if x.dtype != dtype or x.numel() != 1 or x.device != self.device or x.is_neg():
            raise ValueError(f"AdamW.step: {name} as a tensor must be one {dtype} on {self.device}")
        return 1, x.data_ptr()

    def step(self, it, lr, grads=None, grad_scale=1.0) -> None:
        """Step number `it` (from 1) at learning rate `lr` with the gradients `grads` (default: each p.grad) times
        grad_scale; a None gradient leaves its tensor and moments alone. it, lr and grad_scale may be device tensors
        (int64, float32, float32)."""
        self._open()
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        n = len(self.params)
        it, it_dev = self._scalar(it, torch.int64, "it") if isinstance(it, _T) else (it, 0)
        lr, lr_dev = self._scalar(lr, torch.float32, "lr") if isinstance(lr, _T) else (lr, 0)
        grad_scale, scale_dev = self._scalar(grad_scale, torch.float32, "grad_scale") if isinstance(grad_scale, _T) else (grad_scale, 0)
        args = _pack_args(lr, *self.betas, self.eps, self.weight_decay, grad_scale, it, self.seed & 0xFFFFFFFFFFFFFFFF, it_dev, lr_dev, scale_dev)
        why = C.create_string_buffer(256)
        bad = _host.ntcb_host_adamw_step(self.h, self.params, grads, n, *self._plan, self._index, self.state.data_ptr(), args, why, 256)
        if bad == -2:
            raise ValueError(f"AdamW.step: {n} gradients are needed, not {len(grads)}")
        if bad == -3:
            raise RuntimeError("AdamW.step: " + why.value.decode())
        if bad >= 0:
            raise ValueError(f"AdamW.step: gradient {bad} must be a contiguous {self._grad_dtypes[bad]} tensor of {self._sizes[bad]} elements on "
                             f"{self.device}, and its parameter as it was when the plan was made")

    def moments_flat(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(m, v) as flat float32 tensors, tensor i at offsets[i]: the state itself with 32 bits, the values that the
        codes stand for with 8."""
        self._open()
        if self.state_bits == 32:
            return self._mv
        total = self.offsets[-1]
        m = torch.empty(total, dtype=torch.float32, device=self.device)
        v = torch.empty_like(m)
        _call(self.lib.ntcb_adamw_get_moments, "AdamW.moments", self.h, self.state.data_ptr(), m.data_ptr(), v.data_ptr(),
              _raw_stream(self._index))
        return m, v

    def moments(self) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
        """(m, v), each a list of float32 tensors shaped as the parameters."""
        return tuple([flat[o:o + p.numel()].view(p.shape) for o, p in zip(self.offsets, self.params)] for flat in self.moments_flat())

    def set_moments(self, m, v) -> None:
        """Sets the moments from lists of tensors (rounded to nearest with 8-bit states)."""
        self._open()
        flat = []
        for name, xs in (("m", list(m)), ("v", list(v))):
            if len(xs) != len(self.params) or any(x.numel() != n for x, n in zip(xs, self._sizes)):
                raise ValueError(f"AdamW.set_moments: {name} must have one tensor of each parameter's size")
            f = torch.zeros(self.offsets[-1], dtype=torch.float32, device=self.device)
            for o, x in zip(self.offsets, xs):
                f[o:o + x.numel()].copy_(x.reshape(-1))
            flat.append(f)
        _call(self.lib.ntcb_adamw_set_moments, "AdamW.set_moments", self.h, flat[0].data_ptr(), flat[1].data_ptr(),
              self.state.data_ptr(), _raw_stream(self._index))

    def state_dict(self) -> dict:
        """The state (a copy) with what it was laid out for, and the seed of its rounding."""
        return {"state_bits": self.state_bits, "sizes": list(self._sizes), "seed": self.seed, "state": self.state.clone()}

    def load_state_dict(self, d: dict) -> None:
        if d["state_bits"] != self.state_bits or list(d["sizes"]) != self._sizes:
            raise ValueError("AdamW.load_state_dict: the state is of another layout")
        if d["state"].dtype != torch.uint8 or d["state"].numel() != self.state.numel():
            raise ValueError("AdamW.load_state_dict: the state has another size")
        self.state.copy_(d["state"])
        self.seed = d["seed"]
