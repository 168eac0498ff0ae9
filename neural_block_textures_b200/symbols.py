"""Rating symbols under a predictor (ntcb_symbol_logprobs, ntcb_symbol_logprobs_grad): the log probability of each given
symbol (palette index, grid index, DCT token) under a row of logits, the row's entropy and its likeliest symbols, and
the gradient of a rate loss for the logits. Where print_stats rates a level by its counts, this rates it by a model.

    r = symbol_logprobs(logits.detach(), symbols, topk=4)   # logits [n, V] on the GPU, symbols [n]
    bits = -r.logp / math.log(2)
    dlogits = symbol_logprobs_grad(logits, symbols, r.lse, r.entropy, dlogp=-1.0 / n)   # of the mean code length

Calls run on torch's current stream of the logits' device, without synchronising. Nothing is recorded by autograd: logits
that require a gradient are rated with a warning (pass logits.detach()), and symbol_logprobs_grad gives what to hand to
their backward pass.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from . import abi

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}                      # NTCB_F32 ...
SYMBOL_TYPES = {torch.uint8: 0, torch.int16: 1, torch.int32: 2, torch.int64: 3}       # NTCB_SYM_U8 ...


class SymbolLogprobs(NamedTuple):
    logp: torch.Tensor       # [n] float32: log p(symbol), nats; 0 for a negative symbol
    entropy: torch.Tensor    # [n] float32
    lse: torch.Tensor        # [n] float32: log of the sum of exponentials
    top_ids: torch.Tensor    # [n, topk] int32, likeliest first, the lower index first among equals; -1 where none is left
    top_logp: torch.Tensor   # [n, topk] float32; -inf there


_pack_desc = struct.Struct("4i4q").pack   # ntcb_symbol_desc
# torch's current stream of a device as an address; the public call makes an object for it (2 us of a 12 us call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _desc(logits: torch.Tensor, symbols: torch.Tensor, name: str) -> tuple[bytes, int, int, int]:
    """(ntcb_symbol_desc, rows, vocab, device index) of checked arguments."""
    if not isinstance(logits, torch.Tensor) or not isinstance(symbols, torch.Tensor):
        raise TypeError(f"{name}: logits and symbols must be torch tensors")
    if any(x.layout is not torch.strided or x.is_nested for x in (logits, symbols)):
        raise ValueError(f"{name}: logits and symbols must be strided tensors, not sparse or nested ones")
    dtype, symbol_type = DTYPES.get(logits.dtype), SYMBOL_TYPES.get(symbols.dtype)
    if dtype is None:
        raise TypeError(f"{name}: logits must be float32, float16 or bfloat16, not {logits.dtype}")
    if symbol_type is None:
        raise TypeError(f"{name}: symbols must be uint8, int16, int32 or int64, not {symbols.dtype}")
    shape = logits.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{name}: logits must be [rows, vocab] with vocab >= 1, not {tuple(shape)}")
    n, v = shape
    if symbols.shape != (n,):
        raise ValueError(f"{name}: symbols must be [{n}], not {tuple(symbols.shape)}")
    device = logits.get_device()
    if device < 0 or symbols.get_device() != device:
        raise ValueError(f"{name}: logits and symbols must be on one CUDA device")
    row_stride, stride = logits.stride()
    if v > 1 and stride != 1:
        raise ValueError(f"{name}: a row's logits must be contiguous")
    return _pack_desc(device, dtype, symbol_type, 0, n, v, row_stride if n > 1 else v, symbols.stride(0)), n, v, device


def _call(fn, name: str, *args) -> None:
    why = C.create_string_buffer(256)
    if not fn(*args, why, 256):
        raise RuntimeError(f"{name}: {why.value.decode()}")


def _load_host() -> C.PyDLL:
    """The compiled host side (csrc/torch_host.cpp)."""
    abi.load_library()
    path = abi.LIB_PATH.with_name("libntc_b200_torch.so")
    if not path.exists():
        raise RuntimeError(f"{path.name} not found at {path}: build it with `python -m neural_block_textures_b200.build`")
    lib = C.PyDLL(str(path))
    o = C.py_object
    lib.ntcb_host_logprobs.restype, lib.ntcb_host_logprobs.argtypes = o, [o, o, C.c_int]
    lib.ntcb_host_logprobs_grad.restype, lib.ntcb_host_logprobs_grad.argtypes = o, [o] * 6
    p, i = C.c_void_p, C.c_int
    lib.ntcb_host_adamw_step.restype, lib.ntcb_host_adamw_step.argtypes = i, [p, o, o, i, p, p, p, i, p, p, C.c_char_p, C.c_size_t]
    lib.ntcb_host_written.restype, lib.ntcb_host_written.argtypes = o, [o]
    return lib


_host = _load_host()


def _per_row(x: torch.Tensor, n: int, device: int, name: str) -> torch.Tensor:
    if x.dtype is not torch.float32 or x.shape != (n,) or x.get_device() != device:
        raise ValueError(f"symbol_logprobs_grad: {name} must be a float32 tensor of [{n}] on the logits' device")
    return x


def symbol_logprobs(logits: torch.Tensor, symbols: torch.Tensor, topk: int = 0) -> SymbolLogprobs:
    """Log probabilities of `symbols` [n] under `logits` [n, V] with the rows' entropy, log-sum-exp and `topk` (0 .. 32,
    at most V) likeliest symbols, in one pass over the logits. Rows may be strided; a row's logits are contiguous."""
    if 0 <= topk <= abi.MAX_TOPK:
        r = _host.ntcb_host_logprobs(logits, symbols, topk)
        if r is not None:
            return tuple.__new__(SymbolLogprobs, r)   # the class's own __new__ takes its fields one by one: 0.3 us more
    _, n, v, _ = _desc(logits, symbols, "symbol_logprobs")   # says what is wrong
    if logits.is_neg():
        return symbol_logprobs(logits.resolve_neg(), symbols, topk)
    if not 0 <= topk <= min(abi.MAX_TOPK, v):
        raise ValueError(f"symbol_logprobs: topk must be 0 .. {min(abi.MAX_TOPK, v)} here, not {topk}")
    raise ValueError("symbol_logprobs: these tensors cannot be rated")


def symbol_logprobs_grad(logits: torch.Tensor, symbols: torch.Tensor, lse: torch.Tensor, entropy: torch.Tensor | None,
                         dlogp: torch.Tensor | float, dentropy: torch.Tensor | float | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of sum(dlogp * logp + dentropy * entropy) for the logits, in their type, from the forward pass's lse
    and entropy. dlogp / dentropy: [n] float32 (any stride, so an expanded scalar too) or a number for every row.
    out: where to write it, of the logits' shape and type; the logits themselves are allowed, memory
    that overlaps them otherwise is refused, and it must not overlap the other tensors."""
    if out is None and isinstance(dlogp, torch.Tensor) and (dentropy is None or isinstance(dentropy, torch.Tensor)):
        r = _host.ntcb_host_logprobs_grad(logits, symbols, lse, entropy, dlogp, dentropy)
        if r is not None:
            return r
    d, n, v, device = _desc(logits, symbols, "symbol_logprobs_grad")
    dev = logits.device
    if out is not None and out.is_neg():
        raise ValueError("symbol_logprobs_grad: out must not be a negated view")
    # the memory of a negated view holds the values' negatives
    if logits.is_neg():
        return symbol_logprobs_grad(logits.resolve_neg(), symbols, lse, entropy, dlogp, dentropy, out)
    lse, entropy, dlogp, dentropy = (x.resolve_neg() if isinstance(x, torch.Tensor) else x for x in (lse, entropy, dlogp, dentropy))
    if not isinstance(dlogp, torch.Tensor):
        dlogp = torch.full((1,), float(dlogp), device=dev).expand(n)
    if dentropy is not None and not isinstance(dentropy, torch.Tensor):
        dentropy = torch.full((1,), float(dentropy), device=dev).expand(n)
    _per_row(lse, n, device, "lse")
    _per_row(dlogp, n, device, "dlogp")
    if dentropy is not None:
        if entropy is None:
            raise ValueError("symbol_logprobs_grad: dentropy needs the forward pass's entropy")
        _per_row(entropy, n, device, "entropy")
        _per_row(dentropy, n, device, "dentropy")
        entropy = entropy.contiguous()
    if out is None:
        out = logits.new_empty((n, v))
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
        raise ValueError("symbol_logprobs_grad: out must have the logits' shape, type and device")
    elif (v > 1 and out.stride(1) != 1) or (n > 1 and out.stride(0) < v):
        raise ValueError("symbol_logprobs_grad: out's rows must be contiguous and apart from one another")
    lse = lse.contiguous()
    _call(abi.load_library().ntcb_symbol_logprobs_grad, "symbol_logprobs_grad", d, logits.data_ptr(), symbols.data_ptr(),
          lse.data_ptr(), entropy.data_ptr() if dentropy is not None else None, dlogp.data_ptr(), dlogp.stride(0),
          dentropy.data_ptr() if dentropy is not None else None, dentropy.stride(0) if dentropy is not None else 0, out.data_ptr(),
          out.stride(0) if n > 1 else v, _raw_stream(device))
    _host.ntcb_host_written(out)
    return out
