"""Rating symbols under a predictor (ntcb_symbol_logprobs, ntcb_symbol_logprobs_grad): the log probability of each given
symbol (palette index, grid index, DCT token) under a row of logits, the row's entropy and its likeliest symbols, and
the gradient of a rate loss for the logits. Where print_stats rates a level by its counts, this rates it by a model.

    r = symbol_logprobs(logits, symbols, topk=4)          # logits [n, V] on the GPU, symbols [n]
    bits = -r.logp / math.log(2)
    dlogits = symbol_logprobs_grad(logits, symbols, r.lse, r.entropy, dlogp=-1.0 / n)   # of the mean code length

Calls run on torch's current stream of the logits' device, without synchronising; nothing is recorded by autograd.
"""
from __future__ import annotations

import ctypes as C
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


def _desc(logits: torch.Tensor, symbols: torch.Tensor, name: str) -> abi.SymbolDesc:
    if not isinstance(logits, torch.Tensor) or not isinstance(symbols, torch.Tensor):
        raise TypeError(f"{name}: logits and symbols must be torch tensors")
    if logits.dtype not in DTYPES:
        raise TypeError(f"{name}: logits must be float32, float16 or bfloat16, not {logits.dtype}")
    if symbols.dtype not in SYMBOL_TYPES:
        raise TypeError(f"{name}: symbols must be uint8, int16, int32 or int64, not {symbols.dtype}")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"{name}: logits must be [rows, vocab] with vocab >= 1, not {tuple(logits.shape)}")
    n, v = logits.shape
    if symbols.shape != (n,):
        raise ValueError(f"{name}: symbols must be [{n}], not {tuple(symbols.shape)}")
    if not logits.is_cuda or symbols.device != logits.device:
        raise ValueError(f"{name}: logits and symbols must be on one CUDA device")
    row_stride = logits.stride(0) if n > 1 else v
    if v > 1 and logits.stride(1) != 1:
        raise ValueError(f"{name}: a row's logits must be contiguous")
    return abi.SymbolDesc(logits.device.index, DTYPES[logits.dtype], SYMBOL_TYPES[symbols.dtype], 0, n, v, row_stride,
                          symbols.stride(0))


def _call(fn, name: str, *args) -> None:
    why = C.create_string_buffer(256)
    if not fn(*args, why, 256):
        raise RuntimeError(f"{name}: {why.value.decode()}")


def _per_row(x: torch.Tensor, n: int, device: torch.device, name: str) -> torch.Tensor:
    if x.dtype != torch.float32 or x.shape != (n,) or x.device != device:
        raise ValueError(f"symbol_logprobs_grad: {name} must be a float32 tensor of [{n}] on {device}")
    return x


def symbol_logprobs(logits: torch.Tensor, symbols: torch.Tensor, topk: int = 0) -> SymbolLogprobs:
    """Log probabilities of `symbols` [n] under `logits` [n, V] with the rows' entropy, log-sum-exp and `topk` (0 .. 32,
    at most V) likeliest symbols, in one pass over the logits. Rows may be strided; a row's logits are contiguous."""
    d = _desc(logits, symbols, "symbol_logprobs")
    n, v = d.rows, d.vocab
    if not 0 <= topk <= min(abi.MAX_TOPK, v):
        raise ValueError(f"symbol_logprobs: topk must be 0 .. {min(abi.MAX_TOPK, v)} here, not {topk}")
    dev = logits.device
    out = torch.empty(3, n, dtype=torch.float32, device=dev)
    ids = torch.empty(n, topk, dtype=torch.int32, device=dev)
    top = torch.empty(n, topk, dtype=torch.float32, device=dev)
    p = out.data_ptr()
    _call(abi.load_library().ntcb_symbol_logprobs, "symbol_logprobs", C.byref(d), logits.data_ptr(), symbols.data_ptr(), topk,
          p, p + 4 * n, p + 8 * n, ids.data_ptr(), top.data_ptr(), torch.cuda.current_stream(dev).cuda_stream)
    return SymbolLogprobs(out[0], out[1], out[2], ids, top)


def symbol_logprobs_grad(logits: torch.Tensor, symbols: torch.Tensor, lse: torch.Tensor, entropy: torch.Tensor | None,
                         dlogp: torch.Tensor | float, dentropy: torch.Tensor | float | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of sum(dlogp * logp + dentropy * entropy) for the logits, in their type, from the forward pass's lse
    and entropy. dlogp / dentropy: [n] float32 (any stride, so an expanded scalar too) or a number for every row.
    out: where to write it, of the logits' shape and type; the logits themselves are allowed."""
    d = _desc(logits, symbols, "symbol_logprobs_grad")
    n, v = d.rows, d.vocab
    dev = logits.device
    if not isinstance(dlogp, torch.Tensor):
        dlogp = torch.full((1,), float(dlogp), device=dev).expand(n)
    if dentropy is not None and not isinstance(dentropy, torch.Tensor):
        dentropy = torch.full((1,), float(dentropy), device=dev).expand(n)
    _per_row(lse, n, dev, "lse")
    _per_row(dlogp, n, dev, "dlogp")
    if dentropy is not None:
        if entropy is None:
            raise ValueError("symbol_logprobs_grad: dentropy needs the forward pass's entropy")
        _per_row(entropy, n, dev, "entropy")
        _per_row(dentropy, n, dev, "dentropy")
        entropy = entropy.contiguous()
    if out is None:
        out = torch.empty(n, v, dtype=logits.dtype, device=dev)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
        raise ValueError("symbol_logprobs_grad: out must have the logits' shape, type and device")
    elif (v > 1 and out.stride(1) != 1) or (n > 1 and out.stride(0) < v):
        raise ValueError("symbol_logprobs_grad: out's rows must be contiguous and apart from one another")
    elif out.data_ptr() == logits.data_ptr() and n > 1 and out.stride(0) != logits.stride(0):
        raise ValueError("symbol_logprobs_grad: out over the logits needs their row stride")
    lse = lse.contiguous()
    _call(abi.load_library().ntcb_symbol_logprobs_grad, "symbol_logprobs_grad", C.byref(d), logits.data_ptr(), symbols.data_ptr(),
          lse.data_ptr(), entropy.data_ptr() if dentropy is not None else None, dlogp.data_ptr(), dlogp.stride(0),
          dentropy.data_ptr() if dentropy is not None else None, dentropy.stride(0) if dentropy is not None else 0, out.data_ptr(),
          out.stride(0) if n > 1 else v, torch.cuda.current_stream(dev).cuda_stream)
    return out
