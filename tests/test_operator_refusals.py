"""Refusals of the symbol log-probability and AdamW entries, without a GPU: every bad description comes back as 0 (or
NULL) with a reason before a device is touched, the Python layer names the argument, and the ctypes structures have the
C layout."""
import ctypes as C
import shutil
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from neural_block_textures_b200 import AdamW, abi, symbol_logprobs, symbol_logprobs_grad

ROOT = Path(__file__).resolve().parent.parent
BUF = 1 << 20   # an address that is never read


def desc(**kw):
    d = dict(device=-1, dtype=0, symbol_type=2, reserved=0, rows=4, vocab=8, row_stride=8, symbol_stride=1)
    d.update(kw)
    return abi.SymbolDesc(*[d[f] for f, _ in abi.SymbolDesc._fields_])


def forward(d, topk=0, logits=BUF, symbols=BUF, logp=BUF, top=BUF):
    why = C.create_string_buffer(256)
    ok = abi.load_library().ntcb_symbol_logprobs(C.byref(d) if d is not None else None, logits, symbols, topk, logp, BUF, BUF, top, top,
                                                 None, why, 256)
    return ok, why.value.decode()


def gradient(d, dlogp_stride=1, dx_stride=8, dentropy=None, entropy=None, dx=BUF):
    why = C.create_string_buffer(256)
    ok = abi.load_library().ntcb_symbol_logprobs_grad(C.byref(d), BUF, BUF, BUF, entropy, BUF, dlogp_stride, dentropy, 1, dx, dx_stride,
                                                      None, why, 256)
    return ok, why.value.decode()


@pytest.mark.parametrize("kw, word", [
    (dict(dtype=3), "logits"), (dict(dtype=-1), "logits"), (dict(symbol_type=4), "symbols"), (dict(rows=-1), "row count"),
    (dict(vocab=0), "vocab"), (dict(vocab=(1 << 28) + 1, row_stride=1 << 29), "vocab"), (dict(row_stride=7), "row_stride"),
    (dict(row_stride=-8), "row_stride"), (dict(symbol_stride=-1), "symbol_stride"), (dict(rows=1 << 40), "blocks"),
    (dict(rows=1 << 20, vocab=1 << 27, row_stride=1 << 27), "blocks"),
])
def test_bad_descriptions(kw, word):
    for ok, why in (forward(desc(**kw)), gradient(desc(**kw))):
        assert ok == 0 and word in why


def test_bad_arguments():
    assert forward(None) == (0, "null description")
    for topk in (-1, 33):
        assert "topk" in forward(desc(vocab=64, row_stride=64), topk)[1]
    assert "vocab" in forward(desc(), 9)[1]
    assert forward(desc(), logits=None) == (0, "null buffer")
    assert forward(desc(), logp=None) == (0, "null buffer")
    assert forward(desc(), 1, top=None) == (0, "null buffer")
    assert "aligned" in forward(desc(), logits=BUF + 2)[1]
    assert "aligned" in forward(desc(dtype=2), symbols=BUF + 2)[1]
    assert "dlogits_stride" in gradient(desc(), dx_stride=7)[1]
    assert "stride" in gradient(desc(), dlogp_stride=-1)[1]
    assert gradient(desc(), dentropy=BUF) == (0, "null buffer")
    assert "aligned" in gradient(desc(dtype=1), dx=BUF + 1)[1]
    # dlogits over the logits (BUF): shifted, of another stride, or over a broadcast row
    for kw in (dict(dx=BUF + 4), dict(dx=BUF + 4 * 8), dict(dx=BUF, dx_stride=9), dict(dx=BUF - 4)):
        assert "overlaps" in gradient(desc(), **kw)[1]
    assert "overlaps" in gradient(desc(row_stride=0), dx=BUF)[1]
    assert "overlaps" in gradient(desc(row_stride=20), dx=BUF + 4 * 13, dx_stride=20)[1]
    assert "overlaps" not in gradient(desc(rows=0))[1]
    # nothing to do is no refusal, and touches no device
    assert forward(desc(rows=0), logits=None)[0] == 1 and gradient(desc(rows=0))[0] == 1


def create(sizes, param=None, grad=None, bits=32):
    n = len(sizes)
    why = C.create_string_buffer(256)
    h = abi.load_library().ntcb_adamw_create(-1, n, (C.c_longlong * n)(*sizes), (C.c_int * n)(*(param or [0] * n)),
                                             (C.c_int * n)(*(grad or [0] * n)), bits, why, 256)
    return h, why.value.decode()


def test_adamw_plan_refusals():
    assert create([]) == (None, "no tensors")
    assert "state_bits" in create([4], bits=16)[1]
    for sizes in ([-1], [(1 << 36) + 1]):
        assert "size" in create(sizes)[1]
    assert "2^36" in create([1 << 36, 1])[1]
    assert "type" in create([4], param=[3])[1] and "type" in create([4], grad=[-1])[1]
    lib = abi.load_library()
    assert lib.ntcb_adamw_state_bytes(None) == 0 and lib.ntcb_adamw_offset(None, 0) == -1
    lib.ntcb_adamw_destroy(None)
    why = C.create_string_buffer(64)
    assert lib.ntcb_adamw_step(None, None, None, None, None, None, why, 64) == 0 and why.value
    assert lib.ntcb_adamw_get_moments(None, None, None, None, None, why, 64) == 0
    assert lib.ntcb_adamw_set_moments(None, None, None, None, None, why, 64) == 0


def test_without_a_gpu_a_reason():
    if torch.cuda.is_available():
        pytest.skip("this machine has a GPU")
    assert "CUDA" in forward(desc())[1] and "CUDA" in gradient(desc())[1]
    h, why = create([4, 0, 300])
    assert h is None and "CUDA" in why


def test_python_refusals_on_host_tensors():
    x, s = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        symbol_logprobs(x, s)
    with pytest.raises(TypeError, match="float64"):
        symbol_logprobs(x.double(), s)
    with pytest.raises(TypeError, match="int8"):
        symbol_logprobs(x, s.to(torch.int8))
    with pytest.raises(ValueError, match="rows, vocab"):
        symbol_logprobs(x[0], s)
    with pytest.raises(ValueError, match="rows, vocab"):
        symbol_logprobs(x[:, :0], s)
    with pytest.raises(ValueError, match="symbols must be"):
        symbol_logprobs(x, s[:3])
    with pytest.raises(TypeError):
        symbol_logprobs(x, [0, 1, 2, 3])
    with pytest.raises(ValueError, match="CUDA"):
        symbol_logprobs_grad(x, s, x[:, 0], None, -1.0)
    with pytest.raises(ValueError, match="CUDA"):
        AdamW([x])
    with pytest.raises(ValueError, match="no parameters"):
        AdamW([])
    with pytest.raises(TypeError):
        AdamW([x.double()])
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([x], state_bits=4)
    with pytest.raises(ValueError, match="betas"):
        AdamW([x], betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="negative"):
        AdamW([x], weight_decay=-0.1)
    with pytest.raises(TypeError, match="gradients"):
        AdamW([x], grad_dtype=torch.float64)


@pytest.mark.parametrize("cls, name", [(abi.SymbolDesc, "ntcb_symbol_desc"), (abi.AdamWArgs, "ntcb_adamw_args")])
def test_layout_matches_c_header(cls, name, tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    fields = [f for f, _ in cls._fields_]
    src = tmp_path / "l.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"%s\"\nint main(void) {\n  printf(\"sizeof %%zu\\n\", sizeof(%s));\n%s"
                   "  return 0;\n}\n" % (ROOT / "include" / "ntc_b200.h", name,
                                         "".join('  printf("%s %%zu\\n", offsetof(%s, %s));\n' % (f, name, f) for f in fields)))
    exe = tmp_path / "l"
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    out = dict(ln.split() for ln in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(out["sizeof"]) == C.sizeof(cls)
    for f in fields:
        assert getattr(cls, f).offset == int(out[f]), f


def test_eps_below_the_normal_numbers_is_refused():
    """Its reciprocal would be infinite and a zero gradient would leave NaN."""
    for eps in (1e-40, 1.17e-38, 5e-324):
        with pytest.raises(ValueError, match="eps"):
            AdamW([torch.zeros(4, 8)], eps=eps)


HOSTILE = """
import ctypes, torch
from neural_block_textures_b200 import AdamW, symbol_logprobs, symbol_logprobs_grad
from neural_block_textures_b200.symbols import _host

class Hostile(torch.Tensor):   # says that it is on a CUDA device and raises on every question about its shape
    @staticmethod
    def __new__(cls):
        return torch.Tensor._make_wrapper_subclass(cls, (4, 8), dtype=torch.float32, device="cuda", dispatch_sizes_strides_policy="sizes")
    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise KeyError(str(func))

x, s = Hostile(), torch.zeros(4, dtype=torch.int64)
for call in (lambda: symbol_logprobs(x, s), lambda: symbol_logprobs_grad(x, s, s.float(), None, s.float()), lambda: AdamW([x])):
    try:
        call()
        raise SystemExit("no exception")
    except KeyError as e:
        assert "aten" in str(e)
one = (ctypes.c_longlong * 1)(32), (ctypes.c_int * 1)(0), (ctypes.c_int * 1)(0)
try:   # as an optimiser's step: no plan is needed to look at the tensors
    _host.ntcb_host_adamw_step(None, [x], [x], 1, *[ctypes.addressof(a) for a in one], 0, None, None, None, 0)
    raise SystemExit("no exception")
except KeyError:
    print("fine")
"""


def test_exceptions_of_tensors_reach_python():
    """A tensor subclass that raises where its sizes are asked for: its exception arrives, and the process goes on."""
    r = subprocess.run([sys.executable, "-c", HOSTILE], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


def test_nested_and_sparse_tensors_are_refused():
    s = torch.zeros(4, dtype=torch.int64)
    nested = torch.nested.nested_tensor([torch.zeros(3), torch.zeros(5)])
    jagged = torch.nested.nested_tensor([torch.zeros(3), torch.zeros(5)], layout=torch.jagged)
    for x in (nested, jagged, torch.zeros(4, 8).to_sparse()):
        with pytest.raises(ValueError, match="strided"):
            symbol_logprobs(x, s)
        with pytest.raises(ValueError, match="strided"):
            symbol_logprobs_grad(x, s, s.float(), None, -1.0)


def test_buffers_off_their_alignment():
    """Every buffer, not the logits and symbols alone: a 32-bit access off its boundary would fault the device."""
    lib, why = abi.load_library(), C.create_string_buffer(256)
    d = C.byref(desc())
    for bad in range(5):
        out = [BUF + 2 * (i == bad) for i in range(5)]
        assert lib.ntcb_symbol_logprobs(d, BUF, BUF, 2, *out, None, why, 256) == 0 and b"aligned" in why.value
    for bad in range(4):   # lse, entropy, dlogp, dentropy
        lse, entropy, dlogp, dentropy = [BUF + 2 * (i == bad) for i in range(4)]
        assert lib.ntcb_symbol_logprobs_grad(d, BUF, BUF, lse, entropy, dlogp, 1, dentropy, 1, BUF, 8, None, why, 256) == 0 and b"aligned" in why.value


def test_an_optimiser_cannot_be_copied():
    """A copy would free the plan of the original a second time."""
    import copy
    import pickle
    opt = AdamW.__new__(AdamW)
    opt.h = None
    for make in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="state_dict"):
            make(opt)
