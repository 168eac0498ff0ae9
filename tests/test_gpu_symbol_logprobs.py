"""symbol_logprobs and its gradient against their formulas in 64 bits: row lengths around every change of kernel, types,
strides, masks, ties, and the ways a user may call them (streams, graphs, in place, broadcast).

Tolerances, from the roundings counted before the first run. A thread adds at most `seq` terms in a row and partial
sums are joined in at most 40 more roundings; each exponential is off by 2^-22 plus 2^-23 per unit of its exponent,
which weighed with the terms themselves is at most log V. So s is off by (seq + 40 + 8 + 4 log V) 2^-24 relatively, and
so is log s absolutely; H adds u / s, off by the same relatively, at most log V + 1 in size."""
import math

import numpy as np
import pytest
import torch

from neural_block_textures_b200 import symbol_logprobs, symbol_logprobs_grad

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LENGTHS = [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 31, 57, 64, 100, 121, 128, 249, 256, 257, 505, 512, 777, 1017, 1018, 1024, 1025, 2047, 4099, 6001]


def seq(v):
    return 32 if v <= 1024 else -(-v // (8 * 256)) * 8 + 8


def tol(v):
    return (seq(v) + 48 + 4 * math.log(v)) * U


def make(n, v, dtype, seed=0, stride=None, offset=0, symbol=torch.int64, scale=3.0, masks=True):
    gen = torch.Generator().manual_seed(seed)
    stride = stride or v
    store = torch.full((n * stride + offset + 64,), 7.0, dtype=DT[dtype])
    x = store[offset:offset + n * stride].view(n, stride)[:, :v]
    x.copy_((torch.randn(n, v, generator=gen) * scale).to(DT[dtype]))
    s = torch.randint(0, v, (n,), generator=gen)
    if masks and n >= 8:
        x[1] = -math.inf                                        # nothing left
        x[2, : v - 1] = -math.inf                               # one logit
        x[3, v // 2:] = torch.finfo(DT[dtype]).min              # masked by the lowest value
        x[4] = torch.finfo(DT[dtype]).min                       # only lowest values: uniform
        x[5, v // 2 + 1:] = -math.inf
        x[6] = 0.5                                              # all equal
        x[7, ::2] = -0.0                                        # signed zeros are one value
        x[7, 1::2] = 0.0
        s[0] = -1
    cuda = store.cuda()
    xc = cuda[offset:offset + n * stride].view(n, stride)[:, :v]
    return xc, s.to(symbol).cuda(), x.double().numpy(), s.numpy()


def reference(x, s, topk):
    """numpy, 64 bits: (logp, entropy, lse, ids, top)."""
    n, v = x.shape
    logp, ent, lse = np.zeros(n), np.zeros(n), np.zeros(n)
    ids, top = np.full((n, topk), -1), np.full((n, topk), -np.inf)
    for r in range(n):
        row = x[r]
        if np.isnan(row).any() or np.isposinf(row).any():
            logp[r] = ent[r] = lse[r] = np.nan
            top[r] = np.nan
        elif np.isneginf(row).all():
            lse[r] = logp[r] = -np.inf
        else:
            m = row.max()
            e = np.exp(row - m)
            log_s = math.log(math.fsum(e))
            lse[r] = m + log_s   # loses log_s beside the lowest finite value, in 64 bits too: the others use m and log_s
            p = e / math.fsum(e)
            ent[r] = -math.fsum(a * (b - m - log_s) for a, b in zip(p[p > 0], row[p > 0]))
            logp[r] = row[s[r]] - m - log_s if 0 <= s[r] < v else 0.0
            order = np.argsort(-row, kind="stable")[:topk]
            order = order[row[order] > -np.inf]
            ids[r, : len(order)] = order
            top[r, : len(order)] = row[order] - m - log_s
        if s[r] < 0:
            logp[r] = 0.0
        elif s[r] >= v:
            logp[r] = np.nan
    return logp, ent, lse, ids, top


def close(got, want, atol, rtol=2 * U):
    got, want = got.double().cpu().numpy(), np.asarray(want, np.float64)
    with np.errstate(over="ignore"):   # outputs are 32 bits: a difference of the two largest logits is infinite there
        want = np.where(np.isinf(want.astype(np.float32)), np.copysign(np.inf, want), want)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        ok = same | (np.abs(got - want) <= atol + rtol * np.abs(want))
    assert ok.all(), (got[~ok][:5], want[~ok][:5], np.argwhere(~ok)[:5])


def check_forward(x, s, x64, s64, topk):
    v = x.shape[1]
    r = symbol_logprobs(x, s, topk=topk)
    logp, ent, lse, ids, top = reference(x64, s64, topk)
    t = tol(v)
    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    close(r.lse, lse, t)
    close(r.logp, logp, t)
    close(r.top_logp, top, t)
    close(r.entropy, ent, 2 * t * (1 + math.log(v)))
    return r


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("v", LENGTHS)
def test_forward_lengths(v, dtype, cuda_device):
    for topk in sorted({0, 1, min(v, 5), min(v, 32)}):
        check_forward(*make(19, v, dtype, seed=v, symbol=torch.int32), topk)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("v", [4, 6, 15, 30, 90, 200, 256, 300, 700, 1200, 9000])
def test_forward_numbers_of_alternatives(v, dtype, cuda_device):
    x, s, x64, s64 = make(17, v, dtype, seed=v + 1)
    for topk in (2, 3, 4, 8, 9, 16, 17, 31):
        if topk <= v:
            check_forward(x, s, x64, s64, topk)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n, v", [(1, 65536), (1, 16385), (2, 30011), (3, 65535), (9, 20000), (40, 9001), (700, 2100), (1, 300007)])
def test_forward_long_rows(n, v, dtype, cuda_device):
    x, s, x64, s64 = make(n, v, dtype, seed=n + v)
    for topk in (0, 20, 32):
        check_forward(x, s, x64, s64, topk)


@pytest.mark.parametrize("v, stride, offset", [(5, 7, 1), (64, 69, 3), (250, 260, 5), (1000, 1003, 7), (3001, 3010, 1)])
@pytest.mark.parametrize("dtype", list(DT))
def test_forward_strides_and_alignment(v, stride, offset, dtype, cuda_device):
    x, s, x64, s64 = make(23, v, dtype, stride=stride, offset=offset, seed=3)
    check_forward(x, s, x64, s64, min(v, 7))
    wide = torch.stack([s, s + 1], 1)[:, 0]   # symbols two apart
    check_forward(x, wide, x64, s64, 0)
    one = x[9:10].expand(6, v)                # one row, six symbols
    check_forward(one, s[:6], np.repeat(x64[9:10], 6, 0), s64[:6], min(v, 3))


@pytest.mark.parametrize("v", [4, 40, 300, 2000, 40000])
def test_rows_that_are_not_numbers(v, cuda_device):
    x, s, x64, s64 = make(12, v, "f32", seed=9)
    for r, c, bad in [(0, 0, math.nan), (3, v - 1, math.nan), (8, v // 2, math.inf), (9, v - 1, math.nan), (10, 1, math.inf)]:
        x[r, c] = bad
        x64[r, c] = bad
    x[10, 2 % v] = math.inf
    x64[10, 2 % v] = math.inf
    r = check_forward(x, s, x64, s64, 2)
    assert (r.top_ids[[0, 3, 8, 9, 10]] == -1).all()
    d = symbol_logprobs_grad(x, s, r.lse, r.entropy, -1.0, 0.5)
    assert d[[0, 3, 8, 9, 10]].isnan().all() and not d[[1, 2, 4, 5, 6, 7, 11]].isnan().any()


@pytest.mark.parametrize("v", [4, 300, 5000])
def test_symbols_outside_the_alphabet(v, cuda_device):
    x, s, x64, s64 = make(5, v, "f32", seed=4)
    s[:] = torch.tensor([-1, v, -(1 << 40), 1 << 40, v - 1])
    r = check_forward(x, s, x64, s.cpu().numpy(), 1)
    d = symbol_logprobs_grad(x, s, r.lse, r.entropy, 1.0)
    assert (d[[0, 2]] == 0).all() and d[[1, 3]].isnan().all() and d[4].isfinite().all()


@pytest.mark.parametrize("symbol", [torch.uint8, torch.int16, torch.int32, torch.int64])
def test_symbol_types(symbol, cuda_device):
    x, s, x64, s64 = make(33, 100, "f16", symbol=symbol, masks=False)
    check_forward(x, s, x64, s64, 3)


@pytest.mark.parametrize("kind", ["ascending", "descending", "equal", "two_values", "one_thread"])
@pytest.mark.parametrize("v", [256, 1000, 5000, 65536])
def test_alternatives_of_hard_rows(kind, v, cuda_device):
    i = torch.arange(v)
    x = {"ascending": i.float(), "descending": -i.float(), "equal": torch.zeros(v), "two_values": (i % 2).float(),
         "one_thread": torch.where(i // 8 % 256 == 3, 5.0 + (i % 97).float() / 97, 0.0)}[kind] / 16.0
    x = x.repeat(3, 1)
    s = torch.tensor([0, v // 2, v - 1])
    check_forward(x.cuda(), s.cuda(), x.double().numpy(), s.numpy(), 32)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("v", [4, 8, 60, 256, 700, 3000])
def test_subnormal_and_extreme_logits(v, dtype, cuda_device):
    """Subnormal numbers keep their order among themselves and around the two zeros; the largest finite values stand."""
    info = torch.finfo(DT[dtype])
    gen = torch.Generator().manual_seed(v)
    tiny = info.smallest_normal * info.eps   # the smallest subnormal
    x = torch.zeros(6, v, dtype=DT[dtype])
    x[0] = (torch.randint(-3, 4, (v,), generator=gen).double() * tiny).to(DT[dtype])
    x[1] = torch.where(torch.arange(v) % 2 == 0, -0.0, 0.0)
    x[1, v // 2] = tiny
    x[2] = info.max * (torch.randint(0, 2, (v,), generator=gen) * 2 - 1)
    x[3] = info.min
    x[3, v - 1] = info.max
    x[4] = torch.linspace(-60, 60, v).to(DT[dtype])
    x[5, 1:] = -info.max
    s = torch.tensor([0, 1, v - 1, v - 1, v // 2, 0])
    for topk in sorted({1, 2, min(v, 8), min(v, 20)}):
        check_forward(x.cuda(), s.cuda(), x.double().numpy(), s.numpy(), topk)


def grad_reference(x, s, dl, dh):
    n, v = x.shape
    dx, scale = np.zeros((n, v)), np.zeros((n, v))
    _, ent, lse, _, _ = reference(x, s, 0)
    for r in range(n):
        if np.isneginf(lse[r]):
            continue
        m = x[r].max()
        lp = x[r] - m - math.log(math.fsum(np.exp(x[r] - m)))
        p = np.exp(lp)
        lp = np.where(p > 0, lp, 0.0)
        a = dl[r] if s[r] >= 0 else 0.0
        dx[r] = -p * (a + dh[r] * (lp + ent[r]))
        # roundings: the exponent (2^-23 of its size and of lse's), the exponential, the factor, the product; a large lse
        # (256 or more) is replaced by a new sum of the row, off by tol(v)
        size = 4 * abs(lse[r]) if abs(lse[r]) < 256 else 2 * tol(v) / U
        scale[r] = p * (abs(a) + abs(dh[r]) * (np.abs(lp) + ent[r] + 1)) * (8 + 4 * np.abs(lp) + size) * U
        scale[r] += p * abs(dh[r]) * 2 * tol(v) * (1 + math.log(v))
        # probabilities below the smallest normal number are flushed to zero
        scale[r] += 2.0 ** -126 * (abs(a) + abs(dh[r]) * (np.abs(lp) + ent[r] + 1))
        if s[r] >= 0:
            dx[r, s[r]] += a
            scale[r, s[r]] += 2 * U * abs(a)
    return dx, scale


def check_grad(x, s, x64, s64, dl, dh, dtype, **kw):
    r = symbol_logprobs(x, s)
    got = symbol_logprobs_grad(x, s, r.lse, r.entropy, dl, dh, **kw)
    n = len(s64)
    full = lambda g: np.zeros(n) if g is None else g.double().cpu().numpy() if isinstance(g, torch.Tensor) else np.full(n, np.float32(g), np.float64)
    want, scale = grad_reference(x64, s64, full(dl), full(dh))
    info = torch.finfo(DT[dtype])
    err = np.abs(got.double().cpu().numpy() - want)
    bad = ~(err <= scale + np.abs(want) * info.eps / 2 + info.smallest_normal * info.eps)
    assert not bad.any(), (err[bad].max(), np.argwhere(bad)[:4])
    assert got.dtype == DT[dtype]
    return got


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("v", [1, 2, 4, 5, 8, 25, 64, 121, 128, 256, 500, 505, 512, 1000, 4099])
def test_gradient(v, dtype, cuda_device):
    x, s, x64, s64 = make(21, v, dtype, seed=v)
    gen = torch.Generator().manual_seed(v)
    dl, dh = torch.randn(21, generator=gen).cuda(), torch.randn(21, generator=gen).cuda()
    check_grad(x, s, x64, s64, dl, dh, dtype)
    check_grad(x, s, x64, s64, dl, None, dtype)
    check_grad(x, s, x64, s64, -0.25, 0.5, dtype)
    check_grad(x, s, x64, s64, dl[:1].expand(21), torch.stack([dh, dl], 1)[:, 0], dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v, stride, offset", [(4, 5, 1), (63, 69, 3), (1000, 1001, 1), (5003, 5011, 7)])
def test_gradient_strides_and_in_place(v, stride, offset, dtype, cuda_device):
    x, s, x64, s64 = make(14, v, dtype, stride=stride, offset=offset, seed=5)
    want = check_grad(x, s, x64, s64, -1.0, 0.1, dtype)
    store = torch.full((14, v + 9), 3.0, dtype=DT[dtype], device="cuda")
    check_grad(x, s, x64, s64, -1.0, 0.1, dtype, out=store[:, 4:4 + v])
    assert (store[:, :4] == 3).all() and (store[:, 4 + v:] == 3).all()   # nothing beside the rows is written
    r = symbol_logprobs(x, s)
    out = symbol_logprobs_grad(x, s, r.lse, r.entropy, -1.0, 0.1, out=x)
    assert out.data_ptr() == x.data_ptr() and torch.equal(x, want)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("v", [2, 4, 7, 30, 250, 1000, 1100, 2100, 4200, 9000, 40000])
def test_gradient_of_rows_far_from_zero(v, dtype, cuda_device):
    """A softmax does not change with a shift of its logits: rows around a large value, rows wholly masked by large finite
    values (the type's lowest, -1e9 or what the type has of it), one logit beside them; in place gives the same."""
    info = torch.finfo(DT[dtype])
    gen = torch.Generator().manual_seed(v)
    base = torch.randn(9, v, generator=gen) * 2
    x = base.clone()
    x[1] = info.min
    x[2] = max(-1e9, info.min)
    x[3] = info.max
    x[4] = x[4] * 8 + 3000
    x[5] = x[5] * 8 - 3000
    x[6] = info.min
    x[6, v // 2] = 1.0
    x[7] = max(-1e9, info.min)
    x[7, v - 1] = 2.0
    x[8] = x[8] + 300
    x = x.to(DT[dtype])
    s = torch.randint(0, v, (9,), generator=gen)
    x64, s64, x, s = x.double().numpy(), s.numpy(), x.cuda(), s.cuda()
    dl, dh = torch.randn(9, generator=gen).cuda(), torch.randn(9, generator=gen).cuda()
    check_grad(x, s, x64, s64, dl, None, dtype)
    want = check_grad(x, s, x64, s64, dl, dh, dtype)
    check_forward(x, s, x64, s64, min(v, 5))   # its sums may be rounded otherwise than without alternatives
    r = symbol_logprobs(x, s)
    symbol_logprobs_grad(x, s, r.lse, r.entropy, dl, dh, out=x)
    assert torch.equal(x, want)


def test_gradient_against_differences(cuda_device):
    """(f(x + h e) - f(x - h e)) / 2h in 64 bits of the formula, and of the kernel along one direction."""
    n, v, h = 6, 37, 1e-5
    x, s, x64, s64 = make(n, v, "f32", seed=8, masks=False)
    gen = np.random.default_rng(1)
    dl, dh = gen.standard_normal(n), gen.standard_normal(n)
    f = lambda y: float((dl * reference(y, s64, 0)[0] + dh * reference(y, s64, 0)[1]).sum())
    r = symbol_logprobs(x, s)
    got = symbol_logprobs_grad(x, s, r.lse, r.entropy, torch.tensor(dl).float().cuda(), torch.tensor(dh).float().cuda()).double().cpu().numpy()
    for r_, c in [(0, 0), (1, 5), (2, int(s64[2])), (3, 36), (4, int(s64[4])), (5, 20)]:
        e = np.zeros_like(x64)
        e[r_, c] = h
        slope = (f(x64 + e) - f(x64 - e)) / (2 * h)
        # central differences: h^2 / 6 of the third derivative (below 20 here) and 64-bit rounding over h
        assert abs(slope - got[r_, c]) < 20 * h * h + 1e-9 + 1e-5 * (abs(dl[r_]) + abs(dh[r_]))


def test_empty_and_refused(cuda_device):
    x, s, _, _ = make(9, 50, "f32")
    r = symbol_logprobs(x[:0], s[:0], topk=4)
    assert r.logp.shape == (0,) and r.top_ids.shape == (0, 4)
    assert symbol_logprobs_grad(x[:0], s[:0], r.lse, r.entropy, -1.0).shape == (0, 50)
    r = symbol_logprobs(x, s)
    for bad in (lambda: symbol_logprobs(x, s, topk=33), lambda: symbol_logprobs(x[:, :4], s, topk=5), lambda: symbol_logprobs(x, s, topk=-1),
                lambda: symbol_logprobs(x.t(), s[:1].expand(50)), lambda: symbol_logprobs(x, s.cpu()),
                lambda: symbol_logprobs_grad(x, s, r.lse[:4], r.entropy, -1.0), lambda: symbol_logprobs_grad(x, s, r.lse, None, -1.0, 1.0),
                lambda: symbol_logprobs_grad(x, s, r.lse, r.entropy, r.lse.double()),
                lambda: symbol_logprobs_grad(x, s, r.lse, r.entropy, -1.0, out=x.half()),
                lambda: symbol_logprobs_grad(x, s, r.lse, r.entropy, -1.0, out=x[:1].expand(9, 50))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("n, v", [(40, 4), (40, 200), (3, 20000)])
def test_streams_and_graphs(n, v, cuda_device):
    x, s, x64, s64 = make(n, v, "bf16", seed=2)
    want = symbol_logprobs(x, s, topk=3)
    dwant = symbol_logprobs_grad(x, s, want.lse, want.entropy, -1.0, 0.3)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:   # two calls at once
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(symbol_logprobs(x, s, topk=3))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    dl = torch.full((n,), -1.0, device="cuda")
    dh = torch.full((n,), 0.3, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = symbol_logprobs(x, s, topk=3)
        d = symbol_logprobs_grad(x, s, r.lse, r.entropy, dl, dh)
    for _ in range(2):
        r.logp.zero_()
        d.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(r, want)) and torch.equal(d, dwant)
    y, s2, y64, s64b = make(n, v, "bf16", seed=77)
    x.copy_(y)
    s.copy_(s2)
    graph.replay()   # new inputs in the same buffers
    fresh = symbol_logprobs(y, s2, topk=3)
    assert all(torch.equal(a, b) for a, b in zip(r, fresh))


def test_out_between_the_logits_rows(cuda_device):
    store = torch.zeros(7, 40, device="cuda")
    x, s, _, _ = make(7, 16, "f32", seed=3, masks=False)
    store[:, 3:19] = x
    r = symbol_logprobs(store[:, 3:19], s)
    want = symbol_logprobs_grad(x, s, r.lse, r.entropy, -1.0)
    got = symbol_logprobs_grad(store[:, 3:19], s, r.lse, r.entropy, -1.0, out=store[:, 20:36])
    assert torch.equal(got, want) and torch.equal(store[:, 3:19], x) and (store[:, 36:] == 0).all()
    for out in (store[:, 4:20], store.view(-1)[1:1 + 7 * 32].view(7, 32)[:, :16]):
        with pytest.raises(RuntimeError, match="overlaps"):
            symbol_logprobs_grad(store[:, 3:19], s, r.lse, r.entropy, -1.0, out=out)


def test_first_call_inside_a_capture(cuda_device):
    """A fresh process whose first use of the kernels is a captured one."""
    import subprocess
    import sys
    from pathlib import Path
    code = (
        "import torch\n"
        "from neural_block_textures_b200 import AdamW, symbol_logprobs, symbol_logprobs_grad\n"
        "x = torch.randn(50, 300, device='cuda'); s = torch.zeros(50, dtype=torch.int32, device='cuda')\n"
        "dl = torch.full((50,), -1.0, device='cuda'); opt = AdamW([x], state_bits=8, weight_decay=0.0)\n"
        "it = torch.zeros(1, dtype=torch.int64, device='cuda'); g = torch.cuda.CUDAGraph(); torch.cuda.synchronize()\n"
        "with torch.cuda.graph(g):\n"
        "    r = symbol_logprobs(x, s, topk=3); d = symbol_logprobs_grad(x, s, r.lse, r.entropy, dl); it.add_(1); opt.step(it, 0.1, [d])\n"
        "before = x.clone(); g.replay(); torch.cuda.synchronize()\n"
        "moved = before - x; ok = (moved.abs() - 0.1).abs() < 1e-3\n"
        "assert ok[d.abs() > 1e-4].all() and torch.equal(moved[d.abs() > 1e-4].sign(), d[d.abs() > 1e-4].sign()); print('fine')\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


def test_rate_under_the_counts_is_the_progress_prints(cuda_device):
    """Level 0's palette indices rated under the logarithms of their counts: the mean code length and the entropy are the
    order-0 figure that print_stats gives for the level. Every cell shares one row of logits (row stride 0)."""
    from neural_block_textures_b200 import Trainer

    from .helpers import spec_named, target_for
    for name in ("cfg2", "cfg3", "generic"):
        spec = spec_named(name)
        z, p = spec.init_params()
        with Trainer() as tr:
            ok, why = tr.init(spec.model_desc(), z, p, target_for(spec))
            assert ok, why
            for it in range(1, 4):
                tr.mlp_step(it, 0.02, 0.005, 16, 256)
                tr.qat_search()
            stats, _ = tr.print_stats()
            z, _ = tr.download_model()
        level = spec.levels[0]
        bits = entropy = 0.0
        for c, depth in enumerate(spec.qat_bits):
            values = z[:level.size].reshape(-1, level.C)[:, c]
            index = torch.tensor(np.rint((values.astype(np.float64) + 1) / 2 * ((1 << depth) - 1)).astype(np.uint8), device="cuda")
            count = torch.bincount(index.long(), minlength=1 << depth)
            r = symbol_logprobs(count.float().log()[None].expand(len(index), -1), index)
            bits += -r.logp.double().sum().item() / math.log(2)
            entropy += r.entropy[0].double().item() * len(index) / math.log(2)
        # log of a count, log of their sum and their difference: a few 2^-24 of log(4096) each
        for got in (bits, entropy):
            assert abs(got / (spec.W * spec.H) - stats.bpp_ctx_level0) < 2e-5 * max(stats.bpp_ctx_level0, 1.0), name


def test_rows_behind_32_bits(cuda_device):
    """Offsets past 2^32 elements: the last rows of 4.3 G logits."""
    v = 65536
    n = (1 << 16) + 40
    x = torch.empty(n, v, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(1)
    tail = (torch.randn(8, v, generator=gen) * 3).to(torch.bfloat16)
    x[:n - 8] = 0.0
    x[n - 8:] = tail.cuda()
    s = torch.randint(0, v, (n,), generator=gen)
    r = symbol_logprobs(x, s.cuda(), topk=4)
    logp, ent, lse, ids, top = reference(tail.double().numpy(), s[n - 8:].numpy(), 4)
    close(r.logp[n - 8:], logp, tol(v))
    close(r.entropy[n - 8:], ent, 2 * tol(v) * (1 + math.log(v)))
    assert np.array_equal(r.top_ids[n - 8:].cpu().numpy(), ids)
    assert (r.top_ids[:n - 8] == torch.arange(4, device="cuda")).all()
    close(r.lse[:n - 8], np.full(n - 8, math.log(v)), tol(v))
    want = symbol_logprobs_grad(tail.cuda(), s[n - 8:].cuda(), r.lse[n - 8:], r.entropy[n - 8:], -1.0)
    symbol_logprobs_grad(x, s.cuda(), r.lse, r.entropy, -1.0, out=x)
    assert torch.equal(x[n - 8:], want)


def entropy_bound(x, v, long_row):
    """What the entropy of one row may be off by. s sums e^d and u sums e^d d (one sign each, so nothing cancels): every
    term is off by its exponential's 4 U and its exponent's 2.5 U |d| (a constant, a difference and a product rounded),
    every sum and join by the roundings counted in `sums`; log s by two units, the quotient by four, their difference by
    one, the offset of the exponents by 2 U. Lanes add at most 32 pairs one after another and join 6 times; a thread of a
    long row adds 16 pairs and is moved to a new maximum (12 roundings) a round, and the parts join 11 times."""
    d = x[x > -np.inf] - x.max()
    p = np.exp(d)
    p /= math.fsum(p)
    e1, e2 = -math.fsum(p * d), math.fsum(p * d * d)
    log_s = math.log(math.fsum(np.exp(d)))
    rounds = min(8, -(-v // (4 * 4 * 256)))   # few rows: threads of 4 vectors, up to 256 of them a CTA, then more rounds
    sums = 28 * rounds + 12 * 11 if long_row else 40
    rel_s = sums + 6 + 2.5 * e1
    return U * (rel_s * (1 + e1) + (sums + 10) * e1 + 2.5 * e2 + 2 * log_s + 4 * e1 + (log_s + e1))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("v", [3, 4, 11, 16, 60, 250, 256, 700, 1000, 1025, 4099, 9000, 65536])
def test_entropy_of_rows_around_a_value(v, dtype, cuda_device):
    """Logits of an ordinary spread around values up to where the exponents change their form: the entropy does not depend
    on the value, and the gradient's entropy term, which reads it, neither."""
    centres = [0, 3, 30, -100, 300, -300, 1000, -1000, 3000, -3000, 4080, -4080]
    gen = torch.Generator().manual_seed(v)
    x = (torch.randn(len(centres), v, generator=gen) * 2.5 + torch.tensor(centres)[:, None]).to(DT[dtype])
    s = torch.randint(0, v, (len(centres),), generator=gen)
    x64, s64 = x.double().numpy(), s.numpy()
    _, want, _, _, _ = reference(x64, s64, 0)
    limit = np.array([entropy_bound(row, v, v > 250) for row in x64])
    for topk in sorted({0, 1, min(v, 3), min(v, 8), min(v, 20)}):
        r = check_forward(x.cuda(), s.cuda(), x64, s64, topk)
        err = np.abs(r.entropy.double().cpu().numpy() - want)
        assert (err <= limit).all(), (topk, err, limit)
    if v <= 4099:
        dl, dh = torch.randn(len(centres), generator=gen).cuda(), torch.randn(len(centres), generator=gen).cuda()
        check_grad(x.cuda(), s.cuda(), x64, s64, dl, dh, dtype)


def test_negated_views(cuda_device):
    """The imaginary part of a conjugate is a view whose memory holds the values' negatives."""
    negated = lambda n: torch.randn(n, dtype=torch.complex64, device="cuda").conj().imag
    x, s, _, _ = make(9, 40, "f32", masks=False)
    r = symbol_logprobs(x, s)
    dl, dh, lse, h = negated(9), negated(9), negated(9), negated(9)
    assert dl.is_neg() and dh.is_neg()
    for args in ((r.lse, r.entropy, dl, None), (r.lse, r.entropy, dl, dh), (r.lse, h, dl, dh), (lse, r.entropy, -1.0, dh)):
        got = symbol_logprobs_grad(x, s, *args)
        assert torch.equal(got, symbol_logprobs_grad(x, s, *[a.clone() if isinstance(a, torch.Tensor) else a for a in args]))
    column = torch.stack([torch.zeros(9, device="cuda"), -x[:, 0]], 1)   # one logit a row, two floats apart
    one = torch.view_as_complex(column).conj().imag[:, None]
    assert one.is_neg() and torch.equal(one, x[:, :1])
    z = torch.zeros_like(s)
    a, b = symbol_logprobs(one, z, topk=1), symbol_logprobs(x[:, :1], z, topk=1)
    assert torch.equal(a.lse, b.lse) and torch.equal(a.logp, b.logp)
    da, db = (symbol_logprobs_grad(y, z, a.lse, a.entropy, -1.0, 0.5) for y in (one, x[:, :1]))
    assert torch.equal(da, db)
    with pytest.raises(ValueError, match="negated"):
        symbol_logprobs_grad(x[:, :1], z, a.lse, a.entropy, -1.0, out=one)


def test_nested_tensors_and_memory_that_runs_out(cuda_device):
    """torch's own exceptions arrive as what they are."""
    nested = torch.nested.nested_tensor([torch.zeros(3, device="cuda"), torch.zeros(5, device="cuda")])
    s = torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="nested"):
        symbol_logprobs(nested, s)
    with pytest.raises(ValueError, match="nested"):
        symbol_logprobs_grad(nested, s, s.float(), None, s.float())
    row, none = torch.zeros(1, 1 << 20, device="cuda"), torch.zeros(1, dtype=torch.uint8, device="cuda")
    n = 1 << 19   # rows of one shared row: a gradient of 2 TB
    per_row = torch.zeros(1, device="cuda").expand(n)
    with pytest.raises(torch.OutOfMemoryError):
        symbol_logprobs_grad(row.expand(n, 1 << 20), none.expand(n), torch.zeros(n, device="cuda"), None, per_row)


def test_other_threads_run_while_a_call_waits_for_the_queue(cuda_device):
    """More calls than the launch queue holds behind about half a second of device work: a call that waits for a place in
    it does not hold the interpreter."""
    import threading
    import time
    x, s, _, _ = make(6, 9, "f32", masks=False)
    one, half = torch.full((6,), -1.0, device="cuda"), torch.full((6,), 0.5, device="cuda")
    r = symbol_logprobs(x, s)
    symbol_logprobs_grad(x, s, r.lse, r.entropy, one, half)
    torch.cuda.synchronize()
    for call in (lambda: symbol_logprobs(x, s), lambda: symbol_logprobs_grad(x, s, r.lse, r.entropy, one, half)):
        longest, done = [0.0], threading.Event()

        def tick():
            last = time.perf_counter()
            while not done.is_set():
                time.sleep(0.0005)
                now = time.perf_counter()
                longest[0], last = max(longest[0], now - last), now
        thread = threading.Thread(target=tick)
        thread.start()
        torch.cuda._sleep(1_000_000_000)   # device clocks
        begin = time.perf_counter()
        for _ in range(3000):
            call()
        took = time.perf_counter() - begin
        done.set()
        thread.join()
        torch.cuda.synchronize()
        assert longest[0] < max(0.1, took / 4), (longest, took)


@pytest.mark.parametrize("dtype, n, v", [("f32", 1, 300007), ("f32", 3, 40000), ("bf16", 2, 200001), ("f32", 700, 20000), ("f16", 300, 50001), ("f32", 160, 9001)])
def test_gradient_of_long_rows_far_from_zero(dtype, n, v, cuda_device):
    """Rows of many CTAs whose sum is taken anew, few and many of them, beside ordinary ones: the numbers of a call over
    the logits, and, for the first rows, the formula's."""
    gen = torch.Generator().manual_seed(v)
    x = torch.randn(n, v, generator=gen) * 2
    x[::3] += 1000.0
    x[1::3] = max(-1e9, torch.finfo(DT[dtype]).min)
    x[1::3, v // 3] = 2.0
    if n > 4:
        x[4] = torch.finfo(DT[dtype]).min
    x = x.to(DT[dtype])
    s = torch.randint(0, v, (n,), generator=gen)
    dl, dh = torch.randn(n, generator=gen).cuda(), torch.randn(n, generator=gen).cuda()
    few = min(n, 6)
    check_grad(x[:few].cuda(), s[:few].cuda(), x[:few].double().numpy(), s[:few].numpy(), dl[:few], dh[:few], dtype)
    x, s = x.cuda(), s.cuda()
    r = symbol_logprobs(x, s)
    got = symbol_logprobs_grad(x, s, r.lse, r.entropy, dl, dh)
    assert torch.equal(symbol_logprobs_grad(x, s, r.lse, r.entropy, dl, dh, out=x), got)


def test_cost_of_rows_far_from_zero(cuda_device):
    """Few CTAs of a long row take its sum anew, so the cost keeps to the row's length: eight times the logits take less
    than 24 times as long (eight by the bytes; each of a row's CTAs summing all of it would be 64)."""
    times = []
    for v in (1 << 20, 1 << 23):
        x = torch.full((1, v), -1e9, device="cuda")
        s = torch.zeros(1, dtype=torch.int32, device="cuda")
        r = symbol_logprobs(x, s)
        one = torch.ones(1, device="cuda")
        best = math.inf
        for _ in range(5):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            symbol_logprobs_grad(x, s, r.lse, r.entropy, one)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end))
        times.append(best)
    assert times[1] < 24 * times[0], times


def test_logits_that_require_a_gradient(cuda_device):
    """autograd records nothing, and says so: a warning on the caller's line, the same numbers."""
    import warnings

    import torch.autograd.forward_ad as forward_ad
    x, s, _, _ = make(6, 9, "f32", masks=False)
    want = symbol_logprobs(x, s, topk=2)
    leaf = x.clone().requires_grad_()
    with pytest.warns(UserWarning, match="records nothing") as seen:
        got = symbol_logprobs(leaf, s, topk=2)
    assert seen[0].filename == __file__ and not got.logp.requires_grad
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with forward_ad.dual_level(), pytest.warns(UserWarning, match="records nothing"):
        symbol_logprobs(forward_ad.make_dual(x, torch.ones_like(x)), s)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        symbol_logprobs(leaf.detach(), s)
        with torch.no_grad():
            symbol_logprobs(leaf, s)
        with pytest.raises(UserWarning):
            symbol_logprobs(leaf, s)
        d = symbol_logprobs_grad(leaf, s, want.lse, want.entropy, -1.0)   # the gradient itself, handed on
    leaf.backward(d)
    assert torch.equal(leaf.grad, d)


def test_a_gradient_over_the_logits_is_seen_by_backward_passes(cuda_device):
    x, s, _, _ = make(6, 9, "f32", masks=False)
    r = symbol_logprobs(x, s)
    w = torch.ones(6, 9, device="cuda", requires_grad=True)
    loss = (w * x).sum()   # saves x
    symbol_logprobs_grad(x, s, r.lse, r.entropy, -1.0, out=x)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_a_tensor_subclass_that_makes_new_objects(cuda_device):
    class Fresh(torch.Tensor):
        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            r = super().__torch_function__(func, types, args, kwargs or {})
            return r.detach().clone().as_subclass(cls) if func is torch.Tensor.resolve_neg else r
    x, s, _, _ = make(6, 9, "f32", masks=False)
    r = symbol_logprobs(x, s)
    want = symbol_logprobs_grad(x, s, r.lse, r.entropy, -1.0, 0.5)
    assert torch.equal(symbol_logprobs_grad(x.as_subclass(Fresh), s, r.lse, r.entropy.as_subclass(Fresh), -1.0, 0.5).as_subclass(torch.Tensor), want)
