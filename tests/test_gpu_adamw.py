"""AdamW against its formula: 32-bit moments and parameters in 64 bits; the 8-bit codes bit for bit against numpy's
elementary 32-bit operations and the counter noise; sizes, types, alignments, many tensors, graphs and checkpoints.

Tolerances: the moments take three roundings of terms no larger than themselves and the gradient's (4 half steps of
each term). The parameter's update u = lr mh / (sqrt(vh) + eps) takes the moments' roundings, an approximate square
root and quotient (2 + 4 units) and four more: 2^-20 of |u| is above their sum. The parameter adds two roundings, and its own
type's: half of eps relatively, and below the smallest normal number (2^-14 for fp16, which parameters near 0 reach) half
of the subnormals' fixed step, smallest_normal * eps / 2."""
import math

import numpy as np
import pytest
import torch

from neural_block_textures_b200 import AdamW, symbol_logprobs, symbol_logprobs_grad

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = [1, 2, 7, 8, 9, 255, 256, 257, 0, 2047, 2048, 2049, 5000, 100003]
M64 = (1 << 64) - 1


def tensors(sizes, dtype, seed, scale, offset=0):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        t = torch.empty(n + offset + 8, dtype=DT[dtype], device="cuda")
        t[offset:offset + n] = (torch.randn(n, generator=gen) * scale).to(DT[dtype]).cuda()
        out.append(t[offset:offset + n])
    return out


def type_rounding(dtype, want):
    info = torch.finfo(DT[dtype])
    return np.maximum(info.eps / 2 * np.abs(want), info.smallest_normal * info.eps / 2)


def f64(t):
    return t.double().cpu().numpy()


def step64(p, g, m, v, it, lr, b1, b2, eps, wd, scale):
    g = g * scale
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    u = lr * (m / (1 - b1 ** it)) / (np.sqrt(v / (1 - b2 ** it)) + eps)
    return p - lr * wd * p - u, m, v, u


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("pd, gd", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "bf16"), ("bf16", "f16")])
def test_32_bit_states(pd, gd, offset, cuda_device):
    p = tensors(SIZES, pd, 1, 0.5, offset)
    opt = AdamW(p, weight_decay=0.1, betas=(0.9, 0.99), eps=1e-6, grad_dtype=DT[gd])
    m, v = [np.zeros(n) for n in SIZES], [np.zeros(n) for n in SIZES]
    for it in (1, 2, 3):
        g = tensors(SIZES, gd, 10 + it, 0.02, offset)
        before = [f64(t) for t in p]
        m0, v0 = opt.moments()
        m0, v0 = [f64(t) for t in m0], [f64(t) for t in v0]
        opt.step(it, 0.01, g, grad_scale=0.5)
        m1, v1 = opt.moments()
        for i in range(len(SIZES)):
            g64 = f64(g[i])
            want_p, want_m, want_v, u = step64(before[i], g64, m0[i], v0[i], it, 0.01, 0.9, 0.99, 1e-6, 0.1, 0.5)
            assert (np.abs(f64(m1[i]) - want_m) <= 4 * U * (np.abs(m0[i]) + np.abs(g64))).all()
            assert (np.abs(f64(v1[i]) - want_v) <= 5 * U * want_v + 1e-44).all()
            # m may cancel: its absolute error over the denominator
            den = np.sqrt(want_v / (1 - 0.99 ** it)) + 1e-6
            slack = 2.0 ** -20 * np.abs(u) + 0.01 / (1 - 0.9 ** it) * 4 * U * (np.abs(m0[i]) + np.abs(g64)) / den
            assert (np.abs(f64(p[i]) - want_p) <= slack + 2 * U * np.abs(before[i]) + type_rounding(pd, want_p)).all()


# ---- the 8-bit states restated in numpy: elementary 32-bit operations and integers
def mix(x):
    x = (x + 0x9E3779B97F4A7C15) & M64
    x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & M64
    x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & M64
    return x ^ (x >> 31)


def noise(seed, it, tensor, n):
    key = mix((seed & M64) ^ (5 << 56) ^ ((it & 0xFFFFFFFF) << 32) ^ tensor)
    with np.errstate(over="ignore"):
        x = np.uint64(key) + np.arange((n + 1) // 2, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15)
        x = x + np.uint64(0x9E3779B97F4A7C15)
        x = (x ^ (x >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        x = (x ^ (x >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        x = x ^ (x >> np.uint64(31))
    w = np.stack([(x >> np.uint64(s)) & np.uint64(0xFFFF) for s in (0, 16, 32, 48)], 1).reshape(-1, 2)[:n].astype(np.int64)
    return w[:, 0], w[:, 1]


def grid(x, add):
    bits = np.abs(x).view(np.uint32).astype(np.int64)
    return np.where(bits < 0x7F800000, np.minimum((bits + add) >> 20, 0x7F7), 0), bits


def encode(x, add, top):
    n = len(x)
    q, bits = grid(x, add)
    pad = np.concatenate([q, np.zeros(-n % 256, np.int64)]).reshape(-1, 256)
    base = np.maximum(pad.max(1) - top, 0)
    c = np.maximum(q - np.repeat(base, 256)[:n], 0)
    if top == 254:
        c = np.where(bits > 0, np.maximum(c, 1), c)
    c = np.where(bits >= 0x7F800000, top + 1, c)
    if top == 126:
        c = np.where((c > 0) & np.signbit(x), c | 128, c)
    return c, base


def decode(c, base, top):
    mag = c & 127 if top == 126 else c
    bits = np.where(mag == 0, 0, np.where(mag > top, 0x7FC00000, (mag + np.repeat(base, 256)[:len(c)]) << 20)).astype(np.uint32)
    x = bits.view(np.float32)
    return np.where(c & 128, -x, x) if top == 126 else x


def codes(opt, i, n):
    total = opt.offsets[-1]
    raw = opt.state.cpu().numpy()
    o = opt.offsets[i]
    nb = -(-n // 256)
    win = raw[2 * total:].view(np.uint16).astype(np.int64)
    return (raw[o:o + n].astype(np.int64), win[o // 256:o // 256 + nb], raw[total + o:total + o + n].astype(np.int64),
            win[total // 256 + o // 256:total // 256 + o // 256 + nb])


@pytest.mark.parametrize("pd, gd, offset", [("f32", "f32", 0), ("f32", "f32", 1), ("bf16", "bf16", 0), ("f16", "f32", 3), ("bf16", "f16", 1)])
def test_8_bit_states_bit_for_bit(pd, gd, offset, cuda_device):
    seed = 0x1234567890ABCDEF
    p = tensors(SIZES, pd, 1, 0.5, offset)
    opt = AdamW(p, state_bits=8, weight_decay=0.02, seed=seed, grad_dtype=DT[gd])
    f = np.float32
    b1, c1, b2, c2 = f(0.9), f(1 - 0.9), f(0.999), f(1 - 0.999)
    for it in (1, 2, 3, 4):
        g = tensors(SIZES, gd, 20 + it, 0.02, offset)
        if it == 3:
            g[7][5:9] = 0.0                      # a moment that decays
            g[12][100] = 1000.0 if gd != "f16" else 500.0   # a block with one large value
        before = [codes(opt, i, n) for i, n in enumerate(SIZES)]
        pb = [f64(t) for t in p]
        opt.step(it, 0.01, g, grad_scale=0.25)
        vals = opt.moments()
        for i, n in enumerate(SIZES):
            cm, bm, cv, bv = before[i]
            gs = g[i].float().cpu().numpy() * f(0.25)
            m = decode(cm, bm, 126) * b1 + gs * c1
            v = decode(cv, bv, 254) * b2 + (gs * gs) * c2
            rm, rv = noise(seed, it, i, n)
            want = [*encode(m, rm << 4, 126), *encode(v, rv << 4, 254)]
            got = codes(opt, i, n)
            for a, b in zip(got, want):
                assert np.array_equal(a, b)
            assert np.array_equal(vals[0][i].cpu().numpy(), decode(got[0], got[1], 126))
            assert np.array_equal(vals[1][i].cpu().numpy(), decode(got[2], got[3], 254))
            u = 0.01 * (m.astype(np.float64) / (1 - 0.9 ** it)) / (np.sqrt(v.astype(np.float64) / (1 - 0.999 ** it)) + 1e-8)
            want_p = pb[i] * (1 - 0.01 * 0.02) - u
            assert (np.abs(f64(p[i]) - want_p) <= 2.0 ** -20 * np.abs(u) + 2 * U * np.abs(pb[i]) + type_rounding(pd, want_p)).all()


def test_8_bit_values_and_rounding(cuda_device):
    """Set moments round to nearest (half a step: 2^-4 of the value), signs and zeros survive, a second moment above zero
    stays above zero, infinities and NaN become NaN, and stochastic rounding is unbiased."""
    n = 4096
    gen = torch.Generator().manual_seed(3)
    p = [torch.zeros(n, device="cuda")]
    opt = AdamW(p, state_bits=8)
    m = (torch.randn(n, generator=gen) * torch.exp2(-torch.rand(n, generator=gen) * 10)).cuda()
    v = (torch.rand(n, generator=gen) + 0.01).cuda() * torch.exp2(-torch.rand(n, generator=gen) * 25).cuda()
    m[:3] = torch.tensor([0.0, -0.0, 1e-30])
    v[:3] = torch.tensor([0.0, 1e-38, 1e-44])
    opt.set_moments([m], [v])
    m1, v1 = (x[0] for x in opt.moments())
    top = m.abs().view(-1, 256).amax(1).repeat_interleave(256)
    ok = (m1 - m).abs() <= torch.maximum(m.abs() / 16, top * 2.0 ** -15)   # below the window: zero
    assert ok.all() and (m1[:3] == 0).all()
    assert v1[0] == 0 and (v1[1:] > 0).all()
    vtop = v.view(-1, 256).amax(1).repeat_interleave(256)
    assert ((v1 - v).abs() <= torch.maximum(v / 16, vtop * 2.0 ** -30)).all()
    opt.set_moments([m1], [v1])   # what is on the grid stays
    m2, v2 = (x[0] for x in opt.moments())
    assert torch.equal(m1, m2) and torch.equal(v1, v2)
    m[256], m[600], v[900], v[901] = math.nan, -math.inf, math.inf, math.nan
    opt.set_moments([m], [v])
    m3, v3 = (x[0] for x in opt.moments())
    assert m3[[256, 600]].isnan().all() and v3[[900, 901]].isnan().all() and m3.isnan().sum() == 2 and v3.isnan().sum() == 2
    # the mean over elements of 0.9 * 1.0625 * 2^-4 (between two grid values 1/8 of a power of two apart): each rounding
    # is off by less than one step, so the mean of n is off by at most 5 steps / (2 sqrt n)
    opt.set_moments([torch.full((n,), 0.0625)], [torch.full((n,), 2.0 ** -10)])
    opt.step(9, 0.0, [torch.zeros(n, device="cuda")])
    m4, v4 = (x[0].double() for x in opt.moments())
    for got, want in ((m4, 0.9 * 0.0625), (v4, 0.999 * 2.0 ** -10)):
        step = 2.0 ** (math.floor(math.log2(want)) - 3)
        assert len(set(got.tolist())) == 2 and abs(got.mean().item() - want) < 5 * step / (2 * math.sqrt(n))


def test_none_gradients_and_p_grad(cuda_device):
    p = [torch.nn.Parameter(torch.ones(300, device="cuda")), torch.nn.Parameter(torch.ones(40, 5, device="cuda"))]
    opt = AdamW(p, weight_decay=0.0)
    p[0].grad = torch.full((300,), 0.1, device="cuda")
    opt.step(1, 0.1)
    assert (p[1] == 1).all() and (opt.moments()[0][1] == 0).all()
    want = 1 - 0.1 * 0.1 / (0.1 + 1e-8)
    assert (p[0] - want).abs().max() < 1e-6 and opt.moments()[0][1].shape == (40, 5)


def test_nothing_to_do(cuda_device):
    opt = AdamW([torch.zeros(0, device="cuda"), torch.zeros(0, 3, device="cuda")], state_bits=8)
    opt.step(1, 0.1, [torch.zeros(0, device="cuda"), None])
    assert opt.moments()[0][1].shape == (0, 3) and opt.state.numel() == 0
    p = torch.ones(5, device="cuda")
    AdamW([p]).step(1, 0.1, [None])
    assert (p == 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_two_plans_on_two_streams(bits, cuda_device):
    sizes = [70001, 300]
    sets = [tensors(sizes, "f32", s, 0.5) for s in (1, 2, 1, 2)]
    grads = [tensors(sizes, "f32", s, 0.1) for s in (3, 4, 3, 4)]
    for p, g in zip(sets[:2], grads[:2]):
        opt = AdamW(p, state_bits=bits)
        for it in (1, 2, 3):
            opt.step(it, 0.01, g)
    opts = [AdamW(p, state_bits=bits) for p in sets[2:]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in opts]
    for it in (1, 2, 3):
        for st, opt, g in zip(streams, opts, grads[2:]):
            with torch.cuda.stream(st):
                opt.step(it, 0.01, g)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(sets[:2], sets[2:]) for a, b in zip(x, y))


def test_many_tensors_of_mixed_types(cuda_device):
    """More tensors than one launch's arguments hold, with several types in one call."""
    sizes = [(i * 37) % 600 for i in range(4100)]
    kinds = ["f32", "bf16", "f16"]
    flat = [tensors([n], kinds[i % 3], i, 0.5)[0] for i, n in enumerate(sizes)]
    g = [torch.full((n,), 0.01 * (1 + i % 5), dtype=flat[i].dtype, device="cuda") for i, n in enumerate(sizes)]
    before = [f64(t) for t in flat]
    opt = AdamW(flat, weight_decay=0.0, eps=0.0)
    opt.step(1, 0.125, g)
    for i, n in enumerate(sizes):   # the first step moves by lr, whatever the gradient
        eps = torch.finfo(flat[i].dtype).eps
        want = before[i] - 0.125
        assert (np.abs(f64(flat[i]) - want) <= 2.0 ** -20 + eps / 2 * np.abs(want)).all(), i


@pytest.mark.parametrize("bits", [32, 8])
def test_device_scalars_graph_and_checkpoint(bits, cuda_device):
    sizes = [1000, 257, 3]
    a, b = tensors(sizes, "f32", 1, 0.5), tensors(sizes, "f32", 1, 0.5)
    g = tensors(sizes, "f32", 2, 0.1)
    eager, graphed = AdamW(a, state_bits=bits, seed=5), AdamW(b, state_bits=bits, seed=5)
    it = torch.zeros(1, dtype=torch.int64, device="cuda")
    lr = torch.tensor([0.01], device="cuda")
    scale = torch.tensor([0.5], device="cuda")
    with pytest.raises(RuntimeError, match="from the device"):
        dead = torch.cuda.CUDAGraph()
        with torch.cuda.graph(dead):
            it.add_(0)
            graphed.step(1, 0.01, g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        it.add_(1)
        graphed.step(it, lr, g, grad_scale=scale)
    for k in (1, 2, 3):
        if k == 2:
            saved = {kk: (vv.clone() if isinstance(vv, torch.Tensor) else vv) for kk, vv in eager.state_dict().items()}
            saved_p = [t.clone() for t in a]
        lr.fill_(0.01 * k)
        graph.replay()
        eager.step(k, float(np.float32(0.01 * k)), g, grad_scale=0.5)
        torch.cuda.synchronize()
        assert torch.equal(eager.state, graphed.state)
        for x, y in zip(a, b):   # the step sizes may differ in their last 32-bit place
            assert ((x - y).abs() <= 2 * U * x.abs() + 4 * U * 0.1).all()
    final = [t.clone() for t in a]
    again = AdamW(a, state_bits=bits, seed=5)
    again.load_state_dict(saved)
    for t, s in zip(a, saved_p):
        t.copy_(s)
    for k in (2, 3):
        again.step(k, float(np.float32(0.01 * k)), g, grad_scale=0.5)
    assert all(torch.equal(x, y) for x, y in zip(a, final)) and torch.equal(again.state, eager.state)
    with pytest.raises(ValueError, match="layout"):
        AdamW(a[:2], state_bits=bits).load_state_dict(saved)


def test_refusals(cuda_device):
    p = tensors([100, 50], "f32", 1, 1.0)
    opt = AdamW(p)
    g = tensors([100, 50], "f32", 2, 1.0)
    for bad in (lambda: opt.step(1, 0.1, g[:1]), lambda: opt.step(1, 0.1, [g[0], g[0]]), lambda: opt.step(1, 0.1, [g[0].half(), g[1]]),
                lambda: opt.step(1, 0.1, [g[0], g[1].cpu()]), lambda: opt.step(torch.tensor([1]), 0.1, g),
                lambda: opt.step(torch.tensor([1.0], device="cuda"), 0.1, g), lambda: AdamW([p[0], p[0]]), lambda: AdamW([p[0], p[0][50:]]),
                lambda: AdamW([torch.zeros(8, 8, device="cuda").t()]), lambda: opt.set_moments(g, g[:1])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: opt.step(0, 0.1, g), lambda: opt.step(1, -0.1, g), lambda: opt.step(1, math.nan, g), lambda: opt.step(1 << 32, 0.1, g)):
        with pytest.raises(RuntimeError):
            bad()
    opt.close()
    with pytest.raises(RuntimeError, match="closed"):
        opt.step(1, 0.1, g)


def test_gradients_that_are_not_numbers_stay_in_place(cuda_device):
    for bits in (32, 8):
        p = [torch.ones(600, device="cuda")]
        opt = AdamW(p, state_bits=bits)
        g = torch.full((600,), 0.1, device="cuda")
        g[300], g[301] = math.nan, math.inf
        opt.step(1, 0.01, [g])
        bad = torch.zeros(600, dtype=torch.bool, device="cuda")
        bad[300:302] = True
        assert torch.equal(p[0].isnan(), bad)
        m, v = (x[0] for x in opt.moments())
        assert torch.equal(~m.isfinite(), bad) and torch.equal(~v.isfinite(), bad)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_symbol_model_is_trained(bits, cuda_device):
    """The operators as they are used together: a table of logits per context rates palette indices, the gradient of the
    mean code length flows back into the table, AdamW moves it. The first step's gradient is checked against the
    formula and the first update moves every touched logit by the learning rate."""
    gen = torch.Generator().manual_seed(0)
    contexts, v, n = 16, 4, 6000
    ctx = torch.randint(0, contexts, (n,), generator=gen).cuda()
    sym = (torch.randint(0, 2, (n,), generator=gen) * 2 + (torch.arange(n) % 2)).to(torch.uint8).cuda()
    table = torch.zeros(contexts, v, device="cuda")
    opt = AdamW([table], state_bits=bits, weight_decay=0.0)
    for it in range(1, 4):
        logits = table[ctx]
        r = symbol_logprobs(logits, sym, topk=2)
        d = symbol_logprobs_grad(logits, sym, r.lse, r.entropy, -1.0 / n)
        grad = torch.zeros_like(table).index_add_(0, ctx, d)
        if it == 1:
            assert (r.logp + math.log(v)).abs().max() < 1e-6
            count = torch.zeros(contexts, v, dtype=torch.float64, device="cuda").index_put_((ctx, sym.long()), torch.ones((), dtype=torch.float64, device="cuda"), accumulate=True)
            want = (count.sum(1, keepdim=True) / v - count) / n
            assert (grad.double() - want).abs().max() < 1e-5 * want.abs().max() + 600 * U / n
        opt.step(it, 0.05, [grad])
        if it == 1:
            moved = want.abs() > 1e-5
            assert (table + 0.05 * want.sign())[moved].abs().max() < 0.05 * 1e-2   # eps = 1e-8 over |g| > 1e-5: 0.1 %


def test_negated_views_are_refused(cuda_device):
    """Their memory holds the values' negatives: as a parameter, a gradient or a scalar they would act with the wrong sign."""
    one = torch.randn(1, dtype=torch.complex64, device="cuda").conj().imag
    assert one.is_neg() and one.is_contiguous()
    with pytest.raises(ValueError, match="negated"):
        AdamW([one])
    p = torch.ones(1, device="cuda")
    opt = AdamW([p])
    for bad in (lambda: opt.step(1, 0.1, [one]), lambda: opt.step(1, one, [p.clone()]), lambda: opt.step(1, 0.1, [p.clone()], grad_scale=one)):
        with pytest.raises(ValueError):
            bad()
    assert p.item() == 1.0


@pytest.mark.parametrize("bits", [32, 8])
def test_smallest_eps(bits, cuda_device):
    """The smallest eps that is taken leaves a parameter without a gradient where it was; a smaller one is refused, by the
    step too."""
    p = torch.ones(300, device="cuda")
    opt = AdamW([p], state_bits=bits, eps=2.0 ** -126, weight_decay=0.0)
    g = torch.zeros(300, device="cuda")
    opt.step(1, 0.1, [g])
    assert (p == 1).all()
    g[0] = 1.0
    opt.step(2, 0.1, [g])
    assert p[0] < 1 and (p[1:] == 1).all()
    opt.eps = 1e-40
    with pytest.raises(RuntimeError, match="eps"):
        opt.step(3, 0.1, [g])


@pytest.mark.parametrize("bits", [32, 8])
def test_first_step_on_another_stream_at_once(bits, cuda_device):
    """The plan's table is on the device when the plan is made: a stream that does not wait for the legacy one takes the
    first step without a synchronisation in between (it waits for the tensors only)."""
    for n in (300, 5_000_000):
        p = torch.ones(n, device="cuda")
        g = torch.full((n,), 0.5, device="cuda")
        for _ in range(20):
            stream = torch.cuda.Stream()
            opt = AdamW([p], state_bits=bits, weight_decay=0.0)
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                p.fill_(1.0)
                opt.step(1, 0.25, [g])
                assert ((p - 0.75).abs() < 1e-5).all()
            torch.cuda.current_stream().wait_stream(stream)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_outlives_the_optimiser(bits, cuda_device):
    """A captured step goes on working after the object that made it was collected: its plan and its state stay."""
    import gc
    import weakref
    sizes = [70001, 300, 5]
    a, b, g = tensors(sizes, "f32", 1, 0.5), tensors(sizes, "f32", 1, 0.5), tensors(sizes, "f32", 2, 0.1)
    it, lr = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.tensor([0.01], device="cuda")
    opt = AdamW(a, state_bits=bits, seed=3)
    never = AdamW(a[1:2], state_bits=bits)
    assert not opt.lib.ntcb_adamw_captured(opt.h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        it.add_(1)
        opt.step(it, lr, g)
        m, v = opt.moments_flat()
    assert opt.lib.ntcb_adamw_captured(opt.h) and not never.lib.ntcb_adamw_captured(never.h)
    gone = weakref.ref(opt)
    del opt, never
    gc.collect()
    assert gone() is None
    torch.cuda.empty_cache()
    other = [torch.full((1 << k,), 7, dtype=torch.uint8, device="cuda") for k in range(8, 22)]   # takes what was given back
    eager = AdamW(b, state_bits=bits, seed=3)
    for k in (1, 2, 3):
        graph.replay()
        eager.step(k, float(np.float32(0.01)), g)
    torch.cuda.synchronize()
    for x, y in zip(a, b):
        assert ((x - y).abs() <= 3 * (2 * U * y.abs() + 4 * U * 0.1)).all()
    assert all(torch.equal(x, y) for x, y in zip((m, v), eager.moments_flat()))
    assert all((o == 7).all() for o in other)


def test_device_scalars_off_their_alignment(cuda_device):
    """Refused by the C entry before anything is launched."""
    import ctypes as C

    from neural_block_textures_b200 import abi
    p, g = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    opt = AdamW([p])
    spare = torch.zeros(4, dtype=torch.int64, device="cuda").data_ptr()
    why = C.create_string_buffer(256)
    for name, off in (("it_dev", 4), ("lr_dev", 2), ("grad_scale_dev", 1)):
        args = abi.AdamWArgs(lr=0.1, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, grad_scale=1.0, it=1, seed=0)
        setattr(args, name, spare + off)
        ok = opt.lib.ntcb_adamw_step(opt.h, (C.c_void_p * 1)(p.data_ptr()), (C.c_void_p * 1)(g.data_ptr()), opt.state.data_ptr(),
                                     C.addressof(args), None, why, 256)
        assert ok == 0 and b"aligned" in why.value
    assert (p == 1).all()


def test_steps_are_seen_by_backward_passes(cuda_device):
    """A step raises the version of the parameters that it wrote: values saved before it are not used with the new ones."""
    p = [torch.nn.Parameter(torch.ones(40, device="cuda")), torch.nn.Parameter(torch.ones(5, device="cuda"))]
    opt = AdamW(p)
    before = [x._version for x in p]
    loss = (p[0] * p[0]).sum()
    opt.step(1, 0.1, [torch.ones(40, device="cuda"), None])
    assert p[0]._version > before[0] and p[1]._version == before[1]
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    now = p[0]._version
    with pytest.raises(RuntimeError):
        opt.step(1, -0.1, [torch.ones(40, device="cuda"), None])   # refused: nothing was written
    assert p[0]._version == now
    (p[0] * p[0]).sum().backward()
    assert torch.equal(p[0].grad, 2 * p[0].detach())
    with torch.inference_mode():
        q = torch.ones(6, device="cuda")
    AdamW([q]).step(1, 0.1, [torch.ones(6, device="cuda")])   # has no version
    assert (q < 1).all()
