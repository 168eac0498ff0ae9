"""The operators for learned symbol models, as cases to be measured: log probabilities of given symbols (with entropy
and top alternatives) and their gradient, and the AdamW step over many tensors with 32-bit or 8-bit states.

`listed()` names the cases, `draw()` makes more of the same ranges, `prepare()` makes a case's inputs from a seed,
`run()` makes one pass over them: in elementary torch operations where `own` is false, with this package's entry points
where it is true. `exact()` gives the definition in 64 bits, `work()` the bytes and operations of a pass."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SYMBOLS = {"u8": torch.uint8, "i16": torch.int16, "i32": torch.int32, "i64": torch.int64}
LOWEST = torch.finfo(torch.float32).min
BETAS, EPS, DECAY, LR, SCALE, STEP = (0.9, 0.999), 1e-8, 0.01, 2e-3, 0.5, 7
BLOCK = 256            # elements that share the window of their 8-bit states
TOP_M, TOP_V = 126, 254   # the highest finite code of a first / second moment


# --------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # 2-bit palette indices of a full 1024 x 1024 level 0 (the largest benchmark configuration), every cell rated
        # under a predictor's 4 logits, with the best other index beside it (the choice a rate-aware search weighs)
        {"name": "palette_rate", "op": "logprobs", "rows": 1 << 20, "vocab": 4, "stride": 4, "dtype": "f32", "symbol": "u8", "topk": 2},
        # 8-bit grid indices of a 256 x 256 x 4 second level under 256 logits, with the eight likeliest
        {"name": "grid8_rate", "op": "logprobs", "rows": 1 << 18, "vocab": 256, "stride": 256, "dtype": "bf16", "symbol": "i32", "topk": 8},
        # the deepest post-hoc grid (16 bits), one texture tile's indices, no alternatives wanted
        {"name": "grid16_rate", "op": "logprobs", "rows": 2048, "vocab": 65536, "stride": 65536, "dtype": "bf16", "symbol": "i32", "topk": 0},
        # one symbol at a time, as a decoder or a search asks for it: latency counts
        {"name": "grid16_one", "op": "logprobs", "rows": 1, "vocab": 65536, "stride": 65536, "dtype": "f32", "symbol": "i64", "topk": 20},
        # an odd token alphabet inside wider rows (run / level tokens of a DCT level), every alternative asked for
        {"name": "tokens_odd", "op": "logprobs", "rows": 1501, "vocab": 4099, "stride": 4131, "dtype": "f16", "symbol": "i16", "topk": 32},
        # the gradients of the same three shapes of rate loss
        {"name": "palette_grad", "op": "logprobs_grad", "rows": 1 << 20, "vocab": 4, "stride": 4, "dtype": "f32", "symbol": "u8", "entropy": False},
        {"name": "grid8_grad", "op": "logprobs_grad", "rows": 1 << 18, "vocab": 256, "stride": 256, "dtype": "bf16", "symbol": "i32", "entropy": True},
        {"name": "tokens_odd_grad", "op": "logprobs_grad", "rows": 4001, "vocab": 16411, "stride": 16411, "dtype": "f32", "symbol": "i64", "entropy": True},
        # one small texture model (a 64 x 64 x 4 level and six layer tensors): latency
        {"name": "adamw32_one", "op": "adamw", "bits": 32, "models": 1, "level0": 64 * 64 * 4, "level1": 0, "param": "f32", "grad": "f32", "shift": 0},
        # 64 models of the largest benchmark configuration trained together, states in 32 bits and in 8
        {"name": "adamw32_many", "op": "adamw", "bits": 32, "models": 64, "level0": 1024 * 1024 * 2, "level1": 256 * 256 * 4, "param": "f32", "grad": "f32", "shift": 0},
        {"name": "adamw8_many", "op": "adamw", "bits": 8, "models": 64, "level0": 1024 * 1024 * 2, "level1": 256 * 256 * 4, "param": "f32", "grad": "f32", "shift": 0},
        # models of ragged sizes held in bf16 (35 x 29 level sizes and the like, none a multiple of a block)
        {"name": "adamw8_ragged", "op": "adamw", "bits": 8, "models": 37, "level0": 263 * 257 * 5, "level1": 67 * 71 * 3, "param": "bf16", "grad": "bf16", "shift": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs_grad", "adamw", "adamw"])
    if op == "adamw":
        level0 = _log(rng, 300, 3 << 19)
        models = max(1, min(64, _log(rng, 1, 64)))
        return {"op": op, "bits": rng.choice([8, 32]), "models": models, "level0": level0, "level1": _log(rng, 1, 1 + level0 // 4),
                "param": rng.choice(["f32", "f32", "bf16", "f16"]), "grad": rng.choice(["f32", "bf16", "f16"]),
                "shift": rng.choice([0, 0, 1])}
    vocab = rng.choice([_log(rng, 2, 65536), 1 << rng.randint(1, 16), _log(rng, 2, 65536) | 1])
    rows = max(1, min(1 << 20, _log(rng, 1, (1 << 26) // vocab)))
    case = {"op": op, "rows": rows, "vocab": vocab, "stride": vocab + rng.choice([0, 0, 1, 8, 37]),
            "dtype": rng.choice(["f32", "bf16", "f16"]), "symbol": rng.choice(["i32", "i64"] + (["i16"] if vocab <= 32768 else []))}
    if op == "logprobs":
        case["topk"] = min(vocab, rng.choice([0, 1, 2, 5, 8, 20, 32]))
    else:
        case["entropy"] = rng.random() < 0.5
    return case


def _sizes(case):
    """Element counts of the tensors: per model its levels, then weights and biases of a 24-24 MLP."""
    nin = 6 if case["level1"] == 0 else 8
    layers = [nin * 24, 24, 24 * 24, 24, 24 * 3, 3]
    out = []
    for i in range(case["models"]):
        odd = i % 7 if case["param"] != "f32" else 0   # models that are not copies of one another
        out += [case["level0"] + odd] + ([case["level1"] + odd] if case["level1"] else []) + layers
    return out


def _layout(case):
    """Where each tensor starts in a flat buffer (a multiple of a block, or `shift` elements behind one: views that no
    wide load fits), and the buffer's length."""
    starts, at = [], 0
    for n in _sizes(case):
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


def _views(flat, case, shift=0):
    return [flat[s + shift:s + shift + n] for s, n in zip(_layout(case)[0], _sizes(case))]


def work(case):
    size = 4 if case.get("dtype", "f32") == "f32" else 2
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        p = 4 if case["param"] == "f32" else 2
        g = 4 if case["grad"] == "f32" else 2
        # 32 bits: both moments read and written. 8 bits: their codes read and written, a 16-bit window per block and
        # moment, and the moments handed out as the values they stand for.
        states = 16 if case["bits"] == 32 else 4 + 8 * 2 / BLOCK + 8
        return {"bytes": n * (2 * p + g + states), "flops": n * 14}
    n, v = case["rows"], case["vocab"]
    symbol = {"u8": 1, "i16": 2, "i32": 4, "i64": 8}[case["symbol"]]
    if case["op"] == "logprobs":
        return {"bytes": n * (v * size + symbol + 12 + 8 * case["topk"]), "flops": n * v * 5}
    return {"bytes": n * (2 * v * size + symbol + 8 + (8 if case["entropy"] else 0)), "flops": n * v * (8 if case["entropy"] else 4)}


# -------------------------------------------------------------------------------------------------------- inputs

def _logits(case, gen):
    """Logits as a predictor gives them: most rows over the whole alphabet, some over a prefix (a channel of less
    depth; the rest masked with -inf, or with the lowest finite value), a few with nothing left; and symbols, some
    rows without one."""
    n, v, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    store = torch.empty(n, case["stride"], dtype=dtype, device="cuda")
    x = store[:, :v]
    per = max(1, (1 << 26) // v)
    kind = torch.rand(n, device="cuda", generator=gen)
    if n == 1:
        kind.fill_(0.5)   # the single row is an ordinary one
    valid = torch.full((n,), v, dtype=torch.int64, device="cuda")
    part = kind < 0.1
    prefix = (torch.rand(n, device="cuda", generator=gen) * v).long() + 1
    valid = torch.where(part, prefix.clamp(max=v), valid)
    valid = torch.where(kind > 0.995, torch.zeros_like(valid), valid)
    fill = torch.where(kind < 0.05, torch.full_like(kind, torch.finfo(dtype).min), torch.full_like(kind, -math.inf))
    column = torch.arange(v, device="cuda")
    for r in range(0, n, per):
        rows = slice(r, min(n, r + per))
        block = torch.randn(rows.stop - r, v, device="cuda", generator=gen) * 2.5
        x[rows] = torch.where(column < valid[rows, None], block, fill[rows, None]).to(dtype)
    symbols = (torch.rand(n, device="cuda", generator=gen) * valid.clamp(min=1)).long().clamp(max=v - 1)
    if case["symbol"] != "u8" and n > 1:
        symbols = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.02, torch.full_like(symbols, -1), symbols)
    return x, symbols.to(SYMBOLS[case["symbol"]])


def _on_grid(n, gen, scale, span, signed):
    """Moments that 8 bits hold exactly: 4 significant bits, over `span` powers of two below `scale`."""
    e = torch.randint(0, span, (n,), device="cuda", generator=gen)
    k = torch.randint(8, 16, (n,), device="cuda", generator=gen)
    x = torch.ldexp(k.float() * scale, -e)
    if signed:
        x = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.5, -x, x)
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"op": case["op"], "case": case}
    if case["op"] == "adamw":
        pd, gd = DTYPES[case["param"]], DTYPES[case["grad"]]
        total = _layout(case)[1]
        # the models live in flat buffers, as the framework's own latent and weights do
        state.update(it=STEP, seed=seed, flat=torch.zeros(total + BLOCK, dtype=pd, device="cuda"),
                     flat_grad=torch.zeros(total + BLOCK, dtype=gd, device="cuda"),
                     m=torch.zeros(total, device="cuda"), v=torch.zeros(total, device="cuda"))
        state["params"], state["grads"] = _views(state["flat"], case, case["shift"]), _views(state["flat_grad"], case, case["shift"])
        moments = list(zip(_views(state["m"], case), _views(state["v"], case)))
        for p, g, (m, v) in zip(state["params"], state["grads"], moments):
            n = p.numel()
            p.copy_(torch.randn(n, device="cuda", generator=gen) * 0.3)
            spread = torch.randint(-4, 5, (n,), device="cuda", generator=gen)
            g.copy_(torch.ldexp(torch.randn(n, device="cuda", generator=gen) * 4e-3, spread))
            m.copy_(_on_grid(n, gen, 2.0 ** -13, 12, True))
            v.copy_(_on_grid(n, gen, 2.0 ** -18, 20, False))
        if own:
            from neural_block_textures_b200 import AdamW
            opt = AdamW(state["params"], state_bits=case["bits"], betas=BETAS, eps=EPS, weight_decay=DECAY, seed=seed,
                        grad_dtype=gd)
            opt.set_moments(*zip(*moments))
            state["opt"] = opt
            del state["m"], state["v"]
        elif case["bits"] == 8:
            state["codes"] = [(_encode(m, None, TOP_M), _encode(v, None, TOP_V)) for m, v in moments]
        return state
    x, symbols = _logits(case, gen)
    state.update(logits=x, symbols=symbols)
    if case["op"] == "logprobs_grad":
        n = case["rows"]
        lse, entropy = [], []
        for rows in _row_chunks(case):   # what the forward pass left behind
            _, h, l = _rate64(x[rows], symbols[rows])
            lse.append(l.float())
            entropy.append(h.float())
        state.update(lse=torch.cat(lse), entropy=torch.cat(entropy),
                     dlogp=-(0.5 + torch.rand(n, device="cuda", generator=gen)) / n,
                     dentropy=0.1 * torch.randn(n, device="cuda", generator=gen) / n if case["entropy"] else None)
    return state


# ------------------------------------------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "logprobs":
        return _plain_logprobs(state["logits"], state["symbols"], case["topk"])
    if case["op"] == "logprobs_grad":
        return _plain_grad(state)
    return _plain_adamw(state, case)


def _run_own(state, case):
    import neural_block_textures_b200 as nbt
    if case["op"] == "logprobs":
        r = nbt.symbol_logprobs(state["logits"], state["symbols"], topk=case["topk"])
        return {"logp": r.logp, "entropy": r.entropy, "lse": r.lse, "top_ids": r.top_ids, "top_logp": r.top_logp}
    if case["op"] == "logprobs_grad":
        return nbt.symbol_logprobs_grad(state["logits"], state["symbols"], state["lse"], state["entropy"], state["dlogp"],
                                        state["dentropy"])
    opt = state["opt"]
    opt.step(state["it"], LR, state["grads"], grad_scale=SCALE)
    state["it"] += 1
    m, v = opt.moments_flat()
    return {"params": state["flat"], "m": m, "v": v}


def _plain_logprobs(logits, symbols, topk):
    x = logits.float()
    m = x.amax(1, keepdim=True).clamp(min=LOWEST)
    d = x - m
    e = d.exp()
    s = e.sum(1)
    u = torch.where(e > 0, e * d, 0.0).sum(1)
    log_s = s.log()
    some = s > 0
    lse = torch.where(some, m[:, 0] + log_s, -math.inf)
    entropy = torch.where(some, log_s - u / s, 0.0)
    t = symbols.long()
    logp = torch.where(some, d.gather(1, t.clamp(min=0)[:, None])[:, 0] - log_s, -math.inf)
    logp = torch.where(t < 0, 0.0, logp)
    ids, top = [], []
    rest = x.clone() if topk else None
    for _ in range(topk):
        i = rest.argmax(1, keepdim=True)   # the first of equal values
        val = rest.gather(1, i)[:, 0]
        ids.append(torch.where(val == -math.inf, -1, i[:, 0]).int())
        top.append(torch.where(val == -math.inf, -math.inf, val - m[:, 0] - log_s))
        rest.scatter_(1, i, -math.inf)
    n = len(logits)
    return {"logp": logp, "entropy": entropy, "lse": lse,
            "top_ids": torch.stack(ids, 1) if topk else torch.empty(n, 0, dtype=torch.int32, device="cuda"),
            "top_logp": torch.stack(top, 1) if topk else torch.empty(n, 0, device="cuda")}


def _plain_grad(state):
    x, t, lse = state["logits"].float(), state["symbols"].long(), state["lse"][:, None]
    some = lse > -math.inf
    logp = x - lse.clamp(min=LOWEST)
    p = logp.exp()
    dlogp = torch.where(t < 0, 0.0, state["dlogp"])[:, None]
    dx = -dlogp * p
    if state["dentropy"] is not None:
        dx = dx - torch.where(p > 0, state["dentropy"][:, None] * p * (logp + state["entropy"][:, None]), 0.0)
    dx.scatter_add_(1, t.clamp(min=0)[:, None], dlogp)
    return torch.where(some, dx, 0.0).to(state["logits"].dtype)


MASK64 = (1 << 64) - 1
GOLDEN = 0x9E3779B97F4A7C15


def _mix_int(x):
    x = (x + GOLDEN) & MASK64
    x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & MASK64
    x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & MASK64
    return x ^ (x >> 31)


def _signed(x):
    x &= MASK64
    return x - (1 << 64) if x >> 63 else x


def _shift(x, n):
    return (x >> n) & ((1 << (64 - n)) - 1)   # a logical shift of signed 64-bit words


def _noise(seed, it, tensor, n):
    """The counter noise of one tensor at one step: 16 bits for each element's first moment and 16 for its second; two
    neighbours share a 64-bit draw."""
    key = _mix_int((seed & MASK64) ^ (5 << 56) ^ ((it & 0xFFFFFFFF) << 32) ^ tensor)
    x = torch.arange((n + 1) // 2, device="cuda", dtype=torch.int64) * _signed(GOLDEN) + _signed(key + GOLDEN)
    x = (x ^ _shift(x, 30)) * _signed(0xBF58476D1CE4E5B9)
    x = (x ^ _shift(x, 27)) * _signed(0x94D049BB133111EB)
    x = x ^ _shift(x, 31)
    words = torch.stack([x & 0xFFFF, _shift(x, 16) & 0xFFFF, _shift(x, 32) & 0xFFFF, _shift(x, 48)], 1).view(-1, 2)[:n]
    return words[:, 0].int(), words[:, 1].int()


def _encode(x, noise, top):
    """Values to 8-bit codes: the float's exponent and 3 mantissa bits, rounded by `noise` (16 bits above the bits that
    are dropped; None: to nearest), as a distance above the lowest value of the block's window. First moments
    (top 126) carry the sign in bit 7; a second moment above zero keeps at least the lowest code."""
    n = x.numel()
    finite = x.isfinite()
    bits = torch.where(finite, x, 0.0).abs().view(torch.int32)
    q = (bits + (noise << 4 if noise is not None else 1 << 19)) >> 20
    q = torch.where(finite & (bits > 0), q, 0)
    pad = -n % BLOCK
    blocks = torch.nn.functional.pad(q, (0, pad)).view(-1, BLOCK)
    base = (blocks.amax(1) - top).clamp(min=0)
    code = (blocks - base[:, None]).clamp(min=0).view(-1)[:n]
    if top == TOP_V:
        code = torch.where(bits > 0, code.clamp(min=1), code)
    code = torch.where(finite, code, top + 1)
    if top == TOP_M:
        code = code | ((x < 0) & (code > 0)).int() << 7
    return code.to(torch.uint8), base.to(torch.int16)


def _decode(state, top):
    code, base = state[0].int(), state[1].int()
    n = code.numel()
    mag = code & 0x7F if top == TOP_M else code
    q = mag + base.repeat_interleave(BLOCK)[:n]
    x = torch.where(mag > 0, q << 20, 0).view(torch.float32)
    x = torch.where(mag == top + 1, math.nan, x)
    return torch.where(code > 127, -x, x) if top == TOP_M else x


def _plain_adamw(state, case):
    b1, b2 = BETAS
    it = state["it"]
    state["it"] += 1
    step = LR / (1 - b1 ** it)
    inv = 1 / math.sqrt(1 - b2 ** it)
    flat_m, flat_v = state["m"], state["v"]
    moments = list(zip(_views(flat_m, case), _views(flat_v, case)))
    for i, (p, g, (m, v)) in enumerate(zip(state["params"], state["grads"], moments)):
        m0, v0 = m, v
        if case["bits"] == 8:
            m0, v0 = _decode(state["codes"][i][0], TOP_M), _decode(state["codes"][i][1], TOP_V)
        g = g.float() * SCALE
        m1 = m0 * b1 + g * (1 - b1)
        v1 = v0 * b2 + (g * g) * (1 - b2)
        p.copy_(p.float() * (1 - LR * DECAY) - step * m1 / (v1.sqrt() * inv + EPS))
        if case["bits"] == 8:
            rm, rv = _noise(state["seed"], it, i, p.numel())
            state["codes"][i] = _encode(m1, rm, TOP_M), _encode(v1, rv, TOP_V)
            m1, v1 = _decode(state["codes"][i][0], TOP_M), _decode(state["codes"][i][1], TOP_V)
        m.copy_(m1)
        v.copy_(v1)
    return {"params": state["flat"], "m": flat_m, "v": flat_v}


# ------------------------------------------------------------------------------------------------- the definition

def _row_chunks(case):
    per = max(1, (1 << 25) // case["vocab"])
    return [slice(r, min(case["rows"], r + per)) for r in range(0, case["rows"], per)]


def _rate64(x, symbols):
    """(logp, entropy, log-sum-exp) of some rows in 64 bits."""
    x = x.double()
    lse = torch.logsumexp(x, 1)
    empty = torch.isneginf(lse)
    lp = x - torch.where(empty, 0.0, lse)[:, None]
    entropy = -torch.nan_to_num(lp.exp() * lp, nan=0.0, posinf=0.0, neginf=0.0).sum(1)
    t = symbols.long()
    logp = lp.gather(1, t.clamp(min=0)[:, None])[:, 0]
    return torch.where(t < 0, 0.0, logp), entropy, lse


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "adamw":
        return _exact_adamw(state, case)
    x, symbols = state["logits"], state["symbols"]
    if case["op"] == "logprobs_grad":
        return torch.cat([_exact_grad(state, rows) for rows in _row_chunks(case)])
    out = {"logp": [], "entropy": [], "lse": [], "top_ids": [], "top_logp": []}
    for rows in _row_chunks(case):
        logp, entropy, lse = _rate64(x[rows], symbols[rows])
        value, index = x[rows].double(), torch.arange(case["vocab"], device="cuda").expand(len(lse), -1)
        if case["topk"]:
            value, index = value.sort(dim=1, descending=True, stable=True)
        value, index = value[:, :case["topk"]], index[:, :case["topk"]]
        gone = torch.isneginf(value)
        out["top_ids"].append(index.masked_fill(gone, -1).int())
        out["top_logp"].append((value - lse[:, None]).masked_fill(gone, -math.inf))
        for name, part in (("logp", logp), ("entropy", entropy), ("lse", lse)):
            out[name].append(part)
    return {name: torch.cat(parts) for name, parts in out.items()}


def _exact_grad(state, rows):
    x, t = state["logits"][rows].double(), state["symbols"][rows].long()
    logp, entropy, lse = _rate64(state["logits"][rows], t)
    empty = torch.isneginf(lse)
    lp = x - torch.where(empty, 0.0, lse)[:, None]
    p = lp.exp()
    one = torch.zeros_like(x)
    has = (t >= 0) & ~empty
    one[has.nonzero()[:, 0], t[has]] = 1.0
    dx = state["dlogp"][rows].double()[:, None] * (one - p) * has[:, None]
    if state["dentropy"] is not None:
        slope = -torch.nan_to_num(p * (lp + entropy[:, None]), nan=0.0, posinf=0.0, neginf=0.0)
        dx = dx + state["dentropy"][rows].double()[:, None] * slope
    return dx.masked_fill(empty[:, None], 0.0)


def _exact_adamw(state, case):
    b1, b2 = BETAS
    params, m, v = state["flat"].double(), state["m"].double(), state["v"].double()   # the starting moments: exact in 8 bits
    views = zip(_views(params, case, case["shift"]), state["grads"], _views(m, case), _views(v, case))
    for p, g, m1, v1 in views:
        g = g.double() * SCALE
        m1.mul_(b1).add_((1 - b1) * g)
        v1.mul_(b2).add_((1 - b2) * g ** 2)
        mh, vh = m1 / (1 - b1 ** STEP), v1 / (1 - b2 ** STEP)
        p.sub_(LR * DECAY * p + LR * mh / (vh.sqrt() + EPS))
    if case["bits"] == 8:   # stochastically rounded: no such value
        m = v = None
    return {"params": params, "m": m, "v": v}
