"""MXFP4 experts and the adapters' AdamW step, for timing and for checking.

Each case is a dict of plain values. ``listed()`` holds the standing ones,
``draw(rng)`` makes more of the same ranges, ``prepare`` builds what a program
holds before the call, ``run`` is one pass (in plain torch operations, or with
``own`` through the package's public entry points), ``work`` its bytes and
floating-point operations, and ``exact`` the same result in 64 bits.

Kinds of case (``kind``):
  codec   a tensor quantised to MXFP4 (blocks of 32 along the last axis, one
          power-of-two scale each) and read back
  linear  one projection of expert-sorted rows over frozen MXFP4 weights,
          16-bit activations; ``train`` adds the gradient of the rows
  linear4 the same with the rows quantised to MXFP4 as well, so that both
          operands of the product are 4-bit
  adamw   one AdamW step over every adapter factor of a model, moments in 32
          bits or in 8 (blocks of 128, stochastic rounding from a seed)
"""

from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 32      # elements under one MXFP4 scale
STATE_BLOCK = 128  # elements under one exponent of the 8-bit moments
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# Expert geometries: (hidden, ffn, experts).
GEOMETRIES = {"small": (512, 1024, 8), "balanced": (2048, 1408, 64), "many": (2048, 768, 128),
              "heads": (256, 512, 256)}
ADAMW = {"lr": 2e-4, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}
ADAMW_STEP = 37  # steps taken before the measured one
MAX_PRODUCT = 131072 * 2048 * 1408  # rows * in * out of the largest listed product
MAX_STEP = 260_000_000              # elements of the largest listed step


def _codec(lead, cols, dtype):
    return {"kind": "codec", "lead": int(lead), "cols": int(cols), "dtype": dtype}


def _linear(kind, rows, in_f, out_f, experts, zipf=0.0, dtype="bf16", train=False):
    return {"kind": kind, "rows": int(rows), "in": int(in_f), "out": int(out_f),
            "experts": int(experts), "zipf": float(zipf), "dtype": dtype, "train": bool(train)}


def _adamw(geometry, layers, rank, bits, dtype="fp32"):
    return {"kind": "adamw", "geometry": geometry, "layers": int(layers), "rank": int(rank),
            "bits": int(bits), "dtype": dtype}


def listed():
    cases = [
        # Activations of a few tokens: launches and latency.
        ("codec_T16", _codec(16, 2048, "bf16")),
        # An expert projection as it is loaded: 64 experts of 1408 x 2048.
        ("codec_experts", _codec(64 * 1408, 2048, "bf16")),
        # fp32 rows whose length is no multiple of the block.
        ("codec_ragged_fp32", _codec(8191, 1000, "fp32")),
        # 16 tokens, 4 experts each: weights are streamed for a row or two.
        ("linear_rows64", _linear("linear", 64, 2048, 1408, 64)),
        # An ordinary batch with skewed routes, the down projection.
        ("linear_zipf_rows16380", _linear("linear", 16380, 768, 2048, 128, zipf=1.2)),
        # Adapter training: output and the rows' gradient.
        ("linear_train_rows32768", _linear("linear", 32768, 2048, 1408, 64, train=True)),
        # Both operands in 4 bits: a few tokens.
        ("linear4_rows64", _linear("linear4", 64, 2048, 1408, 64)),
        # fp32 rows, an odd count, skewed routes.
        ("linear4_fp32_rows8191", _linear("linear4", 8191, 1408, 2048, 64, zipf=1.2, dtype="fp32")),
        # The largest: a long clip of 32768 tokens, 4 experts each.
        ("linear4_rows131072", _linear("linear4", 131072, 2048, 1408, 64)),
        # One small layer's adapters: 6 tensors, latency counts.
        ("adamw32_small", _adamw("small", 1, 8, 32)),
        # The adapters of a 24-layer model at rank 16: 144 tensors, 255 M values.
        ("adamw32_layers24", _adamw("balanced", 24, 16, 32)),
        # The same model with 8-bit moments.
        ("adamw8_layers24", _adamw("balanced", 24, 16, 8)),
    ]
    return [{"name": name, **case} for name, case in cases]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choices(("codec", "linear", "linear4", "adamw"), weights=(2, 3, 3, 2))[0]
    if kind == "codec":
        cols = _log_uniform(rng, 1, 8192)
        lead = _log_uniform(rng, 1, max(1, 180_000_000 // cols))
        return _codec(min(lead, 4_000_000), cols, rng.choice(("bf16", "fp32")))
    if kind == "adamw":
        geometry = rng.choice(tuple(GEOMETRIES))
        layers, rank = _log_uniform(rng, 1, 24), rng.choice((1, 4, 8, 16, 24, 64))
        bits = rng.choice((8, 32))
        dtype = rng.choice(("fp32", "fp32", "bf16"))
        per_layer = sum(math.prod(s) for s in _shapes(geometry, 1, rank))
        return _adamw(geometry, max(1, min(layers, MAX_STEP // per_layer)), rank, bits, dtype)
    experts = rng.choice((1, 8, 64, 128, 256))
    in_f = 64 * _log_uniform(rng, 1, 64)
    out_f = 64 * _log_uniform(rng, 1, 64)
    while experts > 1 and experts * in_f * out_f > 400_000_000:
        experts //= 2
    rows = _log_uniform(rng, 1, min(131072, MAX_PRODUCT // (in_f * out_f)))
    zipf = rng.choice((0.0, 1.2))
    dtype = rng.choice(("bf16", "bf16", "fp32")) if kind == "linear4" else "bf16"
    train = kind == "linear" and rng.random() < 0.4
    if train:
        rows = max(1, min(rows, 32768))
    return _linear(kind, rows, in_f, out_f, experts, zipf, dtype, train)


# ------------------------------------------------------------------ inputs
def _gen(seed, stream):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + stream)


def _randn(shape, seed, stream, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=_gen(seed, stream), device="cuda") * std).to(dtype)


def _counts(case):
    """Rows per expert: a function of the case. Skewed routes leave experts empty."""
    rows, experts = case["rows"], case["experts"]
    rng = random.Random(7919 * rows + experts)
    order = list(range(experts))
    rng.shuffle(order)
    weight = [0.0] * experts
    for rank, e in enumerate(order):
        weight[e] = (rank + 1.0) ** -case["zipf"] * (1.0 + 0.2 * rng.random())
    if case["zipf"] > 0 and experts > 4:
        for e in order[-(experts // 8):]:
            weight[e] = 0.0
    total = sum(weight)
    counts, left = [0] * experts, rows
    for e in range(experts):
        counts[e] = int(rows * weight[e] / total)
        left -= counts[e]
    live = [e for e in order if weight[e] > 0]
    for i in range(left):
        counts[live[i % len(live)]] += 1
    return counts


def _ends(counts):
    ends, at = [], 0
    for c in counts:
        at += c
        ends.append(at)
    return ends


def _rows(case, seed):
    """Activations: normal rows with a few outlying columns, as hidden states have."""
    x = _randn((case["rows"], case["in"]), seed, 2)
    loud = torch.randperm(case["in"], generator=_gen(seed, 3), device="cuda")[:max(1, case["in"] // 256)]
    x[:, loud] *= 12.0
    return x.to(DTYPES[case["dtype"]])


def _weight(case, seed):
    return _randn((case["experts"], case["out"], case["in"]), seed, 1, torch.bfloat16, 0.02)


def _codec_input(case, seed):
    x = _randn((case["lead"], case["cols"]), seed, 1)
    # Rows of different magnitudes, and a run of zeros.
    x *= torch.exp2(torch.randint(-20, 12, (case["lead"], 1), generator=_gen(seed, 2),
                                  device="cuda").float())
    x[:, :max(1, case["cols"] // 16)] *= (torch.arange(case["lead"], device="cuda") % 5 > 0)[:, None]
    return x.to(DTYPES[case["dtype"]])


def _shapes(geometry, layers, rank):
    d, f, experts = GEOMETRIES[geometry]
    out = []
    for _ in range(layers):
        for in_f, out_f in ((d, f), (d, f), (f, d)):
            out += [(experts, rank, in_f), (experts, out_f, rank)]
    return out


def _layout(case):
    """(offset, shape) of every factor in a flat buffer, each from a multiple of
    128 on, and the buffer's length."""
    spans, at = [], 0
    for shape in _shapes(case["geometry"], case["layers"], case["rank"]):
        spans.append((at, shape))
        at += -(-math.prod(shape) // STATE_BLOCK) * STATE_BLOCK
    return spans, at


def _step_inputs(case, seed):
    """Factors, their gradients, and moments of a run under way, as flat buffers."""
    dtype = DTYPES[case["dtype"]]
    spans, total = _layout(case)
    p, g, m, v = (_randn((total,), seed, i) for i in range(1, 5))
    for i, (at, shape) in enumerate(spans):
        end, scale = at + math.prod(shape), 1e-3 * 4.0 ** (i % 5)
        p[at:end] *= 0.02
        g[at:end] *= scale
        m[at:end] *= 0.3 * scale
        v[at:end] *= scale
        after = spans[i + 1][0] if i + 1 < len(spans) else total
        for t in (p, g, m, v):
            t[end:after] = 0
    return p.to(dtype), g.to(dtype), m, v.square_()


def _views(flat, spans):
    return [flat[at:at + math.prod(shape)].view(shape) for at, shape in spans]


def prepare(case, seed):
    kind = case["kind"]
    if kind == "codec":
        return {"case": case, "x": _codec_input(case, seed)}
    if kind == "adamw":
        p, g, m, v = _step_inputs(case, seed)
        if case["bits"] == 8:
            m, v = _moment_encode(m, 4, True), _moment_encode(v, 5, False)
        if not own:
            return {"case": case, "p": p, "g": g, "m": m, "v": v, "step": ADAMW_STEP}
        from mirai_amd import AdapterAdamW

        spans, _ = _layout(case)
        leaves = [torch.nn.Parameter(t) for t in _views(p, spans)]
        for leaf, t in zip(leaves, _views(g, spans)):
            leaf.grad = t
        opt = AdapterAdamW(leaves, **ADAMW, state_bits=case["bits"], seed=1234)
        names = {32: ("exp_avg", "exp_avg_sq"),
                 8: ("exp_avg_q", "exp_avg_sq_q", "exp_avg_e", "exp_avg_sq_e")}[case["bits"]]
        flats = (m, v) if case["bits"] == 32 else (m[0], v[0], m[1], v[1])
        saved = opt.state_dict()
        for i, (at, shape) in enumerate(spans):
            n, blk = math.prod(shape), -(-math.prod(shape) // STATE_BLOCK)
            cut = [t[at:at + n] if t.numel() == p.numel() else
                   t[at // STATE_BLOCK:at // STATE_BLOCK + blk] for t in flats]
            saved["state"][i] = {"step": ADAMW_STEP,
                                 **{k: t if k[-2:] == "_e" else t.view(shape)
                                    for k, t in zip(names, cut)}}
        opt.load_state_dict(saved)
        return {"case": case, "opt": opt, "p": p}
    x, w = _rows(case, seed), _weight(case, seed)
    ends = _ends(_counts(case))
    state = {"case": case, "x": x, "ends": ends,
             "offsets": torch.tensor(ends, dtype=torch.int32, device="cuda")}
    if case["train"]:
        state["x"] = x.requires_grad_(True)
        state["dy"] = _randn((case["rows"], case["out"]), seed, 4, torch.bfloat16)
    if own:
        from mirai_amd import CompressedGroupedExperts

        module = CompressedGroupedExperts.from_empty(num_experts=case["experts"],
                                                     quant_format="mxfp4")
        module.load_dense_weight("w1", w)
        state["module"] = module
    else:
        state["codes"], state["scales"] = _mx_encode(w)
    return state


# ------------------------------------------------------------- plain forms
def _pow2(e):
    """2^e in 64 bits, exactly, for whole e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _mx_encode(x):
    """(codes [..., B, 32] uint8, scales [..., B] uint8) of the last axis' blocks."""
    cols = x.shape[-1]
    blocks = -(-cols // BLOCK)
    x = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols)).unflatten(-1, (blocks, BLOCK))
    amax = x.float().abs().amax(-1)
    bad = ~torch.isfinite(amax)
    _, e = torch.frexp(torch.where(bad, torch.ones_like(amax), amax))  # amax = f * 2^e, f in [1/2, 1)
    e = torch.where(amax == 0, torch.full_like(e, -127), (e - 3).clamp(-127, 125))
    y = x.abs().double() * _pow2(-e)[..., None]
    # Nearest level, ties to the even code.
    code = torch.zeros(y.shape, dtype=torch.uint8, device=x.device)
    for i in range(7):
        mid = (LEVELS[i] + LEVELS[i + 1]) / 2
        code += ((y > mid) if i % 2 == 0 else (y >= mid)).to(torch.uint8)
    code += 8 * torch.signbit(x).to(torch.uint8)
    scale = torch.where(bad, torch.full_like(e, 128), e) + 127
    return code, scale.to(torch.uint8)


def _mx_values(codes, scales, cols, dtype=torch.float32):
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=dtype, device=codes.device)
    x = table[codes.int()] * _pow2(scales.long() - 127).to(dtype)[..., None]
    x = torch.where((scales == 255)[..., None], torch.full_like(x, math.nan), x)
    return x.flatten(-2)[..., :cols]


def _mix(x):
    """32 well mixed bits of a 32-bit number (held in int64)."""
    mask = 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x9E3779B9) & mask
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & mask
    return x ^ (x >> 16)


def _noise(numel, seed, step, device):
    """Two 16-bit random numbers for each of ``numel`` < 2^32 positions (the first
    parameter group of an optimiser)."""
    key = _mix((_mix(seed & 0xFFFFFFFF) + step) & 0xFFFFFFFF)
    h = torch.arange(numel, dtype=torch.int64, device=device)
    h = h.add_(key).bitwise_and_(0xFFFFFFFF)
    h = h.bitwise_xor_(h >> 16).mul_(0x9E3779B9).bitwise_and_(0xFFFFFFFF)
    h = h.bitwise_xor_(h >> 15).mul_(0xBB67AE85).bitwise_and_(0xFFFFFFFF)
    h = h.bitwise_xor_(h >> 16)
    return (h & 0xFFFF).int(), (h >> 16).int()


def _moment_encode(x, ebits, signed, noise=None):
    """(codes uint8 [n], exponents uint8 [ceil(n / 128)]): sign (if signed), ebits of
    exponent and 3 of mantissa, times 2^E of the block; ``noise`` [n] holds 16
    random bits an element for stochastic rounding (None: to nearest, ties up)."""
    flat = x.reshape(-1)
    n = flat.numel()
    blocks = -(-n // STATE_BLOCK)
    flat = torch.nn.functional.pad(flat, (0, blocks * STATE_BLOCK - n)).view(blocks, STATE_BLOCK)
    amax = flat.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    _, e = torch.frexp(torch.where(bad, torch.ones_like(amax), amax))
    e = torch.where(amax == 0, torch.full_like(e, -126), (e - 1).clamp(-126, 126))
    y = (flat.abs().double() * _pow2(-e)[:, None]).float().reshape(-1)[:n]
    low = 2 - (1 << ebits)  # exponent of the smallest full binade
    sub = y < 2.0 ** low
    y = torch.where(sub, y + 2.0 ** low, y)
    bits = y.contiguous().view(torch.int32)
    bits = bits + (1 << 19 if noise is None else noise << 4)
    code = (bits >> 20) - ((low + 127) << 3) + torch.where(sub, 0, 8)
    code = code.clamp(0, (8 << ebits) - 1)
    if signed:
        code = code + (torch.signbit(x.reshape(-1)).int() << 7)
    code = torch.where(bad.repeat_interleave(STATE_BLOCK)[:n], torch.zeros_like(code), code)
    return code.to(torch.uint8), torch.where(bad, torch.full_like(e, 128), e).add(127).to(torch.uint8)


def _moment_values(codes, exps, ebits, signed, dtype=torch.float32):
    c = codes.int()
    mag = c & 0x7F if signed else c
    low = 2 - (1 << ebits)
    frac, ex = (mag & 7).to(dtype), mag >> 3
    y = torch.where(ex > 0, (1 + frac / 8) * _pow2(ex - 1 + low).to(dtype), frac * (2.0 ** low / 8))
    if signed:
        y = torch.where(c >= 128, -y, y)
    e = exps.repeat_interleave(STATE_BLOCK)[:codes.numel()]
    y = y * _pow2(e.long() - 127).to(dtype)
    return torch.where(e == 255, torch.full_like(y, math.nan), y)


def _segments(state):
    start = 0
    for e, end in enumerate(state["ends"]):
        if end > start:
            yield e, start, end
        start = end


def _plain_linear(state):
    case, x = state["case"], state["x"].detach()
    y = torch.empty((case["rows"], case["out"]), dtype=x.dtype, device=x.device)
    dx = torch.empty_like(x) if case["train"] else None
    for e, a, b in _segments(state):
        w = _mx_values(state["codes"][e], state["scales"][e], case["in"])
        rows = x[a:b].float()
        if case["kind"] == "linear4":
            rows = _mx_values(*_mx_encode(x[a:b]), case["in"])
        y[a:b] = (rows @ w.t()).to(y.dtype)
        if dx is not None:
            dx[a:b] = (state["dy"][a:b].float() @ w).to(dx.dtype)
    return {"y": y, "dx": dx} if case["train"] else y


def _plain_adamw(state):
    case = state["case"]
    state["step"] += 1
    t = state["step"]
    b1, b2 = ADAMW["betas"]
    step_size = ADAMW["lr"] / (1 - b1 ** t)
    root = math.sqrt(1 - b2 ** t)
    p, m, v = state["p"], state["m"], state["v"]
    if case["bits"] == 8:
        m, v = _moment_values(*m, 4, True), _moment_values(*v, 5, False)
    g = state["g"].float()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * (1 - b2) * g
    new = p.float() * (1 - ADAMW["lr"] * ADAMW["weight_decay"])
    p.copy_(new - step_size * (m / (v.sqrt() / root + ADAMW["eps"])))
    if case["bits"] == 32:
        state["m"], state["v"] = m, v
    else:
        low, high = _noise(p.numel(), 1234, t, p.device)
        state["m"], state["v"] = _moment_encode(m, 4, True, low), _moment_encode(v, 5, False, high)
        m, v = _moment_values(*state["m"], 4, True), _moment_values(*state["v"], 5, False)
    return {"params": p, "exp_avg": m, "exp_avg_sq": v}


# --------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "codec":
            x = state["x"]
            return _mx_values(*_mx_encode(x), case["cols"]).to(x.dtype)
        return _plain_adamw(state) if kind == "adamw" else _plain_linear(state)
    if kind == "codec":
        from mirai_amd import mxfp4_dequantize, mxfp4_quantize

        return mxfp4_dequantize(mxfp4_quantize(state["x"]), dtype=state["x"].dtype)
    if kind == "adamw":
        opt = state["opt"]
        opt.step()
        m, v = opt.flat_moments()
        return {"params": state["p"], "exp_avg": m, "exp_avg_sq": v}
    module, x = state["module"], state["x"]
    if kind == "linear4":
        return module.grouped_linear("w1", x, offsets=state["offsets"], activations="mxfp4")
    y = module.grouped_linear("w1", x, offsets=state["offsets"])
    if not case["train"]:
        return y
    (dx,) = torch.autograd.grad(y, x, state["dy"])
    return {"y": y.detach(), "dx": dx}


# -------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    size = {"bf16": 2, "fp32": 4}[case["dtype"]]
    if kind == "codec":
        n = case["lead"] * case["cols"]
        return {"bytes": 2 * size * n, "flops": 0}
    if kind == "adamw":
        n = _layout(case)[1]
        # Parameters and moments read and written, gradients read; 8-bit moments
        # are returned as the fp32 values they stand for.
        moments = 16 if case["bits"] == 32 else 4 + 8
        return {"bytes": n * (3 * size + moments), "flops": 14 * n}
    rows, in_f, out_f = case["rows"], case["in"], case["out"]
    active = sum(c > 0 for c in _counts(case))
    packed = active * in_f * out_f * 17 // 32
    passes = 2 if case["train"] else 1
    return {"bytes": passes * (size * rows * (in_f + out_f) + packed),
            "flops": passes * 2 * rows * in_f * out_f}


# ------------------------------------------------------------------- exact
def _binade(x):
    """floor(log2 x) of positive 64-bit x."""
    return (x.contiguous().view(torch.int64) >> 52) - 1023


def _exact_mx(x):
    """The values x's MXFP4 blocks stand for, in 64 bits, by arithmetic on the
    numbers (no codes): |x| / 2^E rounded to the spacing of its binade."""
    cols = x.shape[-1]
    blocks = -(-cols // BLOCK)
    x = torch.nn.functional.pad(x.double(), (0, blocks * BLOCK - cols)).unflatten(-1, (blocks, BLOCK))
    amax = x.abs().amax(-1, keepdim=True)
    scale = _pow2((_binade(amax.clamp_min(2.0 ** -160)) - 2).clamp(-127, 125))
    y = x / scale
    spacing = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    # torch.round takes ties to even multiples; multiples of the spacing have the parity of the code.
    y = (torch.round(y / spacing) * spacing).clamp(-6, 6)
    return (y * scale).flatten(-2)[..., :cols]


def _exact_moment(x, low, noise):
    """fp32 x -> the values its 8-bit block form stands for: the fraction of a
    spacing, plus the noise, rounded down."""
    flat = x.reshape(-1).double()
    n = flat.numel()
    blocks = -(-n // STATE_BLOCK)
    padded = torch.nn.functional.pad(flat, (0, blocks * STATE_BLOCK - n)).view(blocks, STATE_BLOCK)
    amax = padded.abs().amax(-1).clamp_min(2.0 ** -126)
    scale = _pow2(_binade(amax).clamp(-126, 126)).repeat_interleave(STATE_BLOCK)[:n]
    y = flat.abs() / scale
    base = 2.0 ** low
    # Below the smallest binade the value is first held to 24 bits next to it.
    y = torch.where(y < base, (y + base).float().double() - base, y)
    spacing = _pow2(_binade(y.clamp_min(base)) - 3)
    y = torch.floor(y / spacing + noise.double() / 65536) * spacing
    return (y.clamp(max=1.875) * scale * torch.where(flat < 0, -1.0, 1.0)).view(x.shape)


def _exact_adamw(case, seed):
    p, g, m, v = _step_inputs(case, seed)
    t = ADAMW_STEP + 1
    b1, b2 = ADAMW["betas"]
    g = g.double()
    if case["bits"] == 8:
        # The moments are defined by their fp32 roundings.
        def f(z):
            return z.float().double()

        c = [float(torch.tensor(z, dtype=torch.float32)) for z in (b1, 1 - b1, b2, 1 - b2)]
        half = torch.full((p.numel(),), 32768, device=p.device)
        m = f(f(_exact_moment(m, -14, half) * c[0]) + f(g * c[1]))
        v = f(f(_exact_moment(v, -30, half) * c[2]) + f(f(g * c[3]) * g))
    else:
        m = m.double() * b1 + g * (1 - b1)
        v = v.double() * b2 + g * g * (1 - b2)
    new = p.double() * (1 - ADAMW["lr"] * ADAMW["weight_decay"])
    new -= ADAMW["lr"] / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + ADAMW["eps"])
    if case["bits"] == 8:
        low, high = _noise(p.numel(), 1234, t, p.device)
        m, v = _exact_moment(m.float(), -14, low), _exact_moment(v.float(), -30, high)
    return {"params": new, "exp_avg": m, "exp_avg_sq": v}


def exact(case, seed):
    kind = case["kind"]
    if kind == "codec":
        return _exact_mx(_codec_input(case, seed))
    if kind == "adamw":
        return _exact_adamw(case, seed)
    x, w = _rows(case, seed), _weight(case, seed)
    dy = _randn((case["rows"], case["out"]), seed, 4, torch.bfloat16) if case["train"] else None
    y = torch.empty((case["rows"], case["out"]), dtype=torch.float64, device="cuda")
    dx = torch.empty((case["rows"], case["in"]), dtype=torch.float64, device="cuda")
    start = 0
    for e, end in enumerate(_ends(_counts(case))):
        if end > start:
            we = _exact_mx(w[e])
            rows = x[start:end]
            y[start:end] = (_exact_mx(rows) if kind == "linear4" else rows.double()) @ we.t()
            if dy is not None:
                dx[start:end] = dy[start:end].double() @ we
        start = end
    return {"y": y, "dx": dx} if case["train"] else y
