"""Layer norm and AdamW, as cases to time: the operators of a training step between and behind its
Linear layers, through `axonn_amd.ops`.

A case is one call of one operator:

  norm       y = norm(x) w + b, or of x + residual with the sum as a second result: what stands in
             front of every projection of a pre-norm decoder layer
  norm_grad  its backward pass: dx (with the gradient that reaches the sum from elsewhere), dw, db
  adamw      the AdamW step over a list of tensors, moments in 32 bits
  adamw8     the same with moments in 8 bits, and the moments read back as numbers

`listed()` names twelve of them, `draw()` gives others of the same ranges.  Activations have a few
features far larger than the others, as those of decoders have; gradients and moments are normal
with the scales of a network in training.

With `own` false `run` computes a case in plain torch operations, else by the package's kernels.
`exact` gives the results in 64 bits.

8-bit moments come in blocks of 256 elements with one exponent E per block and moment.  A code of
the first moment is a sign, four bits of exponent and three of mantissa, one of the second five and
three, both with gradual underflow: F(c) = c / 8 for c < 8, else (1 + (c & 7) / 8) 2^((c >> 3) - 1),
and the moments are +-F(c) 2^(E - 141) and F(c) 2^(E - 157).  E is the exponent field of the
block's largest magnitude as a float, the next one from a mantissa of 1.875 on.  A moment between
two codes takes the upper one with the probability of its place between them, drawn from a counter
and the step's seed; a second moment that is not zero takes at least code 1.  `codes` holds, for
every four elements, four codes of the first moment and then four of the second.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LOSS_SCALE = 65536.0
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY = 3e-4, 0.9, 0.999, 1e-8, 0.1
BLOCK = 256


def _norm(name, rows, features, dtype, params="same", residual=False, grad=False):
    return {"name": name, "kind": "norm_grad" if grad else "norm", "rows": rows, "features": features,
            "dtype": dtype, "params": params, "residual": residual}


def _step(name, elements, tensors, dtype, bits):
    return {"name": name, "kind": "adamw" if bits == 32 else "adamw8", "elements": elements,
            "tensors": tensors, "dtype": dtype}


def listed():
    return [
        # Generation: 16 sequences, one token each; the call is all latency.
        _norm("norm_decode_16", 16, 4096, "bf16", residual=True),
        # A prompt of a length that no tile divides, the first norm of a network.
        _norm("norm_prompt_777", 777, 2560, "fp16"),
        # A large batch in a wide network, parameters kept in fp32.
        _norm("norm_train_16384", 16384, 8192, "bf16", params="fp32", residual=True),
        # Full precision, rows of odd length that start anywhere.
        _norm("norm_odd_fp32", 3001, 1025, "fp32"),
        # The backward pass of a small full-precision network: a short call.
        _norm("grad_fp32_64", 64, 1024, "fp32", grad=True),
        # Two sequences of 2048 tokens in a decoder layer, with the residual stream's gradient.
        _norm("grad_decoder_4096", 4096, 4096, "bf16", residual=True, grad=True),
        # A large batch, parameters and their gradients in fp32.
        _norm("grad_train_16384", 16384, 5120, "bf16", params="fp32", grad=True),
        # Odd sizes both ways.
        _norm("grad_odd_fp16", 2999, 4099, "fp16", grad=True),
        # The optimizer of a small full-precision network.
        _step("adamw_4m", 4200000, 12, "fp32", 32),
        # A 1.3e9-parameter model in bf16.
        _step("adamw_1p3e9", 1300000000, 64, "bf16", 32),
        # A small fp16 network with loss scaling.
        _step("adamw8_8m", 8400000, 24, "fp16", 8),
        # A model of half a billion parameters whose moments take two bytes an element, not eight.
        _step("adamw8_5e8", 500000000, 64, "bf16", 8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "norm_grad", "norm_grad", "adamw", "adamw8"))
    if kind in ("norm", "norm_grad"):
        features = _log(rng, 32, 16384)
        if features > 64 and rng.random() < 0.6:   # most networks' widths are multiples of 64
            features -= features % 64
        rows = min(_log(rng, 1, 65536), 16384 * 8192 // features)
        c = _norm("", rows, features, rng.choice(("bf16", "bf16", "fp16", "fp32")),
                  rng.choice(("same", "fp32")), rng.random() < 0.5, kind == "norm_grad")
    else:
        bits = 32 if kind == "adamw" else 8
        c = _step("", _log(rng, 100000, 1000000000 if bits == 32 else 400000000), _log(rng, 1, 300),
                  rng.choice(("bf16", "bf16", "fp16", "fp32")), bits)
    c.pop("name")
    return c


# ---------------------------------------------------------------- prepare ----
def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    with torch.no_grad():
        if case["kind"] in ("norm", "norm_grad"):
            return _prepare_norm(case, gen)
        return _prepare_step(case, gen)


def _prepare_norm(case, gen):
    dtype, rows, features = DTYPES[case["dtype"]], case["rows"], case["features"]
    param = torch.float32 if case["params"] == "fp32" else dtype
    scale = torch.ones(features, device="cuda")
    loud = torch.randperm(features, generator=gen, device="cuda")[:max(1, features // 500)]
    scale[loud] = 20.0
    state = {"case": case,
             "weight": (1 + _normal(gen, features, std=0.1)).to(param),
             "bias": _normal(gen, features, std=0.1, dtype=param),
             "x": (_normal(gen, rows, features) * scale + 0.3).to(dtype)}
    if case["kind"] == "norm":
        state["residual"] = _normal(gen, rows, features, std=0.5, dtype=dtype) if case["residual"] else None
        return state
    std = 1e-3 * (LOSS_SCALE / 256 if dtype == torch.float16 else 1.0)
    state["dy"] = _normal(gen, rows, features, std=std, dtype=dtype)
    state["dsum"] = _normal(gen, rows, features, std=std, dtype=dtype) if case["residual"] else None
    # the statistics that the forward pass kept
    x = state["x"].float()
    state["mean"] = x.mean(-1)
    x -= state["mean"][:, None]
    state["rstd"] = 1.0 / torch.sqrt((x * x).mean(-1) + EPS)
    return state


def _tensor_sizes(total, count):
    """`count` odd and even sizes between a fraction and a few times their mean, a case's own."""
    w = torch.rand(count, generator=torch.Generator().manual_seed(total), dtype=torch.float64)
    w = torch.exp(w * math.log(100.0))
    sizes = [max(1, int(v)) for v in (w / w.sum() * total).tolist()]
    sizes[-1] = max(1, sizes[-1] + total - sum(sizes))
    return sizes


def _prepare_step(case, gen):
    dtype, eight = DTYPES[case["dtype"]], case["kind"] == "adamw8"
    sizes = _tensor_sizes(case["elements"], case["tensors"])
    # one flat buffer of each kind; tensors of 8-bit moments start at whole blocks of it
    spans = [-(-n // BLOCK) * BLOCK if eight else n for n in sizes]
    total, starts = sum(spans), [sum(spans[:i]) for i in range(len(spans))]
    grad_scale = LOSS_SCALE if dtype == torch.float16 else 1.0
    state = {"case": case, "step": 1000, "inv_scale": 1.0 / grad_scale,
             "p": _normal(gen, total, std=0.02),
             "g": _normal(gen, total, std=(1e-5 if dtype == torch.float16 else 1e-3) * grad_scale, dtype=dtype)}
    typical = 1e-5 if dtype == torch.float16 else 1e-3
    m = _normal(gen, total, std=0.3 * typical)
    v = (1 + 0.2 * _normal(gen, total)).abs_().mul_(typical * typical)
    if eight:
        inside = torch.zeros(total, dtype=torch.bool, device="cuda")
        for start, n in zip(starts, sizes):
            inside[start:start + n] = True
        for name in ("p", "g"):
            state[name].mul_(inside)
        state["codes"], state["exponents"] = _pack(m.mul_(inside), v.mul_(inside))
        state["code_views"] = [state["codes"][a // BLOCK:(a + b) // BLOCK] for a, b in zip(starts, spans)]
        state["exponent_views"] = [state["exponents"][a // BLOCK:(a + b) // BLOCK] for a, b in zip(starts, spans)]
    else:
        state["m"], state["v"] = m, v
    state["low"] = state["p"].to(dtype) if dtype != torch.float32 else None
    for name in ("p", "g", "m", "v", "low"):
        if state.get(name) is not None:
            state[name + "_views"] = [state[name][a:a + n] for a, n in zip(starts, sizes)]
    return state


# -------------------------------------------------------------------- run ----
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "norm_grad": _own_norm_grad, "adamw": _own_adamw, "adamw8": _own_adamw8}[kind](state)
    return {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "adamw": _plain_adamw, "adamw8": _plain_adamw8}[kind](state)


def _own_norm(state):
    from axonn_amd import ops

    y, total, _, _ = ops.layer_norm_fwd(state["x"], state["weight"], state["bias"], EPS, residual=state["residual"],
                                        save=False)
    return (y,) if state["residual"] is None else (y, total)


def _own_norm_grad(state):
    from axonn_amd import ops

    return ops.layer_norm_bwd(state["dy"], state["x"], state["weight"], state["mean"], state["rstd"],
                              dsum=state["dsum"])


def _own_adamw(state):
    from axonn_amd import ops

    state["step"] += 1
    ops.mt_adamw(state["g_views"], state["p_views"], state["m_views"], state["v_views"], state.get("low_views"),
                 ops.adamw_hparams(state["step"], LR, BETA1, BETA2, ADAM_EPS, DECAY), state["inv_scale"])
    return state["p"], state["m"], state["v"], state["low"]


def _own_adamw8(state):
    from axonn_amd import ops

    state["step"] += 1
    ops.mt_adamw8(state["g_views"], state["p_views"], state["code_views"], state["exponent_views"],
                  state.get("low_views"), ops.adamw_hparams(state["step"], LR, BETA1, BETA2, ADAM_EPS, DECAY),
                  _seed(state["step"]), state["inv_scale"])
    # (three bits of mantissa: bf16 holds them as they are)
    m, v = ops.adamw8_moments(state["codes"], state["exponents"], dtype=torch.bfloat16)
    return state["p"], m, v, state["low"]


# ------------------------------------------------------------ plain forms ----
def _plain_norm(state):
    h, dtype = state["x"].float(), state["x"].dtype
    total = None
    if state["residual"] is not None:
        total = (h + state["residual"].float()).to(dtype)
        h = total.float()
    d = h - h.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    y = (d * rstd * state["weight"].float() + state["bias"].float()).to(dtype)
    return (y,) if total is None else (y, total)


def _plain_norm_grad(state):
    dtype, param = state["x"].dtype, state["weight"].dtype
    rstd = state["rstd"][:, None]
    xhat = (state["x"].float() - state["mean"][:, None]) * rstd
    dy = state["dy"].float()
    a = dy * state["weight"].float()
    dx = (a - a.mean(-1, keepdim=True) - xhat * (a * xhat).mean(-1, keepdim=True)) * rstd
    if state["dsum"] is not None:
        dx = dx + state["dsum"].float()
    return dx.to(dtype), (dy * xhat).sum(0).to(param), dy.sum(0).to(param)


def _factors(step):
    """1 - lr decay, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)."""
    return 1.0 - LR * DECAY, LR / (1.0 - BETA1 ** step), 1.0 / math.sqrt(1.0 - BETA2 ** step)


def _update(p, m, v, step):
    keep, rate, root = _factors(step)
    return p * keep - rate * (m / (torch.sqrt(v) * root + ADAM_EPS))


def _plain_adamw(state):
    state["step"] += 1
    g = state["g"].float() * state["inv_scale"]
    state["m"] += (g - state["m"]) * (1.0 - BETA1)
    state["v"].mul_(BETA2).add_((1.0 - BETA2) * g * g)
    state["p"].copy_(_update(state["p"], state["m"], state["v"], state["step"]))
    if state["low"] is not None:
        state["low"].copy_(state["p"])
    return state["p"], state["m"], state["v"], state["low"]


def _seed(step):
    """The seed of a step's random words."""
    return (step * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 64)


def _words(blocks, seed, device):
    """The random words of all elements, [blocks, 64, 4], as 64-bit integers below 2^32."""
    low = 0xFFFFFFFF
    q = torch.arange(blocks * 64, dtype=torch.int64, device=device)
    x = ((q & low) ^ (seed & low)) * 0x9E3779B9 & low
    x = ((x ^ (x >> 16)) + (seed >> 32) + (q >> 32) & low) * 0x6A09E667 & low
    x = (x ^ (x >> 15))[:, None]
    w = x * torch.tensor([0xBB67AE85, 0x510E527F, 0x1F83D9AB, 0x5BE0CD19], device=device) & low
    return (w ^ (w >> 16)).view(blocks, 64, 4)


def _magnitudes(device):
    """F(c) of the codes 0 to 255."""
    c = torch.arange(256, device=device)
    return torch.where(c < 8, c / 8.0, (1 + (c & 7) / 8.0) * torch.exp2(((c >> 3) - 1).float()))


def _exponents(largest):
    """E of blocks whose largest magnitudes are these floats."""
    return ((largest.view(torch.int32) + 0x100000) >> 23).clamp(max=255)


def _scaled(x, power):
    """x 2^power, in two factors that a float holds."""
    half = torch.div(power, 2, rounding_mode="floor")
    return x * torch.exp2(half.float()) * torch.exp2((power - half).float())


def _encode(x, words):
    """Codes of magnitudes x, in units of F, given random words below 2^16: the bits of a float with
    three more of its mantissa's are the code, what is behind them is its place on the way to the next."""
    bits = (x * 2.0 ** -126).view(torch.int32)
    return (bits + (words.int() * 16 + 8)) >> 20


def _quantize(m, v, words):
    """(codes, exponents) of moments [blocks, 64, 4] in fp32."""
    exps = torch.stack([_exponents(t.abs().amax((1, 2))) for t in (m, v)], 1)
    cm = _encode(_scaled(m.abs(), (141 - exps[:, 0])[:, None, None]), words & 0xFFFF) | ((m < 0).int() << 7)
    cv = _encode(_scaled(v, (157 - exps[:, 1])[:, None, None]), words >> 16)
    cv = torch.maximum(cv, (v > 0).int())
    return torch.stack([cm, cv], 2).to(torch.uint8).view(-1, 2 * BLOCK), exps.to(torch.uint8)


def _pack(m, v):
    """(codes, exponents) of flat moments."""
    blocks = m.numel() // BLOCK
    return _quantize(m.view(blocks, 64, 4), v.view(blocks, 64, 4), _words(blocks, 0, m.device))


def _moments(codes, exponents):
    """The first and second moments that codes stand for, [blocks, 64, 4] in fp32."""
    c, table = codes.view(-1, 64, 2, 4).int(), _magnitudes(codes.device)
    e = exponents.int()[:, :, None, None]
    m = _scaled(table[c[:, :, 0] & 127], e[:, 0] - 141) * (1 - 2 * (c[:, :, 0] >> 7))
    return m, _scaled(table[c[:, :, 1]], e[:, 1] - 157)


def _plain_adamw8(state):
    state["step"] += 1
    g = (state["g"].float() * state["inv_scale"]).view(-1, 64, 4)
    m, v = _moments(state["codes"], state["exponents"])
    m += (g - m) * (1.0 - BETA1)
    v.mul_(BETA2).add_((1.0 - BETA2) * g * g)
    state["p"].copy_(_update(state["p"], m.view(-1), v.view(-1), state["step"]))
    if state["low"] is not None:
        state["low"].copy_(state["p"])
    codes, exponents = _quantize(m, v, _words(m.shape[0], _seed(state["step"]), g.device))
    state["codes"].copy_(codes)
    state["exponents"].copy_(exponents)
    m, v = _moments(state["codes"], state["exponents"])
    return state["p"], m.view(-1).bfloat16(), v.view(-1).bfloat16(), state["low"]


# -------------------------------------------------------------- in 64 bits ---
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "norm_grad": _exact_norm_grad, "adamw": _exact_adamw,
                "adamw8": _exact_adamw8}[case["kind"]](state)


def _exact_norm(state):
    h = state["x"].double()
    if state["residual"] is not None:
        total = h + state["residual"].double()
        h = total.to(state["x"].dtype).double()   # the norm is that of the sum as it is stored
    var, mean = torch.var_mean(h, -1, correction=0, keepdim=True)
    y = (h - mean) / torch.sqrt(var + EPS) * state["weight"].double() + state["bias"].double()
    return (y,) if state["residual"] is None else (y, total)


def _exact_norm_grad(state):
    """The gradient of sum(dy y) by the chain rule through y = xhat w + b, xhat = (x - mean) rstd."""
    x, dy, n = state["x"].double(), state["dy"].double(), state["case"]["features"]
    rstd = state["rstd"].double()[:, None]
    centred = x - state["mean"].double()[:, None]
    dxhat = dy * state["weight"].double()
    drstd = (dxhat * centred).sum(1, keepdim=True)
    dvar = drstd * rstd ** 3 * -0.5
    dx = dxhat * rstd + centred * (2.0 / n) * dvar
    dx = dx - (dxhat * rstd).sum(1, keepdim=True) / n
    if state["dsum"] is not None:
        dx = dx + state["dsum"].double()
    return dx, torch.einsum("ij,ij->j", dy, centred * rstd), dy.sum(0)


def _exact_step(state, m, v):
    t = state["step"] + 1
    g = state["g"].double() * state["inv_scale"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g.square()
    hat_m, hat_v = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    p = state["p"].double()
    p = p - LR * DECAY * p - LR * hat_m / (hat_v.sqrt() + ADAM_EPS)
    return p, m, v


def _exact_adamw(state):
    p, m, v = _exact_step(state, state["m"].double(), state["v"].double())
    return p, m, v, None if state["low"] is None else p


def _exact_adamw8(state):
    blocks = state["codes"].shape[0]
    t = state["step"] + 1
    codes = state["codes"].view(blocks, 64, 2, 4).double()

    def value(c, bias, which):
        octave = torch.clamp(torch.floor(c / 8) - 1, min=0)
        steps = torch.where(c < 8, c, 8 + torch.remainder(c, 8))
        e = state["exponents"][:, which].double()[:, None, None]
        return steps / 8 * torch.exp2(octave + e - bias)

    first = codes[:, :, 0]
    negative = first >= 128
    m = value(torch.where(negative, first - 128, first), 141, 0)
    m = torch.where(negative, -m, m).reshape(-1)
    v = value(codes[:, :, 1], 157, 1).reshape(-1)
    del codes, first, negative
    p, m, v = _exact_step(state, m, v)
    words = _words(blocks, _seed(t), p.device).view(-1)

    def rounded(x, bias, u, least):
        mantissa, exponent = torch.frexp(x.abs().view(blocks, BLOCK).amax(1))   # 1/2 <= mantissa < 1
        e = exponent + 126 + (mantissa >= 0.9375).int()
        unit = torch.exp2(e.double() - bias)
        y = (x.abs().view(blocks, BLOCK) / unit[:, None]).view(-1)
        octave = torch.clamp(torch.frexp(y)[1] - 1, min=0).double()
        step = torch.exp2(octave - 3)
        y = torch.floor(y / step + u) * step
        if least:
            y = torch.where(x > 0, torch.clamp(y, min=0.125), y)
        return (y.view(blocks, BLOCK) * unit[:, None]).view(-1) * torch.sign(x)

    m = rounded(m, 141, ((words & 0xFFFF).double() + 0.5) / 65536, False)
    v = rounded(v, 157, ((words >> 16).double() + 0.5) / 65536, True)
    return p, m, v, None if state["low"] is None else p


# ------------------------------------------------------------------- work ----
def work(case):
    """Inputs once and outputs once.  The 8-bit moments are read and written by the step, then read
    and written as numbers of two bytes."""
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] in ("norm", "norm_grad"):
        rows, n = case["rows"], case["features"]
        param = 4 if case["params"] == "fp32" else size
        if case["kind"] == "norm":
            return {"bytes": (4 if case["residual"] else 2) * rows * n * size + 2 * n * param, "flops": 8 * rows * n}
        return {"bytes": (4 if case["residual"] else 3) * rows * n * size + 8 * rows + 3 * n * param,
                "flops": 14 * rows * n}
    elements = case["elements"]
    copy = 2 if size == 2 else 0
    if case["kind"] == "adamw":
        return {"bytes": (size + 24 + copy) * elements, "flops": 14 * elements}
    return {"bytes": (size + 12 + copy + 2 + 4) * elements + 6 * (elements // BLOCK), "flops": 20 * elements}
