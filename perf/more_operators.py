"""The operators between two attentions of a transformer layer, for the rows of
many sessions: what is timed and compared.

A case names its operator (`kind`) and its sizes:

  norm     RMS norm of rows, the residual added and kept, the result in 16 or
           32 bits and as 8-bit rows for the products; without a weight the
           rows are quantized as they are (attention's output)
  rope     rotary positions of q and k rows, views of the packed QKV rows
  product  8-bit rows times a Q4_0 weight matrix
  ffn      gated feed-forward of 8-bit rows: both projections, the activation
           and their product, and the projection down

8-bit rows are int8 codes with an fp16 scale for each 32 elements: the least
fp16 that is not below the largest magnitude / 127; a code is the integer
nearest to the value / scale.  Outputs that are held so are returned as the
values that they stand for.  Weights are ggml Q4_0 blocks of 32: an fp16 scale
and 4-bit codes c, for the values (c - 8) * scale.
"""
import math

import torch

own = False


def listed():
    return [
        # one user's token between two layers: latency
        {"name": "norm, one token", "kind": "norm", "rows": 1, "dim": 4096, "type": "float32", "residual": "float32",
         "weight": True, "out": "float32", "codes": True},
        # the tokens of 64 sessions
        {"name": "norm, a token each", "kind": "norm", "rows": 64, "dim": 4096, "type": "float32",
         "residual": "float32", "weight": True, "out": "float32", "codes": True},
        # prompts: 16-bit rows out of a product into a 32-bit residual, 8-bit rows for the next product
        {"name": "norm, prompts", "kind": "norm", "rows": 6000, "dim": 4096, "type": "bfloat16", "residual": "float32",
         "weight": True, "out": "", "codes": True},
        # 48 sessions' q and k at the positions that they are at
        {"name": "rope, a token each", "kind": "rope", "tokens": 48, "heads": 32, "kv": 32, "dim": 128, "rot": 128,
         "interleaved": True, "type": "float32", "longest": 4000, "factor": 1.0, "trained": 0},
        # prompts of a model stretched to eight times its trained length, 32 query heads over 8 kv heads
        {"name": "rope, long prompts", "kind": "rope", "tokens": 5600, "heads": 32, "kv": 8, "dim": 128, "rot": 128,
         "interleaved": False, "type": "bfloat16", "longest": 65536, "factor": 8.0, "trained": 8192},
        # the QKV projection of one token
        {"name": "product, one token", "kind": "product", "rows": 1, "outs": 12288, "cols": 4096, "type": "float32"},
        # the output projection of 64 sessions' tokens
        {"name": "product, 64 sessions", "kind": "product", "rows": 64, "outs": 4096, "cols": 4096, "type": "float32"},
        # a vocabulary's logits for 17 sessions, a size that no tile divides
        {"name": "product, logits", "kind": "product", "rows": 17, "outs": 32001, "cols": 4096, "type": "float32"},
        # the QKV projection of prompts: the largest product
        {"name": "product, prompts", "kind": "product", "rows": 2048, "outs": 12288, "cols": 4096, "type": "bfloat16"},
        # the feed-forward block of one token
        {"name": "ffn, one token", "kind": "ffn", "rows": 1, "dim": 4096, "hidden": 5632, "act": "silu",
         "type": "bfloat16"},
        # of 48 sessions' tokens
        {"name": "ffn, 48 sessions", "kind": "ffn", "rows": 48, "dim": 4096, "hidden": 5632, "act": "silu",
         "type": "bfloat16"},
        # of a batch of prompts, ragged
        {"name": "ffn, prompts", "kind": "ffn", "rows": 1000, "dim": 4096, "hidden": 5632, "act": "silu",
         "type": "bfloat16"},
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        # within the largest listed, and far enough from nothing for the plain form's launches to be seen
        if w["bytes"] <= 2.4e8 and w["flops"] <= 2.1e11:
            return c


_TYPES = ["float32", "float16", "bfloat16"]


def _draw(rng):
    kind = rng.choice(["norm", "norm", "rope", "rope", "product", "product", "product", "ffn", "ffn", "ffn"])
    if kind == "norm":
        codes = rng.random() < 0.7
        dim = 32 * _log_int(rng, 2, 400) if codes else _log_int(rng, 33, 12800)
        weight = not codes or rng.random() < 0.75
        x = rng.choice(_TYPES)
        return {"kind": kind, "rows": _log_int(rng, 1, 12000), "dim": dim, "type": x,
                "residual": rng.choice(["", x, "float32"]) if weight else "", "weight": weight,
                "out": rng.choice(["", x] if codes else [x]) if weight else "", "codes": codes}
    if kind == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        kv = rng.choice([1, 2, 5, 8, 16, 32])
        factor = rng.choice([1.0, 2.0, 8.0, 40.0])
        return {"kind": kind, "tokens": _log_int(rng, 1, 8000), "heads": kv * rng.choice([1, 2, 4]), "kv": kv,
                "dim": dim, "rot": rng.choice([dim, dim // 2, dim // 4]), "interleaved": rng.random() < 0.5,
                "type": rng.choice(_TYPES), "longest": _log_int(rng, 100, 1000000), "factor": factor,
                "trained": rng.choice([0, 4096, 32768]) if factor > 1 else 0}
    c = {"kind": kind, "rows": rng.choice([_log_int(rng, 1, 16), _log_int(rng, 1, 3000)])}
    if kind == "product":
        c.update(outs=_log_int(rng, 33, 32768), cols=32 * _log_int(rng, 2, 400), type=rng.choice(_TYPES))
    else:
        c.update(dim=32 * _log_int(rng, 4, 200), hidden=32 * _log_int(rng, 4, 400), act=rng.choice(["silu", "gelu"]),
                 type=rng.choice(["float16", "bfloat16"]))
    return c


def _size(type_):
    return 0 if not type_ else 4 if type_ == "float32" else 2


def work(c):
    if c["kind"] == "norm":
        n = c["rows"] * c["dim"]
        per = _size(c["type"]) + 2 * _size(c["residual"]) + _size(c["out"]) + (1 + 2 / 32 if c["codes"] else 0)
        return {"bytes": n * per + 4.0 * c["dim"] * c["weight"], "flops": 0.0}
    if c["kind"] == "rope":
        n = c["tokens"] * (c["heads"] + c["kv"]) * c["dim"]
        return {"bytes": 2.0 * n * _size(c["type"]) + 4 * c["tokens"], "flops": 0.0}
    m = c["rows"]
    if c["kind"] == "product":
        n, k = c["outs"], c["cols"]
        return {"bytes": n * k * 18 / 32 + m * k * 34 / 32 + m * n * _size(c["type"]), "flops": 2.0 * m * n * k}
    d, h = c["dim"], c["hidden"]
    return {"bytes": 3 * h * d * 18 / 32 + m * d * 34 / 32 + m * d * _size(c["type"]), "flops": 6.0 * m * d * h}


# ---- inputs ----------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, dim):
    """A layer's rows: N(0, 1), channel by channel of another size, one channel in a hundred far larger."""
    size = torch.exp(0.5 * _normal(g, dim))
    size[torch.rand(dim, generator=g, device="cuda") < 0.01] *= 20.0
    return _normal(g, rows, dim) * size


def _weights(g, outs, cols):
    """Q4_0 codes [outs][cols / 32][32] and scales [outs][cols / 32]."""
    codes = (_normal(g, outs, cols // 32, 32) * 2.7 + 8.0).round_().clamp_(0, 15).to(torch.uint8)
    scales = (0.2 + torch.rand(outs, cols // 32, generator=g, device="cuda")) / math.sqrt(cols) / 3.0
    return codes, scales.half()


def _matrix(codes, scales):
    """What a program keeps of its weights: the library's, or their values."""
    outs, blocks, _ = codes.shape
    if own:
        from bmo_jetson_amd import Q4Weights
        packed = torch.empty(outs, blocks, 18, dtype=torch.uint8, device="cuda")
        packed[:, :, :2] = scales.view(torch.uint8).view(outs, blocks, 2)
        packed[:, :, 2:] = codes[:, :, :16] | (codes[:, :, 16:] << 4)
        w = Q4Weights(outs, blocks * 32)
        w.load(packed, stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        return w
    return ((codes.float() - 8.0) * scales.float()[:, :, None]).view(outs, blocks * 32)


def _split(x):
    """Rows in 8 bits: (codes, scales)."""
    b = x.view(x.shape[0], -1, 32)
    d = b.abs().amax(dim=2) / 127.0
    h = d.half()
    up = (h.view(torch.int16) + 1).view(torch.float16)
    h = torch.where(h.to(x.dtype) < d, up, h)
    s = h.to(x.dtype)[:, :, None]
    q = torch.where(s > 0, (b / s).round(), 0.0)
    return q.to(torch.int8).view(x.shape), h


def _values(codes, scales):
    """What 8-bit rows stand for, in fp16."""
    n = codes.shape[0]
    return (codes.view(n, -1, 32) * scales.view(n, -1, 1)).view(n, -1)


def _rows8(g, rows, cols):
    return _split(_activations(g, rows, cols))


def _type(name):
    return getattr(torch, name)


def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, seed)


def _norm_inputs(c, seed):
    g = _generator(seed * 1000003 + 1)
    x = _activations(g, c["rows"], c["dim"]).to(_type(c["type"]))
    residual = (3.0 * _activations(g, c["rows"], c["dim"])).to(_type(c["residual"])) if c["residual"] else None
    weight = 0.5 + torch.rand(c["dim"], generator=g, device="cuda") if c["weight"] else None
    return x, residual, weight


def _prepare_norm(c, seed):
    x, residual, weight = _norm_inputs(c, seed)
    s = {"kind": "norm", "x": x, "residual": residual, "weight": weight, "eps": 1e-5, "out": None, "codes": None,
         "scales": None}
    if c["out"]:
        s["out"] = torch.empty(c["rows"], c["dim"], dtype=_type(c["out"]), device="cuda")
    if c["codes"]:
        s["codes"] = torch.empty(c["rows"], c["dim"], dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty(c["rows"], c["dim"] // 32, dtype=torch.float16, device="cuda")
    return s


def _rope_inputs(c, seed):
    g = _generator(seed * 1000003 + 2)
    h, kv, n = c["heads"], c["kv"], c["tokens"]
    rows = _normal(g, n, h + 2 * kv, c["dim"]).to(_type(c["type"]))
    positions = torch.randint(0, c["longest"], (n,), generator=g, device="cuda", dtype=torch.int32)
    return rows[:, :h], rows[:, h:h + kv], positions


def _prepare_rope(c, seed):
    q, k, positions = _rope_inputs(c, seed)
    s = {"kind": "rope", "q": q, "k": k, "positions": positions, "interleaved": c["interleaved"], "rot": c["rot"]}
    if own:
        from bmo_jetson_amd import Rope
        s["rope"] = Rope(c["dim"], c["rot"], theta=10000.0, interleaved=c["interleaved"], factor=c["factor"],
                         trained=c["trained"])
        s["out"] = [torch.empty(x.shape, dtype=x.dtype, device="cuda") for x in (q, k)]
    else:
        i = torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda")
        s["rate"], s["magnitude"] = _rates(i, c)
    return s


def _rates(i, c):
    """Radians a position of pair i, and the magnitude, scaled for long contexts (linearly, or by YaRN's
    blend of scaled slow and unscaled fast pairs)."""
    base = 10000.0 ** (-2.0 * i / c["rot"])
    if not c["trained"]:
        return base / c["factor"], 1.0

    def turns(n):  # the pair that turns n times over the trained length
        return c["rot"] * math.log(c["trained"] / (n * 2 * math.pi)) / (2 * math.log(10000.0))

    low, high = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), c["rot"] - 1)
    slow = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    return base * (1.0 - slow) + base / c["factor"] * slow, 0.1 * math.log(c["factor"]) + 1.0


def _product_inputs(c, seed):
    g = _generator(seed * 1000003 + 3)
    return _weights(g, c["outs"], c["cols"]), _rows8(g, c["rows"], c["cols"])


def _prepare_product(c, seed):
    weights, (codes, scales) = _product_inputs(c, seed)
    return {"kind": "product", "w": _matrix(*weights), "codes": codes, "scales": scales,
            "out": torch.empty(c["rows"], c["outs"], dtype=_type(c["type"]), device="cuda")}


def _ffn_inputs(c, seed):
    g = _generator(seed * 1000003 + 4)
    # (the first half of the rows are the gate's, as in the packed matrices of gated models)
    return _weights(g, 2 * c["hidden"], c["dim"]), _weights(g, c["dim"], c["hidden"]), _rows8(g, c["rows"], c["dim"])


def _prepare_ffn(c, seed):
    into, down, (codes, scales) = _ffn_inputs(c, seed)
    m, h = c["rows"], c["hidden"]
    return {"kind": "ffn", "in": _matrix(*into), "down": _matrix(*down), "codes": codes, "scales": scales,
            "act": c["act"], "hidden": torch.empty(m, h, dtype=torch.int8, device="cuda"),
            "hidden_scales": torch.empty(m, h // 32, dtype=torch.float16, device="cuda"),
            "out": torch.empty(m, c["dim"], dtype=_type(c["type"]), device="cuda")}


# ---- run -------------------------------------------------------------------


def run(state):
    return globals()["_run_" + state["kind"]](state)


def _run_norm(s):
    if own:
        from bmo_jetson_amd import quantize_rows, rms_norm
        stream = torch.cuda.current_stream()
        if s["weight"] is None:
            quantize_rows(s["x"], s["codes"], s["scales"], stream=stream)
        else:
            rms_norm(s["x"], s["weight"], s["eps"], residual=s["residual"], out=s["out"], codes=s["codes"],
                     scales=s["scales"], stream=stream)
        values = None if s["codes"] is None else _values(s["codes"], s["scales"])
        return {"residual": s["residual"], "out": s["out"], "values": values}
    y = s["x"].float()
    if s["weight"] is not None:
        if s["residual"] is not None:
            s["residual"].copy_(s["residual"].float() + y)
            y = s["residual"].float()
        y = y * torch.rsqrt((y * y).mean(dim=1, keepdim=True) + s["eps"]) * s["weight"]
    return {"residual": s["residual"], "out": None if s["out"] is None else y.to(s["out"].dtype),
            "values": None if s["codes"] is None else _values(*_split(y))}


def _turn(x, angle, magnitude, rot, interleaved):
    cos, sin = ((f(angle) * magnitude).float()[:, None, :] for f in (torch.cos, torch.sin))
    y = x.float().clone()
    t = y[:, :, :rot]
    a, b = (t[..., 0::2], t[..., 1::2]) if interleaved else (t[..., :rot // 2], t[..., rot // 2:])
    c, d = a * cos - b * sin, a * sin + b * cos
    y[:, :, :rot] = torch.stack((c, d), dim=3).flatten(2) if interleaved else torch.cat((c, d), dim=2)
    return y.to(x.dtype)


def _run_rope(s):
    if own:
        s["rope"].apply(s["positions"], s["q"], s["k"], q_out=s["out"][0], k_out=s["out"][1],
                        stream=torch.cuda.current_stream())
        return {"q": s["out"][0], "k": s["out"][1]}
    angle = s["positions"].double()[:, None] * s["rate"]
    return {n: _turn(s[n], angle, s["magnitude"], s["rot"], s["interleaved"]) for n in ("q", "k")}


def _times(codes, scales, w):
    n = codes.shape[0]
    x = (codes.float().view(n, -1, 32) * scales.float()[:, :, None]).view(n, -1)
    return x @ w.t()


def _run_product(s):
    if own:
        s["w"].product(s["codes"], s["scales"], s["out"], stream=torch.cuda.current_stream())
        return {"out": s["out"]}
    return {"out": _times(s["codes"], s["scales"], s["w"]).to(s["out"].dtype)}


def _activation(x, act):
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))


def _run_ffn(s):
    if own:
        stream = torch.cuda.current_stream()
        s["in"].gated(s["codes"], s["scales"], s["hidden"], s["hidden_scales"], activation=s["act"], stream=stream)
        s["down"].product(s["hidden"], s["hidden_scales"], s["out"], stream=stream)
        return {"out": s["out"]}
    both = _times(s["codes"], s["scales"], s["in"])
    half = both.shape[1] // 2
    codes, scales = _split(_activation(both[:, :half], s["act"]) * both[:, half:])
    return {"out": _times(codes, scales, s["down"]).to(s["out"].dtype)}


# ---- the definitions in 64 bits ----------------------------------------------


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, seed)


def _in_8_bits(x):
    """The values that rows (64 bits) have in 8 bits."""
    blocks = x.reshape(-1, 32)
    largest = blocks.abs().max(dim=1, keepdim=True).values / 127.0
    scale = largest.to(torch.float16)
    scale = torch.where(scale.double() < largest, torch.nextafter(scale.cpu(), torch.tensor(math.inf).half()).to(scale.device),
                        scale).double()
    codes = torch.round(blocks / torch.where(scale > 0, scale, 1.0))
    return (codes * scale).reshape(x.shape)


def _exact_norm(c, seed):
    x, residual, weight = _norm_inputs(c, seed)
    h = x.double()
    if residual is not None:
        h = h + residual.double()
        residual = h.to(residual.dtype) if residual.dtype != torch.float32 else h.float()
        h = residual.double()
    y = h
    if weight is not None:
        y = h / torch.sqrt(h.pow(2).sum(dim=1, keepdim=True) / c["dim"] + 1e-5) * weight.double()
    return {"residual": residual, "out": y if c["out"] else None, "values": _in_8_bits(y) if c["codes"] else None}


def _exact_rope(c, seed):
    q, k, positions = _rope_inputs(c, seed)
    rate, magnitude = _rates(torch.arange(c["rot"] // 2, dtype=torch.float64), c)
    at = positions.double()[:, None] * rate.to("cuda")[None, :]
    turn = torch.polar(torch.full_like(at, magnitude), at)[:, None, :]
    out = {}
    for name, x in (("q", q), ("k", k)):
        y = x.double()
        t = y[..., :c["rot"]].unflatten(2, (-1, 2) if c["interleaved"] else (2, -1))
        pair = 3 if c["interleaved"] else 2
        z = torch.complex(t.select(pair, 0), t.select(pair, 1)) * turn
        y[..., :c["rot"]] = torch.stack((z.real, z.imag), dim=pair).flatten(2)
        out[name] = y
    return out


def _product64(codes, scales, w):
    """Rows of 64-bit values or 8-bit rows times Q4_0 weights, some rows of the matrix at a time."""
    x = codes.double()
    if scales is not None:
        x = (x.unflatten(1, (-1, 32)) * scales.double()[..., None]).flatten(1)
    out = []
    for i in range(0, w[0].shape[0], 4096):
        values = (w[0][i:i + 4096].double() - 8.0) * w[1][i:i + 4096].double()[..., None]
        out.append(torch.mm(x, values.flatten(1).t().contiguous()))
    return torch.cat(out, dim=1)


def _exact_product(c, seed):
    weights, (codes, scales) = _product_inputs(c, seed)
    return {"out": _product64(codes, scales, weights)}


def _exact_ffn(c, seed):
    into, down, (codes, scales) = _ffn_inputs(c, seed)
    gate, up = _product64(codes, scales, into).chunk(2, dim=1)
    if c["act"] == "silu":
        act = gate * torch.sigmoid(gate)
    else:
        act = 0.5 * gate * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate**3)))
    return {"out": _product64(_in_8_bits(act * up), None, down)}
