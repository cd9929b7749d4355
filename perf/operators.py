"""The products of weights in 4 bits: what a decode step, a prompt and a layer
of experts have this engine compute when its weights are microscaled 4-bit
floating point (E2M1 elements, one E8M0 power of two for every 32 of them
along a row).

Four operators:

* ``quantise``: rows to 4 bits and back to the values that they stand for;
* ``linear16``: ``x @ w.T + bias``, x in bfloat16, w in 4 bits;
* ``linear4``: the same with x brought to 4 bits on the way, as w is;
* ``experts``: a whole mixture-of-experts layer for a few tokens: router,
  choice, gate and up, activation, down, weighted sum; experts in 4 bits.

``run`` computes them in 32 bits with elementary operations, or (``own``)
through ``prism_b200.ops``.  ``exact`` computes them in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda:0"
BLOCK, GROUP, TILE = 32, 128, 128      # elements of a scale; K is padded to a group of four blocks; rows of a tile of scales
MOST_WEIGHTS = 37888 * 3584            # the largest listed matrix
MOST_FLOPS = 2.0 * 2048 * 28672 * 4096

# ---- cases --------------------------------------------------------------------------------------------------


def listed():
    return [
        # the activations of a decode step of 16 requests before a product in 4 bits (width of the 7B shape)
        dict(name="quantise step", op="quantise", rows=16, k=3584, dtype="bfloat16"),
        # a layer's gate and up weights when a model folder is loaded (7B shape)
        dict(name="quantise weights", op="quantise", rows=37888, k=3584, dtype="bfloat16"),
        # one request's decode step: q, k and v of the 7B shape, with their bias
        dict(name="qkv 1 token", op="linear16", m=1, n=4608, k=3584, bias=True),
        # a decode step of 16 requests: the down projection of the 7B shape
        dict(name="down 16 tokens", op="linear16", m=16, n=3584, k=18944, bias=False),
        # a decode step of 64 requests: gate and up of the 7B shape
        dict(name="gate up 64 tokens", op="linear16", m=64, n=37888, k=3584, bias=False),
        # a prompt of 2,048 tokens: gate and up of the width-4,096 designs
        dict(name="gate up prompt", op="linear16", m=2048, n=28672, k=4096, bias=False),
        # a decode step of 8 requests, activations in 4 bits too: gate and up of the 0.5B shape
        dict(name="both 8 tokens", op="linear4", m=8, n=9728, k=896, bias=False),
        # a short portion of a prompt with sizes that fill no tile and no block
        dict(name="both odd portion", op="linear4", m=333, n=1001, k=1003, bias=True),
        # a prompt of 2,048 tokens: gate and up of the width-4,096 designs
        dict(name="both prompt", op="linear4", m=2048, n=28672, k=4096, bias=False),
        # one request's decode step through the width-2,048 designs' experts
        dict(name="experts 1 token", op="experts", t=1, h=2048, f=672, e=8, top=2, score="sigmoid", renorm=False, scale_input=True),
        # a decode step of 16 requests through the width-4,096 designs' experts
        dict(name="experts 16 tokens", op="experts", t=16, h=4096, f=1184, e=8, top=2, score="softmax", renorm=True, scale_input=False),
        # a decode step of 64 requests through many small experts
        dict(name="experts 64 tokens", op="experts", t=64, h=2048, f=1024, e=64, top=8, score="softmax", renorm=True, scale_input=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quantise", "linear16", "linear4", "experts"])
    if op == "quantise":
        k = _log(rng, 32, 18944)
        return dict(op=op, rows=_log(rng, 1, min(37888, MOST_WEIGHTS // k)), k=k, dtype=rng.choice(["bfloat16", "float32"]))
    if op == "experts":
        t, h, f = _log(rng, 1, 64), _log(rng, 64, 4096), _log(rng, 32, 2048)
        e = _log(rng, 2, max(2, min(64, 64 * 1024 * 2048 // (h * f))))
        return dict(op=op, t=t, h=h, f=f, e=e, top=rng.randint(1, min(8, e)), score=rng.choice(["softmax", "sigmoid"]),
                    renorm=rng.random() < 0.5, scale_input=rng.random() < 0.5)
    k = _log(rng, 64, 18944)
    n = _log(rng, 64, min(37888, MOST_WEIGHTS // k))
    return dict(op=op, m=_log(rng, 1, min(2048, int(MOST_FLOPS / (2.0 * n * k)))), n=n, k=k, bias=rng.random() < 0.5)


def work(case):
    bits = 17 / 32                      # bytes of an element: half a byte and its share of the scale
    if case["op"] == "quantise":
        n = case["rows"] * case["k"]
        return {"bytes": n * ((2 if case["dtype"] == "bfloat16" else 4) + 2), "flops": 4.0 * n}
    if case["op"] == "experts":
        t, h, f, e, top = (case[s] for s in ("t", "h", "f", "e", "top"))
        live = e * (1.0 - (1.0 - top / e) ** t)          # the experts that t tokens choose between them, at an even choice
        return {"bytes": live * 3 * f * h * bits + 2 * e * h + 4 * t * h, "flops": 6.0 * t * top * f * h + 2.0 * t * e * h}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": n * k * bits + 2 * m * k + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2.0 * m * n * k}


# ---- the format, in elementary operations ---------------------------------------------------------------------


def _blocks(x):
    """Rows in float32, K padded with zeros to whole groups, as ``[..., blocks, 32]``."""
    k = x.shape[-1]
    return torch.nn.functional.pad(x.float(), (0, -k % GROUP)).unflatten(-1, (-1, BLOCK))


def _quantise(x):
    """``(codes 0 to 15 [..., blocks, 32], exponents [..., blocks])``: the exponent is that of the block's largest magnitude
    less two; elements round to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code, and 6 is the most."""
    b = _blocks(x)
    most = b.abs().amax(-1)
    e = torch.where(most > 0, torch.frexp(most).exponent - 3, torch.full_like(most, -127, dtype=torch.int32)).clamp(min=-127)
    v = torch.ldexp(b.abs(), -e.unsqueeze(-1))
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    q = torch.clamp(torch.round(v / step) * step, max=6.0)
    code = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q * 0.5 + 4)).to(torch.uint8)
    return code + 8 * (b < 0).to(torch.uint8), e


def _values(code, e):
    """The values that codes and exponents stand for, float32 ``[..., blocks * 32]``."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=code.device)
    return torch.ldexp(table[code.int()], e.unsqueeze(-1)).flatten(-2)


def _pack(code, e):
    """Codes two a byte (the even element in the low half) and scale bytes in tiles of 128 rows by four blocks: row r's
    four bytes at ``(r % 32) * 16 + r % 128 // 32 * 4`` of its tile."""
    flat = code.flatten(-2)
    codes = flat[..., 0::2] | (flat[..., 1::2] << 4)
    s = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, 0, 0, -e.shape[-2] % TILE))
    s = s.unflatten(-1, (-1, 4)).unflatten(-3, (-1, 4, 32))                        # [..., tile, row / 32, row % 32, group, 4]
    n = s.dim()
    s = s.permute(*range(n - 5), n - 5, n - 2, n - 3, n - 4, n - 1)                # [..., tile, group, row % 32, row / 32, 4]
    return codes.contiguous(), s.flatten(-3).contiguous()


def _unpack(codes, scales, rows):
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, BLOCK))
    s = scales.unflatten(-1, (32, 4, 4))
    n = s.dim()
    s = s.permute(*range(n - 5), n - 5, n - 2, n - 3, n - 4, n - 1).flatten(-2).flatten(-4, -2)
    return code, s[..., :rows, :].int() - 127


def _weight_values(w, k):
    return _values(*_unpack(w["codes"], w["scales"], w["codes"].shape[-2]))[..., :k]


# ---- inputs -----------------------------------------------------------------------------------------------------


def _activations(g, t, k):
    """Normed rows: some channels are several times as large as the others."""
    channel = torch.exp(0.7 * torch.randn(k, generator=g, device=DEV))
    return (torch.randn(t, k, generator=g, device=DEV) * channel).to(torch.bfloat16)


def _weights(g, *shape):
    w = torch.randn(*shape, generator=g, device=DEV).mul_(shape[-1] ** -0.5)
    codes, scales = _pack(*_quantise(w))
    return dict(codes=codes, scales=scales)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 13)
    s = dict(case=case)
    if case["op"] == "quantise":
        x = torch.randn(case["rows"], case["k"], generator=g, device=DEV)
        x = x * torch.exp(0.7 * torch.randn(case["k"], generator=g, device=DEV))
        return dict(s, x=x.to(getattr(torch, case["dtype"])))
    if case["op"] == "experts":
        t, h, f, e = (case[n] for n in ("t", "h", "f", "e"))
        return dict(s, x=_activations(g, t, h), router=(torch.randn(e, h, generator=g, device=DEV) * h ** -0.5).to(torch.bfloat16),
                    gate=_weights(g, e, f, h), up=_weights(g, e, f, h), down=_weights(g, e, h, f))
    m, n, k = case["m"], case["n"], case["k"]
    return dict(s, x=_activations(g, m, k), w=_weights(g, n, k),
                bias=torch.randn(n, generator=g, device=DEV).to(torch.bfloat16) if case["bias"] else None)


# ---- one pass -----------------------------------------------------------------------------------------------------


def _own_weight(ops, w, k):
    return ops.Mxfp4(w["codes"], w["scales"], k)


def _run_own(s):
    from prism_b200 import ops
    case = s["case"]
    if case["op"] == "quantise":
        return ops.mxfp4_quantize(s["x"]).dequantize(torch.bfloat16)
    if case["op"] == "experts":
        h, f = case["h"], case["f"]
        return ops.mxfp4_moe(s["x"], s["router"], _own_weight(ops, s["gate"], h), _own_weight(ops, s["up"], h),
                             _own_weight(ops, s["down"], f), case["top"], softmax=case["score"] == "softmax",
                             renorm=case["renorm"], scale_input=case["scale_input"])
    return ops.mxfp4_linear(s["x"], _own_weight(ops, s["w"], case["k"]), s["bias"], act_bits=16 if case["op"] == "linear16" else 4)


def _run_plain(s):
    case, x = s["case"], s["x"]
    if case["op"] == "quantise":
        return _values(*_quantise(x))[..., :case["k"]].to(torch.bfloat16)
    if case["op"] == "experts":
        t, h, f, e, top = (case[n] for n in ("t", "h", "f", "e", "top"))
        x = x.float()
        z = x @ s["router"].float().t()
        p = torch.exp(z - z.amax(-1, keepdim=True)) if case["score"] == "softmax" else 1 / (1 + torch.exp(-z))
        p = p / p.sum(-1, keepdim=True) if case["score"] == "softmax" else p
        best, index = torch.sort(p, dim=-1, descending=True, stable=True)
        best, index = best[:, :top], index[:, :top]
        best = best / best.sum(-1, keepdim=True) if case["renorm"] else best
        c = torch.zeros(t, e, device=x.device).scatter(1, index, best).t().unsqueeze(-1)         # [e, t, 1], 0: not chosen
        g = x @ _weight_values(s["gate"], h).transpose(1, 2)                                     # [e, t, f]
        u = x @ _weight_values(s["up"], h).transpose(1, 2)
        if case["scale_input"]:
            g, u = g * c, u * c
        a = g / (1 + torch.exp(-g)) * u
        if not case["scale_input"]:
            a = a * c
        return (a @ _weight_values(s["down"], f).transpose(1, 2)).sum(0).to(torch.bfloat16)
    k = case["k"]
    x = _values(*_quantise(x))[..., :k] if case["op"] == "linear4" else x.float()
    y = x @ _weight_values(s["w"], k).t()
    return (y if s["bias"] is None else y + s["bias"].float()).to(torch.bfloat16)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------


def exact(case, seed):
    def values(w, k):
        """Byte by byte from the definition: sign, two bits of exponent, one of fraction; the scale's place by its formula."""
        codes = w["codes"]
        rows, dev = codes.shape[-2], codes.device
        out = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=dev)
        r = torch.arange(rows, device=dev).unsqueeze(1)
        b = torch.arange(codes.shape[-1] // 16, device=dev).unsqueeze(0)
        place = ((r // 128 * w["scales"].shape[-2] + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4)
        power = torch.exp2(w["scales"].flatten(-3)[..., place].double() - 127)                        # [..., rows, blocks]
        for half in (0, 1):
            c = ((codes >> (4 * half)) & 15).double()
            sign = 1 - 2 * torch.floor(c / 8)
            m = c % 8
            ex, fr = torch.floor(m / 2), m % 2
            mag = torch.where(ex == 0, fr * 0.5, torch.exp2(ex - 1) * (1 + fr * 0.5))
            out[..., half::2] = (sign * mag).unflatten(-1, (-1, 16)).mul(power.unsqueeze(-1)).flatten(-2)
        return out[..., :k]

    def quantised(x):
        """The nearest element of each value, by distance to the fifteen of them."""
        x = x.double()
        k = x.shape[-1]
        out = torch.empty_like(x)
        grid = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
        for at in range(0, k, 32):
            block = x[:, at:at + 32]
            most = block.abs().amax(1, keepdim=True)
            p = torch.floor(torch.log2(torch.where(most > 0, most, torch.ones_like(most))))
            p = torch.where(torch.exp2(p) > most, p - 1, p)
            p = torch.where(torch.exp2(p + 1) <= most, p + 1, p)
            scale = torch.exp2(torch.clamp(p - 2, min=-127.0))
            v = block.abs() / scale
            near, dist = torch.zeros_like(v), v.clone()
            for i, value in enumerate(grid[1:], 1):
                d = (v - value).abs()
                closer = (d < dist) | ((d == dist) & (i % 2 == 0))
                near, dist = torch.where(closer, torch.full_like(v, value), near), torch.where(closer, d, dist)
            out[:, at:at + 32] = torch.sign(block) * near * scale
        return out

    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "quantise":
        return quantised(s["x"])
    if case["op"] == "experts":
        top = case["top"]
        z = x @ s["router"].double().t()
        score = torch.softmax(z, -1) if case["score"] == "softmax" else torch.sigmoid(z)
        y = torch.zeros_like(x)
        rank = torch.argsort(-score, dim=-1, stable=True)[:, :top]
        weight = score.gather(1, rank)
        if case["renorm"]:
            weight = weight / weight.sum(1, keepdim=True)
        for e in range(case["e"]):
            tok, place = torch.nonzero(rank == e, as_tuple=True)
            if not tok.numel():
                continue
            one = lambda w, k: values(dict(codes=w["codes"][e], scales=w["scales"][e]), k)      # noqa: E731
            c = weight[tok, place].unsqueeze(1)
            inp = x[tok] * c if case["scale_input"] else x[tok]
            hid = torch.nn.functional.silu(inp @ one(s["gate"], case["h"]).t()) * (inp @ one(s["up"], case["h"]).t())
            out = hid @ one(s["down"], case["f"]).t()
            y[tok] += out if case["scale_input"] else out * c
        return y
    x = quantised(s["x"]) if case["op"] == "linear4" else x
    y = x @ values(s["w"], case["k"]).t()
    return y if s["bias"] is None else y + s["bias"].double()
