"""What a request brings of its own into a batch that it shares: a low-rank
adapter beside every projection, and the settings by which its next token is
drawn.

Two operators:

* ``adapters``: ``out = base + s (x A^T) B^T`` with A, B and s of each token's
  own adapter, or ``out = base`` for a token without one;
* ``draw``: a token from each row of logits by temperature, top-k, top-p and
  min-p, from a given uniform number; how many tokens it was drawn from, and
  the logarithm of the probability that it had.

``run`` computes them with elementary operations, in 32 bits, or 64 where a
value may lie next to a border, or (``own``) through ``prism_b200.ops``.
``exact`` computes them in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
MOST_VALUES = 256 * 152064             # logits of the largest listed draw
MOST_RESULTS = 2048 * 37888            # results of the largest listed product
MOST_WEIGHTS = 64 * 16 * (2 * 3584 + 37888)
MOST_FLOPS = 2.0 * 2048 * 64 * 4 * (2 * 3584 + 37888)      # of the plain form, which applies every adapter to every token

# ---- cases --------------------------------------------------------------------------------------------------


def listed():
    return [
        # one request's decode step: q, k and v of the 7B shape
        dict(name="adapter 1 token", op="adapters", singles=1, portions="", slices=3, n0=3584, n1=512, k=3584, rank=16, most=1,
             dtype="bfloat16"),
        # a decode step of 16 requests that share 8 adapters: the down projection of the 7B shape
        dict(name="adapters 16 tokens", op="adapters", singles=16, portions="", slices=1, n0=3584, n1=0, k=18944, rank=64, most=8,
             dtype="bfloat16"),
        # a decode step of 64 requests with an adapter each: gate and up of the 7B shape
        dict(name="adapters 64 tokens", op="adapters", singles=64, portions="", slices=2, n0=18944, n1=18944, k=3584, rank=16, most=64,
             dtype="bfloat16"),
        # a step of decoding requests and portions of three prompts: q, k and v of the 7B shape
        dict(name="adapters mixed step", op="adapters", singles=45, portions="771,130,512", slices=3, n0=3584, n1=512, k=3584, rank=32,
             most=16, dtype="bfloat16"),
        # prompts of 2,048 tokens in all: gate and up of the 7B shape
        dict(name="adapters prompts", op="adapters", singles=0, portions="1024,600,424", slices=2, n0=18944, n1=18944, k=3584, rank=64,
             most=4, dtype="bfloat16"),
        # a short portion in an engine of 32-bit floats, sizes that fill no tile
        dict(name="adapters odd float32", op="adapters", singles=3, portions="34", slices=2, n0=501, n1=77, k=1003, rank=5, most=3,
             dtype="float32"),
        # one request, the usual settings of a chat: vocabulary of the 7B shape
        dict(name="draw 1 request", op="draw", rows=1, vocab=152064, filters="k p", flat=False),
        # a few requests over a small odd vocabulary
        dict(name="draw odd vocabulary", op="draw", rows=5, vocab=1003, filters="min p", flat=False),
        # requests at high temperature over flat logits: a nucleus of tens of thousands (vocabulary of the 0.5B shape)
        dict(name="draw 8 flat", op="draw", rows=8, vocab=151936, filters="p", flat=True),
        # a decode step of 16 requests by top-p
        dict(name="draw 16 requests", op="draw", rows=16, vocab=152064, filters="p", flat=False),
        # a decode step of 64 requests, each with settings of its own
        dict(name="draw 64 mixed", op="draw", rows=64, vocab=152064, filters="mixed", flat=False),
        # a large batch by top-k and top-p
        dict(name="draw 256 requests", op="draw", rows=256, vocab=152064, filters="k p", flat=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    if rng.random() < 0.5:
        vocab = _log(rng, 32, 152064)
        return dict(op="draw", rows=_log(rng, 1, min(256, MOST_VALUES // vocab)), vocab=vocab,
                    filters=rng.choice(["k", "p", "min p", "k p", "mixed", "none"]), flat=rng.random() < 0.3)
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    slices, k = rng.choice([1, 1, 2, 3]), _log(rng, 32, 18944)
    n0 = _log(rng, 32, min(18944, 37888 // slices))
    n1 = n0 if slices == 2 else _log(rng, 16, n0) if slices == 3 else 0
    n = n0 + (slices - 1) * n1
    rank = _log(rng, 1, 128)
    kept = -(-rank // 16) * 16
    most = _log(rng, 1, max(1, min(64, MOST_WEIGHTS // (kept * (slices * k + n)))))
    room = min(4096, MOST_RESULTS // n, int(MOST_FLOPS / (2.0 * most * kept * (slices * k + n))))
    room = min(room, 512) if dtype == "float32" else room
    singles = rng.choice([0, _log(rng, 1, 64)])
    portions = [_log(rng, 2, max(2, room // 4)) for _ in range(rng.choice([0, 1, 2, 4]))]
    portions = portions or ([] if singles else [7])
    return dict(op="adapters", singles=singles, portions=",".join(str(p) for p in portions), slices=slices, n0=n0, n1=n1, k=k, rank=rank,
                most=most, dtype=dtype)


def _sizes(case):
    """``(tokens of the portions, tokens in all, rows of each slice)``"""
    portions = [int(p) for p in case["portions"].split(",") if p]
    return portions, case["singles"] + sum(portions), [case["n0"]] + [case["n1"]] * (case["slices"] - 1)


def work(case):
    if case["op"] == "draw":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 24 * case["rows"], "flops": 4.0 * n}
    portions, t, rows = _sizes(case)
    size, k, n, r = (2 if case["dtype"] == "bfloat16" else 4), case["k"], sum(rows), case["rank"]
    live = case["most"] * (1.0 - (1.0 - 1.0 / case["most"]) ** (case["singles"] + len(portions)))       # adapters that are used, at an even choice
    weights = case["slices"] * r * k + n * r
    return {"bytes": size * (t * k + 2 * t * n + live * weights) + 4 * t, "flops": 2.0 * t * weights}


# ---- inputs ---------------------------------------------------------------------------------------------------


def _logits(g, rows, vocab, flat):
    """Logits as a trained model's: a wide body, and a few tokens far above it, more of them in some rows than in others."""
    x = torch.randn(rows, vocab, generator=g, device=DEV)
    if flat:
        return x
    few = min(vocab, 200)
    at = torch.rand(rows, vocab, generator=g, device=DEV).argsort(1)[:, :few]
    top = 14.0 - 1.6 * torch.log1p(torch.arange(few, device=DEV)) * (0.5 + torch.rand(rows, 1, generator=g, device=DEV))
    return (1.8 * x).scatter_add(1, at, top)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)
    rand = lambda *shape: torch.rand(*shape, generator=g, device=DEV)            # noqa: E731
    if case["op"] == "draw":
        R, V, f = case["rows"], case["vocab"], case["filters"]
        s = dict(case=case, x=_logits(g, R, V, case["flat"]), u=rand(R), t=0.5 + rand(R) * (1.0 if case["flat"] else 0.7))
        which = torch.randint(0, 6, (R,), generator=g, device=DEV)               # mixed: greedy, by temperature alone, k, p, min-p, all
        have = lambda name, kinds: (f.startswith(name) or f.endswith(" " + name)) if f != "mixed" else sum(which == w for w in kinds) > 0      # noqa: E731
        pick = lambda on, value, off: torch.where(torch.as_tensor(on, device=DEV), value, torch.full_like(value, off))      # noqa: E731
        s["top_k"] = pick(have("k", (2, 5)), torch.randint(1, 101, (R,), generator=g, device=DEV).int(), 0)
        s["top_p"] = pick(f in ("p", "k p") if f != "mixed" else have("p", (3, 5)), 0.8 + 0.19 * rand(R), 1.0)
        s["min_p"] = pick(f == "min p" if f != "mixed" else have("min p", (4, 5)), 0.01 + 0.1 * rand(R), 0.0)
        if f == "mixed":
            s["t"] = torch.where(which == 0, torch.zeros_like(s["t"]), s["t"])
        return s
    portions, t, rows = _sizes(case)
    L, G, r, k, n, dt = case["most"], case["slices"], case["rank"], case["k"], sum(rows), getattr(torch, case["dtype"])
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)          # noqa: E731
    # one adapter for a decoding request, one for all tokens of a portion; some requests have none
    own_ids = torch.randint(-1 if L > 1 else 0, L, (case["singles"] + len(portions),), generator=g, device=DEV).int()
    if L >= case["singles"] > 8:
        own_ids[:case["singles"]] = torch.randperm(L, generator=g, device=DEV).int()[:case["singles"]]
    counts = torch.tensor([1] * case["singles"] + portions, device=DEV)
    # the rank in memory is a whole number of sixteens, a row of A a whole number of eights, zeros beyond
    kept, wide = -(-r // 16) * 16, -(-k // 8) * 8
    a, b = torch.zeros(L, G, kept, wide, device=DEV, dtype=dt), torch.zeros(L, n, kept, device=DEV, dtype=dt)
    a[:, :, :r, :k] = (randn(L, G, r, k) * k ** -0.5).to(dt)
    b[:, :, :r] = (randn(L, n, r) * (0.5 * r ** -0.5)).to(dt)
    x = randn(t, k) * torch.exp(0.7 * randn(k))
    return dict(case=case, x=x.to(dt), base=randn(t, n).to(dt), a=a, b=b, scale=0.5 + 1.5 * rand(L),
                ids=torch.repeat_interleave(own_ids, counts))


# ---- one pass -----------------------------------------------------------------------------------------------------


def _run_own(s):
    from prism_b200 import ops
    case = s["case"]
    if case["op"] == "draw":
        out, kept = torch.empty(2, case["rows"], dtype=torch.int32, device=DEV)
        logprob = torch.empty(case["rows"], device=DEV)
        ops.sample_filtered(s["x"], s["t"], s["u"], out, top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], kept=kept, logprob=logprob)
        return out, kept, logprob
    low = ops.LowRank(s["a"], s["b"], s["scale"], rows=_sizes(case)[2], k=case["k"])
    return ops.low_rank(s["x"], low, s["ids"], base=s["base"], singles=case["singles"])


def _run_plain(s):
    case = s["case"]
    if case["op"] == "draw":
        x, t = s["x"].double(), s["t"].double().unsqueeze(1)
        V = case["vocab"]
        best, index = torch.sort(x, dim=1, descending=True, stable=True)
        w = torch.exp((best - best[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
        place = torch.arange(V, device=x.device).unsqueeze(0)
        k = torch.where(s["top_k"] > 0, s["top_k"], torch.full_like(s["top_k"], V)).unsqueeze(1)
        w = w * (place < k)
        before = torch.cumsum(w, 1) - w
        p = s["top_p"].double().unsqueeze(1)
        kept = (p >= 1) | (before < p * w.sum(1, keepdim=True)) | (place == 0)
        kept = kept & (w >= s["min_p"].double().unsqueeze(1))
        count = (kept & (w > 0)).sum(1)
        w = torch.zeros_like(w).scatter(1, index, w * kept)
        run = torch.cumsum(w, 1)
        target = s["u"].double().unsqueeze(1) * run[:, -1:]
        token = (run <= target).sum(1)
        logprob = torch.log(w.gather(1, token.clamp(max=V - 1).unsqueeze(1)) / run[:, -1:]).squeeze(1)
        any_ = s["t"] > 0
        return (torch.where(any_, token, index[:, 0]).int(), torch.where(any_, count, torch.ones_like(count)).int(),
                torch.where(any_, logprob, torch.zeros_like(logprob)).float())
    _, t, rows = _sizes(case)
    L, G, r, k = case["most"], case["slices"], case["rank"], case["k"]
    x, ids = s["x"].float(), s["ids"]
    mine = (ids.unsqueeze(1) == torch.arange(L, device=x.device)).float() * s["scale"]                # [t, L]
    a, b = s["a"][:, :, :r, :k].float(), s["b"][:, :, :r].float()
    h = (x @ a.reshape(L * G * r, k).t()).view(t, L, G, r) * mine.view(t, L, 1, 1)
    parts = torch.split(b, rows, 1)
    delta = torch.cat([h[:, :, g].reshape(t, L * r) @ parts[g].permute(0, 2, 1).reshape(L * r, rows[g]) for g in range(G)], 1)
    return (s["base"].float() + delta).to(s["base"].dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "draw":
        x, t, u, top_k, top_p, min_p = (s[n].double().cpu().numpy() for n in ("x", "t", "u", "top_k", "top_p", "min_p"))
        out, kept = np.ones((2, case["rows"]), dtype=np.int32)
        logprob = np.zeros(case["rows"])
        for i in range(case["rows"]):
            if not t[i] > 0:
                out[i] = int(np.argmax(x[i]))
                continue
            # the kept tokens from the likeliest down; only values that a draw can meet are put in order
            z = (x[i] - x[i].max()) / t[i]
            order = np.argsort(-z, kind="stable")
            if top_k[i] > 0:
                order = order[:int(top_k[i])]
            p = np.exp(z[order] - np.logaddexp.reduce(z[order]))
            if top_p[i] < 1:
                order = order[:max(1, int(np.searchsorted(np.cumsum(p), top_p[i])) + 1)]
            order = order[z[order] >= (np.log(min_p[i]) if min_p[i] > 0 else -np.inf)]
            chosen = np.sort(order)
            p = np.exp(z[chosen])
            run = np.cumsum(p)
            at = min(len(chosen) - 1, int(np.searchsorted(run, u[i] * run[-1], side="right")))
            out[i], kept[i], logprob[i] = chosen[at], len(chosen), z[chosen[at]] - np.logaddexp.reduce(z[chosen])
        return torch.from_numpy(out), torch.from_numpy(kept), torch.from_numpy(logprob)
    _, t, rows = _sizes(case)
    x, y = s["x"].double(), s["base"].double()
    a, b, scale = s["a"].double(), s["b"].double(), s["scale"].double()
    for e in range(case["most"]):
        tok = torch.nonzero(s["ids"] == e).squeeze(1)
        at = 0
        for g, n in enumerate(rows):
            y[tok, at:at + n] += scale[e] * (x[tok] @ a[e, g, :, :case["k"]].t() @ b[e, at:at + n].t())
            at += n
    return y
