"""Filtered draws on the GPU against the definition, row by row in 64 bits with numpy.

Tokens and counts are compared for equality.  Both sides decide in 64 bits: a draw or a cut would have to fall within about 1e-12 of
a border of two tokens to come out differently, 1e-7 a row for the largest rows here.  A logarithm of a probability is rounded once to
float32: half a step of it, 2^-24 of itself, beside 2^-40 for the whole-number weights."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _ops():
    from prism_b200 import ops
    return ops


def plain_row(x, t, u, k, p, m):
    """(token, kept, logprob) of one row of float32 logits, from the definition."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any():
        return 0, 0, -math.inf
    if not t > 0:
        return int(np.argmax(x)), 1, 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(x == x.max(), 0.0, (x - x.max()) / np.float64(t))
    z = np.where(np.isnan(z), -np.inf, z)
    order = np.argsort(-x, kind="stable")                # logit down, index up
    if k > 0:
        order = order[:k]
    if p < 1:
        # 80-bit sums: n roundings of 2^-53 would pass a weight at the cut of a prefix that leaves 2^-23 to 300,000 tokens
        run = np.cumsum(np.exp(z[order]), dtype=np.longdouble)
        order = order[:int(np.searchsorted(run, np.longdouble(p) * run[-1])) + 1]
    order = order[z[order] > -np.inf]
    if m > 0:
        order = order[z[order] >= math.log(min(m, 1.0))]
    chosen = np.sort(order)
    run = np.cumsum(np.exp(z[chosen]))
    at = int(np.searchsorted(run, np.float64(u) * run[-1], side="right"))
    at = min(at, len(chosen) - 1)
    return int(chosen[at]), len(chosen), float(z[chosen[at]] - math.log(run[-1]))


def draw(x, t, u, k=None, p=None, m=None, rows=None):
    R = x.shape[0]
    dev = lambda v, dt: None if v is None else torch.as_tensor(np.asarray(v), dtype=dt).to(DEV)      # noqa: E731
    out, kept = torch.full((2, R), -7, dtype=torch.int32, device=DEV)
    lp = torch.full((R,), 7.0, device=DEV)
    _ops().sample_filtered(x, dev(t, torch.float32), dev(u, torch.float32), out, dev(k, torch.int32), dev(p, torch.float32), dev(m, torch.float32),
                           dev(rows, torch.int32), kept, lp)
    return out.tolist(), kept.tolist(), lp.tolist()


def check(x, t, u, k=None, p=None, m=None):
    R = x.shape[0]
    f = lambda v, off: np.full(R, off) if v is None else np.asarray(v)                                # noqa: E731
    t32, u32 = np.asarray(t, dtype=np.float32), np.asarray(u, dtype=np.float32)
    p32, m32 = f(p, 1.0).astype(np.float32), f(m, 0.0).astype(np.float32)
    got = draw(x, t32, u32, k, None if p is None else p32, None if m is None else m32)
    xs = x.cpu().numpy()
    for i in range(R):
        tok, kept, lp = plain_row(xs[i], t32[i], u32[i], int(f(k, 0)[i]), p32[i], m32[i])
        assert (got[0][i], got[1][i]) == (tok, kept), (i, t32[i], u32[i], f(k, 0)[i], p32[i], m32[i])
        assert got[2][i] == lp or abs(got[2][i] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -40, (i, got[2][i], lp)


def logits(R, V, seed, spread=2.0, peaks=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * spread
    if peaks:
        for i in range(R):
            at = torch.randperm(V, generator=g)[:20]
            x[i, at] += torch.linspace(12, 2, 20)[:len(at)]
    return x.to(DEV)


SETTINGS = [dict(), dict(k=5), dict(k=50), dict(p=0.9), dict(p=0.37), dict(m=0.05), dict(k=50, p=0.9), dict(k=7, m=0.2), dict(p=0.8, m=0.01),
            dict(k=1000, p=0.99, m=0.001), dict(k=1), dict(p=0.0), dict(m=1.0), dict(m=3.0), dict(p=0.9999999)]


@pytest.mark.parametrize("V", [1, 2, 31, 255, 1003, 4096, 4097, 9000, 16385, 50257, 152064, 330001, 400000])
@pytest.mark.parametrize("peaks", [True, False])
def test_settings(V, peaks):
    R = len(SETTINGS)
    rng = np.random.RandomState(V % 1000 + peaks)
    x = logits(R, V, V + peaks, peaks=peaks)
    t = 0.3 + 1.5 * rng.rand(R)
    check(x, t, rng.rand(R), [s.get("k", 0) for s in SETTINGS], [s.get("p", 1.0) for s in SETTINGS], [s.get("m", 0.0) for s in SETTINGS])


@pytest.mark.parametrize("t", [0.0, -1.0, 1e-30, 1e-4, 0.01, 0.5, 4.0, 100.0, 1e30, math.inf])
def test_temperatures(t):
    R, V = 12, 5003
    rng = np.random.RandomState(3)
    x = logits(R, V, 11)
    check(x, [t] * R, rng.rand(R), rng.randint(0, 60, R), 0.3 + 0.75 * rng.rand(R), 0.02 * rng.rand(R) - 0.005)


def test_absent_settings():
    x = logits(4, 3001, 5)
    u = [0.1, 0.5, 0.9, 0.99]
    check(x, [0.8] * 4, u)
    check(x, [0.8] * 4, u, k=[3, 0, -4, 9])
    check(x, [0.8] * 4, u, p=[0.5, 1.0, 2.0, 0.9])
    check(x, [0.8] * 4, u, m=[0.5, 0.0, -1.0, 0.1])
    tok, kept, lp = draw(x, None, u)
    assert tok == x.argmax(1).tolist() and kept == [1] * 4 and lp == [0.0] * 4


@pytest.mark.parametrize("V", [300, 20000])
def test_equal_logits(V):
    """Ties go to the lowest index, in cuts as in draws."""
    R = 10
    rng = np.random.RandomState(1)
    few = torch.randint(0, 4, (R, V), generator=torch.Generator().manual_seed(9)).float().to(DEV)
    few[::2] *= -0.0                                     # zeros of both signs are one value
    k, u = [1, 2, 17, V // 3, V - 1, V, V + 5, 100, 3, 250], rng.rand(R)
    check(few, [0.7] * R, u, k)
    check(few, [0.7] * R, u, p=[0.5, 0.25, 0.3, 0.999, 0.01, 0.6, 0.1, 0.75, 0.9, 0.125])
    check(torch.full((R, V), 3.25, device=DEV), [1.0] * R, u, k, [0.5] * R)


@pytest.mark.parametrize("V", [70, 9001])
def test_masked_infinite_and_missing(V):
    x = logits(9, V, 21).cpu()
    x[0] = -math.inf                                     # nothing left
    x[1] = math.nan
    x[2, :] = -math.inf
    x[2, V // 2] = -2.5                                  # one left
    x[3, ::2] = -math.inf
    x[4, 1:] = torch.finfo(torch.float32).min            # masked by the lowest value
    x[5, :] = torch.finfo(torch.float32).min
    x[6, ::3] = math.nan
    x[7, 5], x[7, 9] = math.inf, math.inf
    x[8, 3] = 3.0e38
    x = x.to(DEV)
    u = np.linspace(0.02, 0.97, 9)
    for t in (0.0, 0.7, 3.0):
        check(x, [t] * 9, u)
        check(x, [t] * 9, u, k=[5] * 9, p=[0.9] * 9, m=[0.01] * 9)
        check(x, [t] * 9, u, k=[V - 1] * 9)
        check(x, [t] * 9, u, p=[0.999999] * 9)


def test_uniform_numbers_at_their_ends():
    R, V = 6, 6000
    x = logits(R, V, 31)
    for u in (0.0, 1 - 2.0 ** -24, 2.0 ** -24):
        check(x, [0.9] * R, [u] * R, k=[0, 1, 2, 30, 0, 500], p=[1, 1, 0.9, 1, 0.95, 0.5])
    # what is not in [0, 1) is taken as its nearer end
    a = draw(x, [0.9] * R, [-0.5] * R, k=[9] * R)
    assert a == draw(x, [0.9] * R, [0.0] * R, k=[9] * R)
    last = draw(x, [0.9] * R, [1.0] * R, k=[9] * R)
    assert last == draw(x, [0.9] * R, [math.nan] * R, k=[9] * R)
    for i in range(R):
        assert last[0][i] == x[i].topk(9).indices.max().item()


def test_rows_that_are_wanted():
    """The others' results stay, rows may have a stride and any alignment, and a row's result is its own."""
    V, R = 12345, 7
    wide = logits(R, V + 3, 41)
    x = wide[:, 1:V + 1]                                 # neither 16-byte aligned nor contiguous
    t, u, k, p = [0.8] * R, [0.05, 0.3, 0.4, 0.6, 0.7, 0.8, 0.95], [0, 40, 0, 5, 0, 300, 1], [0.9, 1, 1, 0.9, 0.5, 0.99, 1]
    check(x, t, u, k, p)
    whole = draw(x, t, u, k, p)
    some = draw(x, t, u, k, p, rows=[5, 0, 3])
    for i in range(R):
        assert tuple(s[i] for s in some) == (tuple(s[i] for s in whole) if i in (5, 0, 3) else (-7, -7, 7.0))
    for i in range(R):
        one = draw(x[i:i + 1], t[i:i + 1], u[i:i + 1], k[i:i + 1], p[i:i + 1])
        assert tuple(s[0] for s in one) == tuple(s[i] for s in whole)
    assert draw(x, t, u, k, p) == whole


def test_a_row_number_outside_the_logits_is_reported():
    ops = _ops()
    x = logits(3, 500, 1)
    got = draw(x, [0.5] * 3, [0.5] * 3, rows=[1, 3, -1])
    assert [got[0][0], got[0][2]] == [-7, -7] and got[0][1] >= 0
    with pytest.raises(ops.KernelError, match="row outside"):
        ops.check_tc_errors()
    ops.check_tc_errors()


def test_many_rows():
    R, V = 300, 2000
    rng = np.random.RandomState(5)
    check(logits(R, V, 51, peaks=False), 0.5 + rng.rand(R), rng.rand(R), rng.randint(0, 100, R), 0.7 + 0.4 * rng.rand(R), 0.05 * rng.rand(R))


def test_captured_and_replayed_on_other_streams():
    ops = _ops()
    R, V = 5, 40000
    x = [logits(R, V, 60 + i) for i in range(3)]
    u, t, k, p = (torch.tensor(v, device=DEV) for v in ([0.1, 0.3, 0.5, 0.7, 0.9], [0.6] * 5, [40] * 5, [0.95] * 5))
    k = k.int()
    want = []
    for xi in x:
        out = torch.empty(R, dtype=torch.int32, device=DEV)
        ops.sample_filtered(xi, t, u, out, k, p)
        want.append(out.tolist())
    graphs = []
    for _ in range(2):                                   # two graphs of one call, replayed side by side on streams of their own
        buf, out = x[0].clone(), torch.empty(R, dtype=torch.int32, device=DEV)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.sample_filtered(buf, t, u, out, k, p)
        graphs.append((g, buf, out, torch.cuda.Stream()))
    for a, b in ((0, 1), (2, 0), (1, 2)):
        for (g, buf, out, s), i in zip(graphs, (a, b)):
            buf.copy_(x[i])
        torch.cuda.synchronize()
        for g, _, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert graphs[0][2].tolist() == want[a] and graphs[1][2].tolist() == want[b]


def test_agrees_with_the_unfiltered_sampler_where_a_draw_is_clear():
    ops = _ops()
    R, V = 64, 30000
    x = logits(R, V, 71)
    g = torch.Generator().manual_seed(2)
    t, u = (0.5 + torch.rand(R, generator=g)).to(DEV), torch.rand(R, generator=g).to(DEV)
    a, b = torch.empty(2, R, dtype=torch.int32, device=DEV)
    ops.sample(x, t, u, a)
    ops.sample_filtered(x, t, u, b)
    # the float32 sampler's running sum is off by up to 2^-20 of the total: rows whose draw is nearer to a border may differ
    w = torch.exp((x.double() - x.double().amax(1, keepdim=True)) / t.double().unsqueeze(1))
    run = w.cumsum(1) / w.sum(1, keepdim=True)
    clear = (run - u.double().unsqueeze(1)).abs().amin(1) > 2.0 ** -18
    assert clear.sum() > R // 2 and torch.equal(a[clear], b[clear])


def test_refusals():
    ops = _ops()
    x, one = logits(2, 100, 1), torch.ones(2, device=DEV)
    out = torch.zeros(2, dtype=torch.int32, device=DEV)
    bad = [
        dict(logits=x.double()), dict(logits=x.t()), dict(logits=x[0]), dict(logits=x[:, ::2]), dict(logits=x[:, :0]), dict(u=one.double()), dict(u=one[:1]), dict(out=out.long()),
        dict(out=out.cpu()), dict(logits=x.cpu()), dict(top_k=one), dict(top_p=out), dict(min_p=one.half()), dict(kept=one), dict(logprob=out),
        dict(rows=torch.zeros(3, dtype=torch.int32, device=DEV)), dict(rows=one), dict(temperature=one.unsqueeze(0)), dict(u=None), dict(out=None),
        dict(top_k=torch.zeros(4, dtype=torch.int32, device=DEV)[::2]),
    ]
    for change in bad:
        args = dict(dict(logits=x, temperature=one, u=one * 0.5, out=out), **change)
        with pytest.raises(ops.KernelError):
            ops.sample_filtered(**args)
    ops.sample_filtered(x[:0], None, one[:0], out[:0])
    ops.sample_filtered(x, None, one, out, rows=out[:0])
    assert out.tolist() == [0, 0]


@pytest.mark.parametrize("V", [70, 9001])
def test_settings_that_are_no_numbers_and_masks_at_any_temperature(V):
    x = logits(6, V, 41)
    x[:, ::3] = -math.inf
    x[:, 1] = float("nan")
    nan = float("nan")
    # an infinite temperature makes all tokens alike, save those that are masked; a setting that is NaN is off
    check(x.to(DEV), [math.inf, math.inf, math.inf, 1.0, 1.0, 3e38], [0.0, 0.5, 1 - 2.0 ** -24, 0.3, 0.6, 0.9], k=[0, 20, 0, 0, 9, 0],
          p=[1.0, 1.0, 0.5, nan, nan, 0.7], m=[0.0, 0.0, 0.9, nan, 0.01, nan])


def test_refuses_more_than_it_takes():
    ops = _ops()
    x = torch.zeros(1, 520001, device=DEV)
    u, out = torch.zeros(1, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(ops.KernelError, match="520000"):
        ops.sample_filtered(x, None, u, out)
    x = torch.zeros(65536, 1, device=DEV)
    u, out = torch.zeros(65536, device=DEV), torch.zeros(65536, dtype=torch.int32, device=DEV)
    with pytest.raises(ops.KernelError, match="65536"):
        ops.sample_filtered(x, None, u, out)
