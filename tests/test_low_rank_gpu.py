"""Low-rank adapters on the GPU against the formula in 64 bits.

Tolerances.  Sums are in float32.  In whatever order K products are added, each addition is off by at most one step, 2^-23 of the sum of the
magnitudes so far: a hidden value by (K + 2) 2^-23 of sum |x a|, a result by (r + 3) 2^-23 of sum |h b| beside what the hidden values bring
along, plus 2^-16 of sum |h b| where they enter the second product as two bfloat16 terms (each leaves 2^-8 of what it rounds).  Storing
rounds by half a step: 2^-8 of a bfloat16 result, 2^-24 of a float32 one.  As roundings are not all of one sign, the whole result's
relative 2-norm error must stay below 2^-8 (bfloat16) or 2^-16 (float32) too."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _ops():
    from prism_b200 import ops
    return ops


def stack(L, rows, K, rank, dtype, seed, ranks=None):
    """A ``LowRank`` of random adapters with ranks up to ``rank``, and its parts in 64 bits."""
    ops = _ops()
    g = torch.Generator().manual_seed(seed)
    low = ops.LowRank.empty(L, rank, rows, K, dtype, DEV)
    for e in range(L):
        r = rank if ranks is None else ranks[e]
        low.put(e, [((torch.randn(r, K, generator=g) * K ** -0.5).to(dtype), (torch.randn(n, r, generator=g) * r ** -0.5).to(dtype)) for n in rows],
                0.25 + e % 3)
    return low


def plain(x, low, ids, base):
    """``(result, bound on the float32 sums' error)`` in 64 bits."""
    x, a, b, scale = x.double(), low.a.double(), low.b.double(), low.scale.double()
    y = torch.zeros(x.shape[0], low.n, dtype=torch.float64, device=x.device) if base is None else base.double().clone()
    tol = torch.zeros_like(y)
    for e in range(low.count):
        tok = torch.nonzero(ids == e).squeeze(1)
        at = 0
        for g, n in enumerate(low.rows):
            A, B = a[e, g, :, :low.k], b[e, at:at + n]
            h = scale[e] * (x[tok] @ A.t())
            y[tok, at:at + n] += h @ B.t()
            hb = h.abs() @ B.abs().t()
            tol[tok, at:at + n] = (low.k + 2) * 2.0 ** -23 * (scale[e] * (x[tok].abs() @ A.abs().t()) @ B.abs().t()) \
                + ((low.rank + 3) * 2.0 ** -23 + (2.0 ** -16 if x.shape[0] else 0)) * hb
            at += n
    return y, tol + 2.0 ** -23 * y.abs()


def check(got, want, tol):
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).abs()
    finite = bool(torch.isfinite(got).all())
    assert finite
    over = (err - tol - half * (want.abs() + tol)).amax().item() if want.numel() else 0
    assert over <= 0, over
    if want.numel():
        assert err.norm() <= want.norm() * (2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -16)


def inputs(T, K, N, dtype, out_dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, K, generator=g) * torch.exp(0.5 * torch.randn(K, generator=g))).to(dtype).to(DEV)
    return x, torch.randn(T, N, generator=g).to(out_dtype).to(DEV)


def ids_of(runs):
    return torch.tensor([e for e, n in runs for _ in range(n)], dtype=torch.int32, device=DEV)


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32), (torch.float32, torch.bfloat16)]


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("rows,K,rank", [((64,), 64, 16), ((501, 77), 1003, 5), ((1,), 1, 1), ((130, 64, 8), 520, 33), ((896, 128, 128), 896, 128),
                                         ((3, 5, 7, 9, 2, 1, 4, 6), 40, 8)])
def test_sizes(dtype, out_dtype, rows, K, rank):
    ops = _ops()
    low = stack(4, rows, K, rank, dtype, K)
    for T, seed in ((1, 1), (2, 2), (7, 3), (64, 4), (65, 5), (200, 6)):
        x, base = inputs(T, K, sum(rows), dtype, out_dtype, seed)
        g = torch.Generator().manual_seed(seed)
        ids = torch.randint(-1, 4, (T,), generator=g).int().to(DEV)
        check(ops.low_rank(x, low, ids, base), *plain(x, low, ids, base))
        ids = torch.sort(ids).values
        for singles in (0, T // 2, T):
            check(ops.low_rank(x, low, ids, base, singles=singles), *plain(x, low, ids, base))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("runs,singles", [
    ([(0, 128)], 0), ([(2, 300)], 0), ([(0, 127), (1, 2), (2, 129)], 0), ([(1, 1), (0, 1), (-1, 1), (1, 1), (2, 130), (0, 70)], 4),
    ([(-1, 140)], 0), ([(0, 50), (-1, 100), (0, 50)], 0), ([(i % 3, 1) for i in range(130)], 0), ([(0, 5), (1, 500)], 2), ([(1, 17)], 0)])
def test_runs(dtype, runs, singles):
    ops = _ops()
    rows, K = (256, 72), 328
    low = stack(3, rows, K, 24, dtype, 5, ranks=[24, 1, 9])
    ids = ids_of(runs)
    x, base = inputs(len(ids), K, sum(rows), dtype, dtype, 9)
    want = plain(x, low, ids, base)
    got = ops.low_rank(x, low, ids, base, singles=singles)
    check(got, *want)
    assert torch.equal(got[ids < 0], base[ids < 0])              # a token without an adapter: the shared result, bit by bit
    assert torch.equal(got, ops.low_rank(x, low, ids, base, singles=singles))


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("T,singles", [(3, 3), (150, 0), (150, 20)])
def test_in_place_without_a_base_and_with_strides(dtype, out_dtype, T, singles):
    ops = _ops()
    rows, K = (65, 40), 136
    low = stack(2, rows, K, 16, dtype, 7)
    ids = ids_of([(1, 2), (-1, 1), (0, T - 3)])
    N = sum(rows)
    wide_x, wide = inputs(T, K + 24, N + 31, dtype, out_dtype, 3)
    x, base = wide_x[:, 8:8 + K], wide[:, 3:3 + N]
    want = plain(x, low, ids, base)
    check(ops.low_rank(x, low, ids, base, singles=singles), *want)
    none = ops.low_rank(x, low, ids, singles=singles)
    assert none.dtype == dtype
    check(none, *plain(x, low, ids, None))
    assert (none[2] == 0).all()
    before = wide.clone()
    assert ops.low_rank(x, low, ids, base, out=base, singles=singles) is base
    check(base, *want)
    before[:, 3:3 + N] = base
    assert torch.equal(before, wide)                              # nothing beside the columns


def test_infinities_and_nan_stay_in_their_rows():
    ops = _ops()
    low = stack(2, (96,), 72, 16, torch.bfloat16, 11)
    for T, singles in ((6, 6), (140, 0)):
        ids = ids_of([(0, 3), (-1, 1), (1, T - 4)])
        x, base = inputs(T, 72, 96, torch.bfloat16, torch.bfloat16, 13)
        clean = ops.low_rank(x, low, ids, base, singles=singles)
        x[1, 5], x[3, 7], x[4, 0] = float("nan"), float("inf"), float("inf")
        got = ops.low_rank(x, low, ids, base, singles=singles)
        same = [i for i in range(T) if i not in (1, 4)]           # row 3 has no adapter: its x is not read into anything
        assert torch.equal(got[same], clean[same])
        assert torch.isnan(got[1]).all() and not torch.isfinite(got[4]).any()


def test_numbers_outside_the_stack_add_nothing_and_are_reported():
    ops = _ops()
    low = stack(2, (64,), 64, 16, torch.bfloat16, 17)
    for T, singles in ((5, 5), (150, 0)):
        x, base = inputs(T, 64, 64, torch.bfloat16, torch.bfloat16, 19)
        ids = ids_of([(0, 2), (2, 1), (1, T - 4), (2 ** 30, 1)])
        clean = torch.where(ids < 2, ids, torch.full_like(ids, -1))
        want = ops.low_rank(x, low, clean, base, singles=singles)
        ops.check_tc_errors()
        assert torch.equal(ops.low_rank(x, low, ids, base, singles=singles), want)
        with pytest.raises(ops.KernelError, match="outside its stack"):
            ops.check_tc_errors()
        ops.check_tc_errors()


def test_tokens_are_each_their_own():
    """Singles: a token's result does not depend on its neighbours."""
    ops = _ops()
    low = stack(8, (700, 130), 500, 32, torch.bfloat16, 23)
    x, base = inputs(40, 500, 830, torch.bfloat16, torch.bfloat16, 29)
    ids = torch.randint(-1, 8, (40,), generator=torch.Generator().manual_seed(3)).int().to(DEV)
    got = ops.low_rank(x, low, ids, base)
    check(got, *plain(x, low, ids, base))


def test_captured_and_replayed_on_other_streams():
    ops = _ops()
    low = stack(4, (300, 60), 264, 16, torch.bfloat16, 31)
    for T, singles in ((8, 8), (300, 4)):
        data = [inputs(T, 264, 360, torch.bfloat16, torch.bfloat16, 40 + i) for i in range(3)]
        g = torch.Generator().manual_seed(4)
        ids = [torch.sort(torch.randint(-1, 4, (T,), generator=g).int()).values.to(DEV) for _ in range(3)]
        want = [ops.low_rank(x, low, i, b, singles=singles) for (x, b), i in zip(data, ids)]
        graphs = []
        for _ in range(2):
            xb, bb, ib = data[0][0].clone(), data[0][1].clone(), ids[0].clone()
            torch.cuda.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                out = ops.low_rank(xb, low, ib, bb, singles=singles)
            graphs.append((gr, xb, bb, ib, out, torch.cuda.Stream()))
        for pair in ((0, 1), (2, 0), (1, 2)):
            for (gr, xb, bb, ib, out, s), i in zip(graphs, pair):
                xb.copy_(data[i][0]), bb.copy_(data[i][1]), ib.copy_(ids[i])
            torch.cuda.synchronize()
            for gr, _, _, _, _, s in graphs:
                with torch.cuda.stream(s):
                    gr.replay()
            torch.cuda.synchronize()
            for (_, _, _, _, out, _), i in zip(graphs, pair):
                assert torch.equal(out, want[i])


def test_large():
    """Sizes of the 7B shape: a decode step and a portion, an adapter each."""
    ops = _ops()
    rows, K, L = (3584, 512, 512), 3584, 3
    low = stack(L, rows, K, 64, torch.bfloat16, 37)
    for runs, singles in (([(i % 4 - 1, 1) for i in range(33)], 33), ([(0, 1), (1, 400), (2, 333)], 1)):
        ids = ids_of(runs)
        x, base = inputs(len(ids), K, sum(rows), torch.bfloat16, torch.bfloat16, 41)
        check(ops.low_rank(x, low, ids, base, singles=singles), *plain(x, low, ids, base))


def test_stack_and_its_refusals():
    ops = _ops()
    low = stack(2, (64, 32), 100, 20, torch.bfloat16, 43)
    assert low.rank == 32 and low.a.shape == (2, 2, 32, 104) and low.b.shape == (2, 96, 32)
    x, base = inputs(3, 100, 96, torch.bfloat16, torch.bfloat16, 47)
    ids = ids_of([(0, 1), (1, 2)])
    low.put(1, [None, (torch.ones(3, 100, dtype=torch.bfloat16), torch.ones(32, 3, dtype=torch.bfloat16))], 0.5)
    got = ops.low_rank(x, low, ids, base)
    check(got, *plain(x, low, ids, base))
    assert torch.equal(got[1:, :64], base[1:, :64])
    E = ops.KernelError
    bad = [dict(x=x.float()), dict(x=x[:, :99]), dict(x=x.cpu()), dict(x=x.t()), dict(ids=ids.long()), dict(ids=ids[:2]), dict(ids=ids.cpu()),
           dict(base=base[:, :95]), dict(base=base.half()), dict(base=base.t().contiguous().t()), dict(out=torch.empty(3, 96, device=DEV)),
           dict(out=torch.empty(2, 96, device=DEV, dtype=torch.bfloat16)), dict(base=None, out=torch.empty(1, 96, device=DEV, dtype=torch.bfloat16).expand(3, 96)),
           dict(x=x[:, ::1].as_strided((3, 100), (1, 2)))]
    for change in bad:
        with pytest.raises(E):
            ops.low_rank(**dict(dict(x=x, low=low, ids=ids, base=base), **change))
    assert ops.low_rank(x[:0], low, ids[:0], base[:0]).shape == (0, 96)


@pytest.mark.parametrize("ids", [(-1,), (0,), (0, 1, 2, 3), (0, -1, 2)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_calls_queued_behind_each_other(ids, dtype):
    """Many calls in flight, with wide rows: every box of the shared result passes through shared memory often, in no fixed order of arrival.  The
    results of all of them are the first one's, bit by bit, as nothing in a sum depends on time."""
    from prism_b200 import ops
    T, K, n, r = 1024, 64, 37888, 16
    g = torch.Generator(device="cuda").manual_seed(7)
    a = torch.randn(4, 1, r, K, generator=g, device="cuda").bfloat16()
    b = torch.randn(4, n, r, generator=g, device="cuda").bfloat16()
    low = ops.LowRank(a, b, torch.ones(4, device="cuda"), rows=(n,))
    x = torch.randn(T, K, generator=g, device="cuda").bfloat16()
    base = torch.randn(T, n, generator=g, device="cuda").to(dtype)
    at = torch.tensor(ids, dtype=torch.int32, device="cuda").repeat(T)[:T].contiguous()
    want = ops.low_rank(x, low, at, base=base, singles=0)
    torch.cuda.synchronize()
    none = at < 0
    assert torch.equal(want[none], base[none])
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    outs = [torch.empty_like(base) for _ in range(3)]
    for i in range(60):
        ops.low_rank(x, low, at, base=base, out=outs[i % 3], singles=0)
        if i % 3 == 2:
            for o in outs:
                wrong += (o != want).sum()
                o.fill_(float("nan"))
    assert int(wrong) == 0
    ops.check_tc_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("T,n,singles", [(200, 256, 0), (200, 100, 0), (40, 256, 40), (150, 257, 10)])
def test_tokens_without_an_adapter_keep_their_bits(dtype, T, n, singles):
    ops = _ops()
    low = stack(3, (n,), 128, 16, torch.bfloat16, 5)
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(T, 128, generator=g, device=DEV).bfloat16()
    base = torch.randn(T, n, generator=g, device=DEV).to(dtype)
    base[:, ::7] = -0.0
    base[:, 3::11] = float("inf")
    for ids in (torch.arange(T) % 4 - 1, torch.full((T,), -1), torch.where(torch.arange(T) < T // 2, 1, -1)):
        ids = ids.int().to(DEV)
        out = ops.low_rank(x, low, ids, base=base, singles=singles)
        same = base.clone()
        ops.low_rank(x, low, ids, base=same, out=same, singles=singles)
        whole = torch.int16 if dtype is torch.bfloat16 else torch.int32
        none = ids < 0
        assert torch.equal(out.view(whole)[none], base.view(whole)[none]) and torch.equal(same.view(whole), out.view(whole))


@pytest.mark.parametrize("T", [5, 40, 200])
def test_one_row_for_all_tokens(T):
    ops = _ops()
    low = stack(2, (96,), 64, 16, torch.bfloat16, 6)
    x, base = inputs(T, 64, 96, torch.bfloat16, torch.bfloat16, 3)
    x = x[:1].expand(T, 64)
    ids = (torch.arange(T, device=DEV) % 3 - 1).int()
    check(ops.low_rank(x, low, ids, base=base, singles=0), *plain(x, low, ids, base))
    check(ops.low_rank(x, low, ids, base=base, singles=T), *plain(x, low, ids, base))


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("rows,K,rank", [((130, 65), 1003, 5), ((257,), 70, 100), ((96, 8, 40), 512, 128)])
@pytest.mark.parametrize("lengths", [(47,), (95,), (96,), (128,), (255,), (256,), (1, 126), (40, 1, 90, 33, 160), (300, 200)], ids=str)
def test_portions_of_every_length(dtype, out_dtype, rows, K, rank, lengths):
    """On both sides of the lengths from which portions are taken in tiles; some have no adapter, some tiles several."""
    low = stack(3, rows, K, rank, dtype, 11)
    ids = ids_of([(i % 4 - 1 if len(lengths) > 1 else 1, n) for i, n in enumerate(lengths)])
    x, base = inputs(ids.numel(), K, sum(rows), dtype, out_dtype, 12)
    check(_ops().low_rank(x, low, ids, base=base, singles=0), *plain(x, low, ids, base))


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("rows", [(18944, 18944), (20000, 136, 18000), (40001,)], ids=str)
@pytest.mark.parametrize("lengths", [(1024, 600, 424), (2048,), (5, 1100, 3, 2, 900), (1,) * 130 + (1000,)], ids=lambda v: str(len(v)))
def test_wide_results_of_many_tokens(out_dtype, rows, lengths):
    """Enough for all CTAs to share the work evenly, in parts of several tiles of tokens and slices; also with tiles of more adapters than tensor memory
    holds side by side, and columns that are no place for TMA."""
    low = stack(6, rows, 64, 16, torch.bfloat16, 21)
    ids = ids_of([(i % 7 - 1 if len(lengths) > 1 else 1, n) for i, n in enumerate(lengths)])
    x, base = inputs(ids.numel(), 64, sum(rows), torch.bfloat16, out_dtype, 22)
    want, tol = plain(x, low, ids, base)
    got = _ops().low_rank(x, low, ids, base=base, singles=0)
    check(got, want, tol)
    none = ids < 0
    assert torch.equal(got[none], base[none])
    for _ in range(3):
        again = _ops().low_rank(x, low, ids, base=base, singles=0)
        assert torch.equal(again, got)
    _ops().check_tc_errors()


@pytest.mark.parametrize("rows,rank", [((64, 130), 64), ((200, 64, 64, 8), 64), ((64, 40, 200), 128), ((16,) * 8, 64), ((72,) * 4, 128), ((128,), 16)], ids=str)
@pytest.mark.parametrize("T", [1900, 2200, 5000])
def test_hidden_values_of_many_tiles(rows, rank, T):
    """Up to 512 hidden values a token, more clusters than run at a time, one and two CTAs an SM; calls behind each other, with tiles of several adapters."""
    ops = _ops()
    low = stack(5, rows, 320, rank, torch.bfloat16, 31)
    x, base = inputs(T, 320, sum(rows), torch.bfloat16, torch.float32, 32)
    at = torch.arange(T, device=DEV)
    several = [(at * 7 // T - 1).clamp(max=4).int(), (at // 50 % 6 - 1).int(), torch.zeros_like(at).int()]
    outs = [ops.low_rank(x, low, ids, base=base, singles=0) for _ in range(4) for ids in several]
    for i, ids in enumerate(several):
        check(outs[i], *plain(x, low, ids, base))
        for other in outs[i + 3::3]:
            assert torch.equal(outs[i], other)
    ops.check_tc_errors()
