"""Low-rank adapters on the GPU: what is part of an adapter and what only fills up its stack, and what calls may do beside each other."""

import threading

import pytest
import torch

from test_low_rank_gpu import DEV, _ops, check, ids_of, inputs, plain, stack

pytestmark = pytest.mark.gpu


def exactly(x, low, ids, base, own):
    """The definition in 64 bits with each adapter's matrices as they are, without the stack's room: ``own[e][slice]`` is ``(A, B)`` or None."""
    y = base.double().clone()
    for e, slices in enumerate(own):
        tok = torch.nonzero(ids == e).squeeze(1)
        at = 0
        for n, ab in zip(low.rows, slices):
            if ab is not None:
                a, b = ab[0].to(DEV).double(), ab[1].to(DEV).double()
                # row by row: a matrix product may add zeros for places that are not there
                h = low.scale[e].double() * (x[tok].double().unsqueeze(1) * a).sum(2)
                y[tok, at:at + n] += (h.unsqueeze(1) * b).sum(2)
            at += n
    return y


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)], ids=str)
@pytest.mark.parametrize("T,singles", [(12, 12), (40, 40), (140, 0), (300, 0), (300, 30)])
@pytest.mark.parametrize("room", [16, 40, 128])
def test_infinities_do_not_meet_the_room_beyond_an_adapter_s_rank(dtype, out_dtype, T, singles, room):
    """An infinite activation makes an adapter's own hidden values infinite.  What lies behind its rank in the stack, and slices that it does not have, are
    not part of the formula: results are infinities there and the shared ones here, not NaN."""
    ops = _ops()
    rows, K = (72, 40, 64), 136
    g = torch.Generator().manual_seed(room)
    signs = lambda *s: torch.where(torch.rand(*s, generator=g) < 0.5, -1.0, 1.0) * (0.5 + torch.rand(*s, generator=g))          # noqa: E731
    ab = lambda r, n: ((signs(1, K).expand(r, K) * 0.25).to(dtype), (signs(n, 1).expand(n, r) * 0.5).to(dtype))                 # noqa: E731
    # of one adapter all hidden values have one sign, and a result's terms too: sums of infinities of one sign
    own = [[ab(1, 72), None, ab(2, 64)], [None, ab(5, 40), None], [None, None, None], [ab(16, 72), ab(16, 40), ab(16, 64)]]
    low = ops.LowRank.empty(4, room, rows, K, dtype, DEV)
    for e, slices in enumerate(own):
        low.put(e, slices, 0.5 + e)
    ids = ids_of([(e, 1) for e in (0, 1, 2, 3, -1)] * 2 + [(0, 1), (3, T - 11)])
    x, base = inputs(T, K, sum(rows), dtype, out_dtype, 5)
    x[5:10, 17], x[10, 3], x[T - 1, 64] = float("inf"), float("-inf"), float("inf")
    want = exactly(x, low, ids, base, own)
    got = ops.low_rank(x, low, ids, base, singles=singles)
    limits = ~torch.isfinite(want)
    assert limits[5].any() and not limits[5].all() and not limits[7].any() and not torch.isnan(want).any()
    assert torch.equal(got[limits].double(), want[limits])
    clean = x.clone()
    clean[~torch.isfinite(x)] = 0
    finite, tol = plain(clean, low, ids, base)
    rest = ~limits.any(1)
    check(got[rest], finite[rest], tol[rest])
    none = torch.zeros_like(limits)                       # slices that the row's adapter does not have
    none[(ids == 0), 72:112] = none[(ids == 1), :72] = none[(ids == 1), 112:] = none[(ids == 2)] = none[(ids < 0)] = True
    assert torch.equal(got[none], base[none])


def test_a_stack_that_is_not_filled_by_put_counts_whole():
    """A and B given, or written into an empty stack: all r rows count, until ``put`` says how many an adapter has."""
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    a, b = (torch.randn(2, 2, 16, 72, generator=g) / 8).bfloat16().to(DEV), torch.randn(2, 96, 16, generator=g).bfloat16().to(DEV)
    given = ops.LowRank(a, b, torch.ones(2, device=DEV), rows=(64, 32))
    filled = ops.LowRank.empty(2, 16, (64, 32), 72, torch.bfloat16, DEV)
    filled.a.copy_(a), filled.b.copy_(b), filled.scale.fill_(1.0)
    for T, singles in ((9, 9), (140, 0)):
        x, base = inputs(T, 72, 96, torch.bfloat16, torch.float32, 9)
        ids = (torch.arange(T, device=DEV) % 3 - 1).int()
        want, tol = plain(x, given, ids, base)
        for low in (given, filled):
            check(ops.low_rank(x, low, ids, base, singles=singles), want, tol)
    filled.put(1, [(a[1, 0, :3].cpu(), b[1, :64, :3].cpu()), None], 2.0)
    assert filled.ranks.tolist() == [[16, 16], [3, 0]]
    ids = torch.ones(9, dtype=torch.int32, device=DEV)
    x, base = inputs(9, 72, 96, torch.bfloat16, torch.float32, 9)
    check(ops.low_rank(x, filled, ids, base), *plain(x, filled, ids, base))


def test_the_first_call_of_a_thread():
    """A thread that has not called CUDA yet has no context there; memory comes from what torch keeps, so nothing before the kernels needs one."""
    ops = _ops()
    low = stack(2, (256,), 64, 16, torch.bfloat16, 1)
    ids = ids_of([(0, 100), (1, 60)])
    x, base = inputs(160, 64, 256, torch.bfloat16, torch.bfloat16, 1)
    w, few = torch.randn(256, 64, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV), x[:8].contiguous()
    calls = [lambda: ops.low_rank(x, low, ids, base, singles=0), lambda: ops.low_rank(x, low, ids, base, singles=160), lambda: ops.linear(few, w)]
    want = [call().clone() for call in calls]
    for call in calls:
        call()                                       # its result's memory is free again
    torch.cuda.synchronize()
    got = [None] * len(calls)

    def work(i):
        try:
            got[i] = calls[i]()
        except Exception as e:                       # noqa: BLE001
            got[i] = e
    for i in range(len(calls)):
        t = threading.Thread(target=work, args=(i,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.is_tensor(a), a
        assert torch.equal(a, b)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=str)
def test_threads_with_ranks_of_either_kind(out_dtype):
    """Ranks up to 64 and above want different amounts of shared memory of one kernel, whose limit belongs to the kernel and not to a call: no thread's call
    lowers it under another's.  The library's entry is called by itself, as Python's lock between calls would keep them apart."""
    ops = _ops()
    T, K, N, G = 160, 64, 256, 1
    lib, err = ops.lib(), ops.mxfp4._err_word(torch.device(DEV))
    jobs = []
    for rank in (16, 128, 64, 80):
        low = stack(2, (N,), K, rank, torch.bfloat16, rank)
        ids = ids_of([(0, 100), (1, T - 100)])
        x, base = inputs(T, K, N, torch.bfloat16, out_dtype, rank)
        want = ops.low_rank(x, low, ids, base, singles=0)
        check(want, *plain(x, low, ids, base))
        out, hidden = torch.empty_like(base), torch.empty(2 * T * G * low.rank + 2 * 2, dtype=torch.bfloat16, device=DEV)
        stream = torch.cuda.Stream()
        args = (x.data_ptr(), K, low.a.data_ptr(), low.b.data_ptr(), low.scale.data_ptr(), low.ranks.data_ptr(), ids.data_ptr(), base.data_ptr(), N,
                out.data_ptr(), N, out_dtype is torch.bfloat16, T, *low._sizes, hidden.data_ptr(), ops.num_sms(), err, stream.cuda_stream)
        jobs.append((args, want, out, (low, ids, x, base, hidden, stream)))
    torch.cuda.synchronize()
    said, start = [], threading.Barrier(len(jobs))

    def work(args):
        start.wait(30)
        said.extend(code for code in (lib.prism_low_rank_tile(*args) for _ in range(8000)) if code != 0)
    threads = [threading.Thread(target=work, args=(j[0],)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert said == [], (len(said), set(said))
    for _, want, out, _ in jobs:
        assert torch.equal(out, want)
    ops.check_tc_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("T,singles", [(65535, 65535), (65536, 65536), (70000, 70000), (131100, 131080), (66000, 65900), (70001, 3)])
def test_more_single_tokens_than_a_launch_has_room_for(dtype, T, singles):
    """How the tokens are laid out changes no result's meaning: not with more singles than one launch takes either."""
    low = stack(3, (24,), 24, 4, dtype, 3)
    x, base = inputs(T, 24, 24, dtype, dtype, 7)
    ids = (torch.arange(T, device=DEV) % 4 - 1).int()
    got = _ops().low_rank(x, low, ids, base, singles=singles)
    check(got, *plain(x, low, ids, base))
    assert torch.equal(got[ids < 0], base[ids < 0])
    again = base.clone()
    _ops().low_rank(x, low, ids, again, out=again, singles=singles)
    assert torch.equal(again, got)


@pytest.mark.parametrize("dtype,out_dtype,T", [(torch.bfloat16, torch.bfloat16, 65535 * 128 + 300), (torch.bfloat16, torch.float32, 65535 * 128 + 1),
                                               (torch.float32, torch.float32, 65535 * 32 + 300)], ids=str)
def test_more_tiles_than_a_launch_has_room_for(dtype, out_dtype, T):
    ops = _ops()
    low = stack(3, (8,), 8, 4, dtype, 3)
    g = torch.Generator(device=DEV).manual_seed(3)
    x, base = torch.randn(T, 8, generator=g, device=DEV).to(dtype), torch.randn(T, 8, generator=g, device=DEV).to(out_dtype)
    ids = (torch.arange(T, device=DEV) // 1000 % 4 - 1).int()
    got = ops.low_rank(x, low, ids, base, singles=0)
    check(got, *plain(x, low, ids, base))
    ops.check_tc_errors()


def narrow(x, low, ids, base):
    """``(result, bound)`` in 64 bits where hidden values stay in float32: any order of additions of K, r and one more products, 2^-23 of the sum of
    the magnitudes each, as in test_low_rank_gpu, but nothing for two bfloat16 terms."""
    x, a, b, scale = x.double(), low.a.double(), low.b.double(), low.scale.double()
    y = base.double().clone()
    tol = 2.0 ** -23 * y.abs()
    for e in range(low.count):
        tok = torch.nonzero(ids == e).squeeze(1)
        at = 0
        for g, n in enumerate(low.rows):
            A, B = a[e, g, :, :low.k], b[e, at:at + n]
            h = scale[e] * (x[tok] @ A.t())
            y[tok, at:at + n] += h @ B.t()
            tol[tok, at:at + n] += 2.0 ** -23 * ((low.k + 2) * (scale[e] * (x[tok].abs() @ A.abs().t()) @ B.abs().t()) + (low.rank + 4) * (h.abs() @ B.abs().t()))
            at += n
    return y, tol


@pytest.mark.parametrize("rows,K,rank", [((64,), 64, 16), ((501, 77), 1003, 5), ((130, 64, 8), 520, 33), ((896, 128, 128), 896, 128)])
@pytest.mark.parametrize("dtype,T,singles", [(torch.float32, 1, 1), (torch.float32, 40, 40), (torch.float32, 200, 200), (torch.float32, 300, 0), (torch.float32, 300, 20),
                                             (torch.bfloat16, 1, 1), (torch.bfloat16, 40, 40), (torch.bfloat16, 64, 64), (torch.bfloat16, 200, 200)], ids=str)
def test_hidden_values_keep_32_bits_off_the_tensor_cores(rows, K, rank, dtype, T, singles):
    """Beside the bound of every result the whole's relative 2-norm error stays below 2^-20: roundings of half a step, 2^-24, that are not all of one
    sign, in chains of K / 8 products at most (1,003: sqrt(125 / 3) half steps of a hidden value, 2^-21.3).  Two bfloat16 terms leave 2^-17 of a hidden value each
    and would pass neither."""
    low = stack(4, rows, K, rank, dtype, K)
    x, base = inputs(T, K, sum(rows), dtype, torch.float32, T)
    base *= 2.0 ** -6                                     # so that the adapters' part is most of the result
    ids = torch.sort(torch.randint(0, 4, (T,), generator=torch.Generator().manual_seed(T)).int()).values.to(DEV)
    want, tol = narrow(x, low, ids, base)
    err = (_ops().low_rank(x, low, ids, base, singles=singles).double() - want).abs()
    assert (err <= tol + 2.0 ** -24 * (want.abs() + tol)).all()
    assert err.norm() <= 2.0 ** -20 * want.norm()


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)], ids=str)
@pytest.mark.parametrize("T,singles", [(1, 1), (40, 40), (64, 64), (200, 0), (300, 0), (300, 40), (1000, 0)])
def test_a_token_s_bits_do_not_depend_on_its_neighbours(dtype, out_dtype, T, singles):
    """With as many tokens laid out in the same way: whatever the others' activations and adapters are, how many adapters share a tile, and beside NaN."""
    ops = _ops()
    rows, K = (700, 130, 24), 500
    low = stack(8, rows, K, 32, dtype, 23)
    x, base = inputs(T, K, sum(rows), dtype, out_dtype, 29)
    g = torch.Generator().manual_seed(T)
    ids = torch.sort(torch.randint(-1, 3, (T,), generator=g).int()).values.to(DEV)
    kept = (torch.rand(T, generator=g) < 0.3).to(DEV)
    kept[0] = True
    want = ops.low_rank(x, low, ids, base, singles=singles)
    for others in (torch.full((T,), -1), torch.full((T,), 7), torch.randint(-1, 8, (T,), generator=g), torch.arange(T) % 9 - 1):
        x2, base2 = inputs(T, K, sum(rows), dtype, out_dtype, 31)
        x2[::3] = float("nan")
        x2[kept], base2[kept] = x[kept], base[kept]
        ids2 = torch.where(kept, ids, others.int().to(DEV))
        got = ops.low_rank(x2, low, ids2, base2, singles=singles)
        assert torch.equal(got[kept], want[kept])
