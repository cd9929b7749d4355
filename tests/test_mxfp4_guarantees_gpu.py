"""What the 4-bit operators promise beyond their values at ordinary inputs: how far an expert's hidden values are held; that a
wait that runs out is an error and nothing else; that no kernel runs in a workspace that is too small for it; that an experts' layer is right on any
number of SMs; that threads and streams do not disturb one another.

Tolerances.  A product's float32 sum is within 2^-18 of the sum of |x w| of the 64-bit one (``test_mxfp4_gpu``)."""

import ctypes
import threading

import pytest
import torch

from test_mxfp4_gpu import DEV, _acts, _check_linear, _experts, _gen, _ops, decode, plain_moe

pytestmark = pytest.mark.gpu

SUM = 2.0 ** -18


@pytest.mark.parametrize("T,E,F,H", [(1, 2, 32, 64), (5, 3, 100, 256), (16, 2, 672, 700), (20, 2, 130, 256), (64, 2, 200, 256), (64, 1, 256, 512), (64, 16, 64, 128)])
def test_hidden_values_keep_fourteen_bits(T, E, F, H):
    """One choice of weight 1 a token, and down products that each read one hidden value: so the result shows what is
    held of it, 2^-14 of itself and 2^-27 of the largest of its block of 32 (two 8-bit terms would hold 2^-9).  Beside that
    only the errors of g and u, through silu (slope below 1.1) and the product."""
    ops = _ops()
    x = _acts(T, H, T + F)
    router = (_acts(E, H, 4) * H ** -0.5).to(torch.bfloat16)
    gate, up, _ = _experts(E, F, H, F)
    sparse = torch.zeros(E, H, F)
    sparse[:, torch.arange(H), torch.arange(H) % F] = torch.where(torch.rand(E, H, generator=_gen(3)) < 0.5, -1.0, 1.0)
    down = ops.mxfp4_quantize(sparse.to(DEV))
    assert torch.equal(down.dequantize(torch.float32).cpu(), sparse)
    got = ops.mxfp4_moe(x, router, gate, up, down, 1, True, True, False, out_dtype=torch.float32).double()
    pick = torch.argsort(-torch.softmax(x.double() @ router.double().t(), -1), dim=1, stable=True)[:, 0]
    for t in range(T):
        e, a = int(pick[t]), x[t].double()
        wg, wu = decode(gate[e]).to(DEV), decode(up[e]).to(DEV)
        g, u = wg @ a, wu @ a
        eg, eu = (wg.abs() @ a.abs()) * SUM, (wu.abs() @ a.abs()) * SUM
        s = torch.nn.functional.silu(g)
        h = s * u
        block = torch.nn.functional.pad(h.abs(), (0, -F % 32)).view(-1, 32).amax(1).repeat_interleave(32)[:F]
        bound = h.abs() * (2.0 ** -14 + 2.0 ** -20) + block * 2.0 ** -27 + 1.1 * eg * (u.abs() + eu) + s.abs() * eu
        at = torch.arange(H, device=DEV) % F
        far = (got[t] - sparse[e, torch.arange(H), at.cpu()].to(DEV).double() * h[at]).abs() - bound[at]
        assert (far <= 0).all(), (t, far.max().item(), (far > 0).double().mean().item())


def _moe_args(T, H=256, F=200, E=6, seed=1):
    router = (_acts(E, H, 4) * H ** -0.5).to(torch.bfloat16)
    return (_acts(T, H, seed), router, *_experts(E, F, H, 2), 2, True, True, False)


@pytest.mark.parametrize("T", [1, 12, 40])
def test_a_wait_that_runs_out_leaves_no_result_and_no_trace(T):
    """One arrival short at the barrier behind the router: every block gives up after the wait's limit, the result stays
    untouched, the error is raised once, and the next call is right."""
    ops = _ops()
    args = _moe_args(T)
    want = ops.mxfp4_moe(*args)
    out = torch.full_like(want, 7.0)
    torch.cuda.synchronize()
    control = ops.mxfp4._streams[(torch.cuda.current_device(), ops._stream())].counters
    assert not control.any()
    control[0] = -1
    ops.mxfp4_moe(*args, out=out)
    torch.cuda.synchronize()
    with pytest.raises(ops.KernelError, match="wait"):
        ops.check_tc_errors()
    assert (out == 7).all() and not control.any()
    assert torch.equal(ops.mxfp4_moe(*args), want)
    ops.check_tc_errors()


@pytest.mark.parametrize("M,act_bits", [(1, 16), (8, 4), (40, 16), (300, 4), (300, 16)])
def test_a_product_s_workspace_that_is_too_small_is_refused(M, act_bits):
    ops = _ops()
    N, K = 700, 2000
    x, w, out = _acts(M, K, 1), ops.mxfp4_quantize(_acts(N, K, 2)), torch.full((M, N), 7.0, device=DEV)
    need = (ctypes.c_longlong * 2)()
    assert ops.lib().prism_mxfp4_linear_workspace(M, N, K, act_bits, ctypes.addressof(need)) == 0
    work, counters = torch.empty(need[0], dtype=torch.uint8, device=DEV), torch.zeros(4096, dtype=torch.int32, device=DEV)

    def call(nbytes):
        return ops.lib().prism_mxfp4_linear(work.data_ptr(), nbytes, counters.data_ptr(), x.data_ptr(), K, w.codes.data_ptr(), w.scales.data_ptr(), None, 0, out.data_ptr(), ops.F32, N, M, N, K, act_bits,
                                            ops._tc_err_word(x.device).data_ptr(), ops._stream())
    assert call(need[0] - 1) == call(0) == -1
    torch.cuda.synchronize()
    assert (out == 7).all()
    assert need[1] == (6 if M <= 8 else 0) and call(need[0]) == 0
    assert torch.equal(out, ops.mxfp4_linear(x, w, out_dtype=torch.float32, act_bits=act_bits))


def test_workspaces_grow_with_the_calls():
    """A stream's first call is small and a later one needs more than the stream has, or more than it keeps."""
    ops = _ops()
    side = torch.cuda.Stream()
    for M, N, K in ((1, 200, 300), (400, 2100, 1200), (2048, 1024, 8192), (1, 200, 300)):
        x, w = _acts(M, K, 1), ops.mxfp4_quantize(_acts(N, K, 2))
        want = ops.mxfp4_linear(x, w)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = ops.mxfp4_linear(x, w)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        assert all(own.work.numel() <= ops.mxfp4._SCRATCH for own in ops.mxfp4._streams.values())
    args = _moe_args(64, 2048, 1024, 8)
    assert torch.equal(ops.mxfp4_moe(*args), ops.mxfp4_moe(*args))


@pytest.mark.parametrize("ctas", [1, 5, 16, 60])
@pytest.mark.parametrize("T,E,F,H,top", [(64, 40, 40, 200, 3), (64, 6, 70, 256, 2), (33, 1, 33, 96, 1), (7, 9, 200, 130, 4)])
def test_fewer_blocks_than_tokens_choose_for_every_token(ctas, T, E, F, H, top, monkeypatch):
    """As on a part of a GPU: a block then has the logits of more than two tokens, one share after another."""
    ops = _ops()
    x, router = _acts(T, H, T), (_acts(E, H, 4) * H ** -0.5).to(torch.bfloat16)
    gate, up, down = _experts(E, F, H, 2)
    dv = [decode(w).to(DEV) for w in (gate, up, down)]
    want, bound = plain_moe(x, router, *dv, top, True, True, False)
    monkeypatch.setattr(ops.mxfp4, "MOE_CTAS", ctas)
    got = ops.mxfp4_moe(x, router, gate, up, down, top, True, True, False, out_dtype=torch.float32)
    ops.check_tc_errors()
    assert ((got.double() - want).abs() <= bound * 2.0 ** -8).all()
    choice = ops.MoeChoice(None, 2, 1) if E % 2 == 0 and E // 2 >= top else None
    if choice is not None:
        want, bound = plain_moe(x, router, *dv, top, False, False, True, choice=choice)
        got = ops.mxfp4_moe(x, router, gate, up, down, top, False, False, True, choice=choice, out_dtype=torch.float32)
        assert ((got.double() - want).abs() <= bound * 2.0 ** -8).all()


@pytest.mark.parametrize("M,act_bits", [(64, 16), (200, 16), (64, 4), (200, 4), (3, 16)])
def test_two_threads_on_one_stream(M, act_bits):
    """Threads that share the default stream get the bits of their own inputs, whatever the order of their launches."""
    ops = _ops()
    w = ops.mxfp4_quantize(_acts(1500, 2100, 2))
    xs = [_acts(M, 2100, 30 + i) for i in range(2)]
    want = [ops.mxfp4_linear(x, w, act_bits=act_bits) for x in xs]
    got = [[], []]

    def work(i):
        for _ in range(200):
            got[i].append(ops.mxfp4_linear(xs[i], w, act_bits=act_bits))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    ops.check_tc_errors()
    for i in range(2):
        assert len(got[i]) == 200 and all(torch.equal(y, want[i]) for y in got[i])


def test_two_streams_at_once():
    """Different inputs on two streams with no wait between them: the bits of each alone."""
    ops = _ops()
    streams = [torch.cuda.Stream() for _ in range(2)]
    w = ops.mxfp4_quantize(_acts(1500, 2100, 2))
    cases = [[(_acts(M, 2100, 10 * i + M), bits) for M in (1, 9, 64, 200) for bits in (16, 4)] for i in range(2)]
    want = [[ops.mxfp4_linear(x, w, act_bits=b) for x, b in c] for c in cases]
    args = [[_moe_args(T, seed=50 + i) for T in (1, 12, 40)] for i in range(2)]
    layers = [[ops.mxfp4_moe(*a) for a in c] for c in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(([ops.mxfp4_linear(x, w, act_bits=b) for x, b in cases[i]], [ops.mxfp4_moe(*a) for a in args[i]]))
    torch.cuda.synchronize()
    ops.check_tc_errors()
    for i in range(2):
        for products, moes in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(products, want[i])) and all(torch.equal(a, b) for a, b in zip(moes, layers[i]))


@pytest.mark.parametrize("T", [1, 16, 33, 64])
def test_a_layer_of_experts_replays_and_repeats(T):
    """The same bits again, among other calls and from a captured graph, whose inputs may change between replays."""
    ops = _ops()
    args = _moe_args(T, 512, 300, 9)
    want = ops.mxfp4_moe(*args)
    other = (_acts(T, 512, 99),) + args[1:]
    want_other = ops.mxfp4_moe(*other)
    assert not torch.equal(want, want_other)
    x = args[0].clone()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        y = ops.mxfp4_moe(x, *args[1:])
        z = ops.mxfp4_moe(x, *args[1:])
    for i in range(6):
        assert torch.equal(ops.mxfp4_moe(*args), want)
        x.copy_(other[0] if i % 2 else args[0])
        g.replay()
        g.replay()
        assert torch.equal(y, want_other if i % 2 else want) and torch.equal(z, y)
    ops.check_tc_errors()


def test_graphs_of_two_streams_at_once():
    """Two captured steps of several calls, replayed on two streams with no wait between them."""
    ops = _ops()
    w = ops.mxfp4_quantize(_acts(1500, 2100, 2))
    steps = []
    for i in range(2):
        xs, layer = [_acts(M, 2100, 10 * i + M) for M in (1, 64)], _moe_args(12, seed=40 + i)
        want = [ops.mxfp4_linear(x, w, act_bits=b) for x in xs for b in (16, 4)] + [ops.mxfp4_moe(*layer)]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = [ops.mxfp4_linear(x, w, act_bits=b) for x in xs for b in (16, 4)] + [ops.mxfp4_moe(*layer)]
        steps.append((g, torch.cuda.Stream(), got, want, xs, layer))
    torch.cuda.synchronize()
    for _ in range(30):
        for g, stream, *_ in steps:
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    ops.check_tc_errors()
    assert all(torch.equal(a, b) for _, _, got, want, *_ in steps for a, b in zip(got, want))


@pytest.mark.parametrize("T,E,top,H,F", [(64, 256, 16, 128, 32), (64, 16, 16, 96, 40), (1, 256, 16, 200, 64), (64, 256, 1, 64, 33), (64, 64, 16, 1003, 31)])
def test_the_most_experts_and_choices(T, E, top, H, F):
    ops = _ops()
    x, router = _acts(T, H, T), (_acts(E, H, 4) * H ** -0.5).to(torch.bfloat16)
    gate, up, down = _experts(E, F, H, 2)
    want, bound = plain_moe(x, router, *[decode(w).to(DEV) for w in (gate, up, down)], top, True, True, False)
    got = ops.mxfp4_moe(x, router, gate, up, down, top, True, True, False, out_dtype=torch.float32)
    assert ((got.double() - want).abs() <= bound * 2.0 ** -8).all()


@pytest.mark.parametrize("M", [1, 16, 40, 200])
@pytest.mark.parametrize("below", [6, 13, 18, 21])
def test_activations_far_below_their_block_s_largest(M, below):
    """Every block of x holds one large value, which meets weights of zero, and values some 2^-``below`` of it: these are read
    exactly down to 2^-14 of the largest and to within 2^-22 of it below."""
    ops = _ops()
    N, K = 200, 640
    g = _gen(M + below)
    x = (torch.rand(M, K, generator=g) * 2 + 2) * 2.0 ** -below * torch.where(torch.rand(M, K, generator=g) < 0.5, -1.0, 1.0)
    x[:, ::32] = 1 + torch.rand(M, K // 32, generator=g)
    x = x.to(torch.bfloat16).to(DEV)
    wf = torch.randn(N, K, generator=g)
    wf[:, ::32] = 0
    w = ops.mxfp4_quantize(wf.to(DEV))
    wv = decode(w).to(DEV)
    want = x.double() @ wv.t()
    small = torch.ones(K, dtype=torch.float64, device=DEV)
    small[::32] = 0
    bound = (x.double().abs() * small) @ wv.abs().t() * SUM
    if below > 13:
        bound = bound + x.double()[:, ::32].abs().repeat_interleave(32, 1) @ wv.abs().t() * 2.0 ** -22
    far = (ops.mxfp4_linear(x, w, out_dtype=torch.float32).double() - want).abs() - bound
    assert (far <= 0).all(), (far.max().item(), (far > 0).double().mean().item())


@pytest.mark.parametrize("N", [4096 * 128, 4096 * 128 + 1])
@pytest.mark.parametrize("act_bits", [16, 4])
def test_as_many_rows_as_the_stream_s_counters_and_one_more(N, act_bits):
    """Beyond 4,096 tiles a few tokens go through the form of many."""
    ops = _ops()
    x, w = _acts(2, 40, 1), ops.mxfp4_quantize(_acts(N, 40, 2))
    got = ops.mxfp4_linear(x, w, act_bits=act_bits)
    at = torch.cat([torch.arange(300), torch.arange(N - 300, N)]).to(DEV)
    few = ops.mxfp4_quantize(_acts(N, 40, 2)[at])
    assert torch.equal(got[:, at], ops.mxfp4_linear(x, few, act_bits=act_bits))
    _check_linear(x, few, None, act_bits, got=got[:, at].contiguous())


def test_results_whose_rows_overlap_are_refused():
    ops = _ops()
    x, w, stack = _acts(4, 200, 1), ops.mxfp4_quantize(_acts(96, 200, 2)), ops.mxfp4_quantize(torch.stack([_acts(8, 64, i) for i in range(3)]))
    line = torch.empty(4 * 300, dtype=torch.bfloat16, device=DEV)
    layer = _moe_args(4, 256)
    for call in (lambda: ops.mxfp4_linear(x, w, out=line[:96].expand(4, 96)), lambda: ops.mxfp4_linear(x, w, out=line.as_strided((4, 96), (95, 1))),
                 lambda: stack.dequantize(out=line[:512].view(1, 8, 64).expand(3, 8, 64)), lambda: stack.dequantize(out=line.as_strided((3, 8, 64), (256, 64, 1))),
                 lambda: ops.mxfp4_moe(*layer, out=line[:256].expand(4, 256)), lambda: ops.mxfp4_moe(*layer, out=line.as_strided((4, 256), (128, 1)))):
        with pytest.raises(ops.KernelError):
            call()
    one = line.as_strided((1, 96), (1, 1))                         # a single row's stride says nothing
    assert torch.equal(ops.mxfp4_linear(x[:1], w, out=one), ops.mxfp4_linear(x[:1], w))


@pytest.mark.parametrize("T", [16, 40, 64])
def test_a_token_that_is_not_a_number_among_many(T):
    """It is a row of NaN, and the other tokens' bits are as without it (every expert has tokens either way)."""
    ops = _ops()
    x, *rest = _moe_args(T, 256, 96, 2)
    clean = ops.mxfp4_moe(x, *rest)
    y = x.clone()
    y[5, 200], y[T - 1, 0] = float("nan"), float("inf")
    got = ops.mxfp4_moe(y, *rest)
    keep = [t for t in range(T) if t not in (5, T - 1)]
    assert torch.isnan(got[[5, T - 1]]).all() and torch.equal(got[keep], clean[keep])
