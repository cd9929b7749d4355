"""Microscaled 4-bit floating point on the GPU: quantisation, products and the experts' layer against plain implementations
in 64 bits.

Tolerances.  Quantisation is exact: the codes' values are compared for equality.  A product's float32 sum differs from the
64-bit one by its roundings: at most K * 2^-24 of the sum of |x w| if every addition rounded the worst way, taken as 2^-18 of
it for the rows here (K up to 5,000: a random walk of K roundings is below 80 * 2^-24; and the tensor cores may drop bits of
a 32-wide partial sum, 2^-21 of its largest term); a bfloat16 result adds 2^-9 of itself.  16-bit activations are read to
within 2^-22 of their block's largest, which the same bound covers.  In the experts' layer the hidden values are rounded to 8
significant bits (2^-9 each), so its bound is 2^-8 of the sum of |h w| beside the result's own rounding."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _ops():
    from prism_b200 import ops
    return ops


def _gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def _acts(m, k, seed, dtype=torch.bfloat16):
    g = _gen(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g))
    return x.to(dtype).to(DEV)


def plain_quantise(x):
    """The values (float64, on the CPU) that the rows of ``x`` are brought to, element by element from the definition."""
    x = x.detach().cpu().double()
    out = torch.empty_like(x)
    for at in range(0, x.shape[-1], 32):
        b = x[..., at:at + 32]
        bad = ~torch.isfinite(b).all(-1)
        most = torch.where(torch.isfinite(b), b, torch.zeros_like(b)).abs().amax(-1)
        e = torch.tensor([max(math.frexp(v)[1] - 3, -127) if v > 0 else -127 for v in most.flatten().tolist()], dtype=torch.float64)
        scale = torch.exp2(e).view(most.shape).unsqueeze(-1)
        v = b.abs() / scale
        near = torch.zeros_like(v)
        dist = v.clone()
        for i, q in enumerate(GRID[1:], 1):
            d = (v - q).abs()
            take = (d < dist) | ((d == dist) & (i % 2 == 0))
            near, dist = torch.where(take, torch.full_like(v, q), near), torch.where(take, d, dist)
        val = torch.sign(b) * near * scale
        out[..., at:at + 32] = torch.where(bad.unsqueeze(-1), torch.full_like(val, float("nan")), val)
    return out


def decode(q):
    """The values of an ``Mxfp4``'s bytes (float64, on the CPU), by the format's definition."""
    codes, scales = q.codes.cpu(), q.scales.cpu()
    N, K = q.shape[-2:]
    flat_c, flat_s = codes.view(-1, N, codes.shape[-1]), scales.view(-1, scales.shape[-3], scales.shape[-2], 512)
    out = torch.empty(flat_c.shape[0], N, K, dtype=torch.float64)
    grid = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64)
    r, b = torch.arange(N), torch.arange(-(-K // 32))
    byte = (r % 32 * 16 + r % 128 // 32 * 4).unsqueeze(1) + (b % 4).unsqueeze(0)
    for m in range(flat_c.shape[0]):
        c = torch.stack((flat_c[m] & 15, flat_c[m] >> 4), -1).flatten(1)[:, :K].long()
        s = flat_s[m][(r // 128).unsqueeze(1), (b // 4).unsqueeze(0), byte].double()
        s = torch.where(s == 255, torch.full_like(s, float("nan")), torch.exp2(s - 127))
        out[m] = grid[c] * s.repeat_interleave(32, 1)[:, :K]
    return out.view(*q.shape[:-2], N, K)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


# ---- quantisation ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (3, 31), (5, 33), (127, 128), (129, 130), (40, 1000), (300, 1003), (2, 5000)])
def test_quantise_is_the_definition(rows, K, dtype):
    ops = _ops()
    x = _acts(rows, K, rows * 1000 + K, dtype)
    q = ops.mxfp4_quantize(x)
    want = plain_quantise(x)
    assert same(decode(q), want)
    for dt in (torch.bfloat16, torch.float32):
        got = q.dequantize(dt)
        assert got.dtype == dt and same(got.cpu().double(), want)
    assert not q.codes.view(rows, -1)[:, (K + 31) // 32 * 16:].any()          # zero beyond K


def test_quantise_special_blocks():
    ops = _ops()
    x = torch.zeros(8, 96)
    x[0, :32] = torch.linspace(-7.99, 7.99, 32)                # saturates above 6
    x[0, 40] = 2.0 ** -140                                     # the smallest exponents
    x[0, 70] = -2.0 ** -126
    x[1, 3] = float("nan")
    x[1, 40] = float("inf")
    x[2, 0], x[2, 1] = 3.3e38, -1.0
    x[3, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 4.0])   # ties
    x = x.to(DEV)
    q = ops.mxfp4_quantize(x)
    want = plain_quantise(x)
    assert same(decode(q), want) and same(q.dequantize(torch.float32).cpu().double(), want)
    assert torch.isnan(q.dequantize()[1, :64]).all() and not torch.isnan(q.dequantize()[1, 64:]).any()


def test_quantise_strides_and_stacks():
    ops = _ops()
    wide = _acts(37, 1000, 5)
    for view in (wide[:, 3:300], wide[:, 8:264], wide[::2, 16:80]):
        assert same(decode(ops.mxfp4_quantize(view)), plain_quantise(view))
    stack = torch.stack([_acts(130, 200, s) for s in range(3)])
    q = ops.mxfp4_quantize(stack)
    assert same(decode(q), plain_quantise(stack)) and same(decode(q[1]), plain_quantise(stack[1]))
    assert same(q.dequantize().cpu().double(), plain_quantise(stack))


# ---- products ------------------------------------------------------------------------------------------------------------

def _check_linear(x, w, bias, act_bits, out_dtype=torch.bfloat16, got=None):
    ops = _ops()
    got = ops.mxfp4_linear(x, w, bias, out_dtype=out_dtype, act_bits=act_bits) if got is None else got
    xv = plain_quantise(x) if act_bits == 4 else x.cpu().double()
    wv = decode(w)
    want = xv.to(DEV) @ wv.to(DEV).t()
    bound = (xv.abs().to(DEV) @ wv.abs().to(DEV).t()) * 2.0 ** -18
    if bias is not None:
        want = want + bias.double()
    if out_dtype == torch.bfloat16:
        bound = bound + want.abs() * 2.0 ** -8
    assert got.dtype == out_dtype
    far = (got.double() - want).abs() - bound
    assert (far <= 1e-30).all(), (tuple(x.shape), tuple(w.shape), act_bits, far.max().item(), (far > 0).float().mean().item())


@pytest.mark.parametrize("act_bits", [16, 4])
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 1), (1, 128, 128), (1, 4608, 3584), (2, 130, 260), (7, 1000, 1003), (8, 9728, 896), (15, 77, 33), (16, 3584, 4992), (17, 256, 512),
    (31, 127, 640), (32, 512, 2048), (33, 300, 96), (64, 1001, 1280), (65, 384, 384), (100, 129, 1000), (128, 2048, 256), (129, 640, 1003),
    (256, 256, 4096), (300, 1111, 700), (1000, 500, 2176)])
def test_linear(M, N, K, act_bits):
    ops = _ops()
    x = _acts(M, K, M + N)
    w = ops.mxfp4_quantize(_acts(N, K, K + 1))
    bias = _acts(1, N, 3)[0] if (M + N) % 2 else None
    _check_linear(x, w, bias, act_bits)
    if M in (1, 16, 33, 129):
        _check_linear(x, w, bias if bias is None else bias.float(), act_bits, torch.float32)


@pytest.mark.parametrize("act_bits", [16, 4])
@pytest.mark.parametrize("M", [1, 5, 40, 200])
def test_linear_strides(M, act_bits):
    """Rows with strides of their own, unaligned starts, an output that is a column block of a wider buffer."""
    ops = _ops()
    base = _acts(M + 1, 1100, 9)
    w = ops.mxfp4_quantize(_acts(200, 500, 10))
    for x in (base[:M, 3:503], base[1:, 8:508], base[:M, 600:1100]):
        buf = torch.full((M, 260), 7.0, dtype=torch.bfloat16, device=DEV)
        got = ops.mxfp4_linear(x, w, None, out=buf[:, 30:230], act_bits=act_bits)
        _check_linear(x, w, None, act_bits, got=got)
        assert (buf[:, :30] == 7).all() and (buf[:, 230:] == 7).all()


@pytest.mark.parametrize("act_bits", [16, 4])
@pytest.mark.parametrize("M", [3, 90])
def test_linear_special_values(M, act_bits):
    """A row of x with an infinity or NaN is NaN and the others are as without it; a weight's NaN block reaches its output only;
    blocks whose values are far apart; rows of zeros."""
    ops = _ops()
    x = _acts(M, 320, 1)
    x[:, 64:96] *= 2.0 ** -60
    x[:, 96:128] *= 2.0 ** 40
    x[2] = 0
    wf = _acts(200, 320, 2, torch.float32)
    wf[:, 96:128] *= 2.0 ** -40
    w = ops.mxfp4_quantize(wf)
    _check_linear(x, w, None, act_bits)
    clean = ops.mxfp4_linear(x, w, act_bits=act_bits)
    assert not clean[2].any()
    y = x.clone()
    y[0, 5], y[1, 300] = float("nan"), float("-inf")
    got = ops.mxfp4_linear(y, w, act_bits=act_bits)
    assert torch.isnan(got[:2]).all() and torch.equal(got[2:], clean[2:])
    wf[7, 40] = float("inf")
    got = ops.mxfp4_linear(x, ops.mxfp4_quantize(wf), act_bits=act_bits)
    assert torch.isnan(got[:, 7]).all()
    keep = [i for i in range(200) if i != 7]
    assert torch.equal(got[:, keep], clean[:, keep])


@pytest.mark.parametrize("act_bits", [16, 4])
@pytest.mark.parametrize("M,N,K", [(1, 2000, 3000), (16, 700, 9000), (50, 4000, 1500), (400, 2100, 1200)])
def test_linear_repeats_bit_for_bit(M, N, K, act_bits):
    """The same bits again, alone, among other work and on another stream."""
    ops = _ops()
    x, w = _acts(M, K, 1), ops.mxfp4_quantize(_acts(N, K, 2))
    want = ops.mxfp4_linear(x, w, act_bits=act_bits)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for i in range(6):
        other = ops.mxfp4_linear(_acts(M, K, 50 + i), w, act_bits=act_bits)
        assert torch.equal(ops.mxfp4_linear(x, w, act_bits=act_bits), want)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = ops.mxfp4_linear(x, w, act_bits=act_bits)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(again, want) and other.shape == want.shape


def test_linear_in_a_graph():
    ops = _ops()
    w = ops.mxfp4_quantize(_acts(900, 1280, 2))
    for M in (1, 16, 60, 200):
        for act_bits in (16, 4):
            x = _acts(M, 1280, 1)
            ops.mxfp4_linear(x, w, act_bits=act_bits)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = ops.mxfp4_linear(x, w, act_bits=act_bits)
            x.copy_(_acts(M, 1280, 77))
            g.replay()
            g.replay()
            torch.cuda.synchronize()
            _check_linear(x, w, None, act_bits, got=y)


# ---- the experts' layer ------------------------------------------------------------------------------------------------

def plain_moe(x, router, gate, up, down, top, softmax, renorm, scale_input, act="silu", limit=0.0, bias=None, choice=None):
    """``(result, bound)`` in float64: the bound is the sum of |h w| of the down products."""
    x, z = x.double(), x.double() @ router.double().t()
    if bias is not None:
        z = z + bias.double()
    s = torch.softmax(z, -1) if softmax else torch.sigmoid(z)
    c = s.clone() if choice is None or choice.correction is None else s + choice.correction.double()
    if choice is not None and choice.keep < choice.groups:
        per = c.shape[1] // choice.groups
        best = c.view(-1, choice.groups, per).amax(-1)
        kept = torch.zeros_like(best).scatter(1, torch.argsort(-best, dim=1, stable=True)[:, :choice.keep], 1.0)
        c = torch.where(kept.repeat_interleave(per, 1) > 0, c, torch.full_like(c, -math.inf))
    pick = torch.argsort(-c, dim=1, stable=True)[:, :top]
    w = s.gather(1, pick)
    if renorm:
        w = w / (w.sum(1, keepdim=True) + (0 if choice is None else choice.sum_eps))
    if choice is not None:
        w = w * choice.scale
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    for e in range(router.shape[0]):
        t, j = torch.nonzero(pick == e, as_tuple=True)
        if not t.numel():
            continue
        a = x[t] * w[t, j].unsqueeze(1) if scale_input else x[t]
        g, u = a @ gate[e].t(), a @ up[e].t()
        if act == "silu":
            h = torch.nn.functional.silu(g) * u
        elif act == "gelu_tanh":
            h = torch.nn.functional.gelu(g, approximate="tanh") * u
        else:
            gc = g.clamp(max=limit)
            h = gc * torch.sigmoid(1.702 * gc) * (u.clamp(-limit, limit) + 1)
        if not scale_input:
            h = h * w[t, j].unsqueeze(1)
        y[t] += h @ down[e].t()
        bound[t] += h.abs() @ down[e].abs().t()
    return y, bound


def _experts(E, F, H, seed):
    ops = _ops()
    g = _gen(seed)
    mk = lambda *s: ops.mxfp4_quantize((torch.randn(*s, generator=g) * s[-1] ** -0.5).to(DEV))      # noqa: E731
    return mk(E, F, H), mk(E, F, H), mk(E, H, F)


@pytest.mark.parametrize("T,H,F,E,top,softmax,renorm,scale_input", [
    (1, 128, 128, 4, 1, False, False, True), (1, 2048, 672, 8, 2, False, False, True), (2, 64, 32, 2, 2, True, True, False),
    (3, 200, 100, 5, 3, True, False, False), (8, 1003, 77, 7, 2, False, True, True), (16, 4096, 1184, 8, 2, True, True, False),
    (17, 512, 640, 16, 4, True, True, False), (33, 384, 129, 3, 1, False, False, False), (64, 1024, 256, 64, 8, True, True, False),
    (64, 640, 512, 8, 8, False, True, True), (5, 96, 2048, 33, 6, True, True, True)])
def test_moe(T, H, F, E, top, softmax, renorm, scale_input):
    ops = _ops()
    x = _acts(T, H, T + H)
    router = (_acts(E, H, 4) * H ** -0.5).to(torch.bfloat16)
    gate, up, down = _experts(E, F, H, F)
    dv = [decode(w).to(DEV) for w in (gate, up, down)]
    want, bound = plain_moe(x, router, *dv, top, softmax, renorm, scale_input)
    for dt in (torch.bfloat16, torch.float32):
        got = ops.mxfp4_moe(x, router, gate, up, down, top, softmax, renorm, scale_input, out_dtype=dt)
        far = (got.double() - want).abs() - bound * 2.0 ** -8 - (want.abs() * 2.0 ** -8 if dt == torch.bfloat16 else 0)
        assert got.dtype == dt and (far <= 0).all(), (far.max().item(), (far > 0).float().mean().item())


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "clamped"])
@pytest.mark.parametrize("T", [1, 20])
def test_moe_choices_and_activations(T, act):
    """A float32 router with a bias; a correction, groups, a scale and an epsilon on the weights; the other activations."""
    ops = _ops()
    E, F, H, top = 12, 160, 256, 3
    g = _gen(6)
    x = _acts(T, H, 8)
    router, bias = torch.randn(E, H, generator=g).to(DEV) * H ** -0.5, torch.randn(E, generator=g).to(DEV)
    choice = ops.MoeChoice(torch.randn(E, generator=g).to(DEV), 4, 2, 2.5, 1e-3)
    gate, up, down = _experts(E, F, H, 3)
    dv = [decode(w).to(DEV) for w in (gate, up, down)]
    want, bound = plain_moe(x, router, *dv, top, True, True, False, act, 1.5, bias, choice)
    got = ops.mxfp4_moe(x, router, gate, up, down, top, True, True, False, act, 1.5, bias, choice, out_dtype=torch.float32)
    assert ((got.double() - want).abs() <= bound * 2.0 ** -8).all()


def test_moe_ties_and_special_values():
    """Equal scores: the lower index; a token that is not a number leaves the others as they are; rows with strides; repeats."""
    ops = _ops()
    E, F, H, T = 6, 96, 160, 9
    gate, up, down = _experts(E, F, H, 2)
    x = _acts(T, H + 8, 3)[:, 8:]
    router = torch.zeros(E, H, dtype=torch.bfloat16, device=DEV)
    dv = [decode(w).to(DEV) for w in (gate, up, down)]
    want, bound = plain_moe(x, router, *dv, 2, True, True, False)
    got = ops.mxfp4_moe(x, router, gate, up, down, 2, True, True, False, out_dtype=torch.float32)
    assert ((got.double() - want).abs() <= bound * 2.0 ** -8).all()
    buf = torch.full((T, H + 10), 3.0, device=DEV)
    assert torch.equal(ops.mxfp4_moe(x, router, gate, up, down, 2, True, True, False, out=buf[:, 5:5 + H]), got)
    assert (buf[:, :5] == 3).all() and (buf[:, 5 + H:] == 3).all()
    y = x.clone()
    y[4, 7] = float("nan")
    bad = ops.mxfp4_moe(y, router, gate, up, down, 2, True, True, False, out_dtype=torch.float32)
    keep = [t for t in range(T) if t != 4]
    assert torch.isnan(bad[4]).all() and torch.equal(bad[keep], got[keep])


# ---- refusals ------------------------------------------------------------------------------------------------------------

def test_refusals():
    ops = _ops()
    K = ops.KernelError
    w = ops.mxfp4_quantize(_acts(100, 200, 1))
    x = _acts(4, 200, 2)
    bad = [
        lambda: ops.mxfp4_quantize(x.half()), lambda: ops.mxfp4_quantize(x[0]), lambda: ops.mxfp4_quantize(x.t()),
        lambda: ops.mxfp4_quantize(x.cpu()), lambda: ops.mxfp4_quantize(x[:0]), lambda: w.dequantize(torch.float16), lambda: w[0],
        lambda: ops.Mxfp4(w.codes, w.scales, 300), lambda: ops.Mxfp4(w.codes, w.scales[:, :1], 200), lambda: ops.Mxfp4(w.codes[:, 1:], w.scales, 200),
        lambda: ops.mxfp4_linear(x[:, :199], w), lambda: ops.mxfp4_linear(x.float(), w), lambda: ops.mxfp4_linear(x, w, act_bits=8),
        lambda: ops.mxfp4_linear(x.cpu(), w), lambda: ops.mxfp4_linear(x, w, x[0]), lambda: ops.mxfp4_linear(x, w, out_dtype=torch.float16),
        lambda: ops.mxfp4_linear(x, w, out=torch.empty(4, 99, device=DEV)), lambda: ops.mxfp4_linear(x.t().contiguous().t(), w),
    ]
    gate, up, down = _experts(4, 40, 200, 1)
    router = _acts(4, 200, 5)
    moe = lambda *a, **k: lambda: ops.mxfp4_moe(*a, **k)      # noqa: E731
    bad += [
        moe(x, router[:3], gate, up, down, 2), moe(x, router, gate, up, down, 0), moe(x, router, gate, up, down, 5),
        moe(x, router, gate, down, down, 2), moe(x, router, gate, up, up, 2), moe(x, router, gate[0], up[0], down[0], 1),
        moe(x, router, gate, up, down, 2, choice=ops.MoeChoice(None, 4, 1)), moe(x[:, :100], router, gate, up, down, 2), moe(x.float(), router, gate, up, down, 2), moe(x, router, gate, up, down, 2, act="relu"),
        moe(_acts(65, 200, 1), router, gate, up, down, 2), moe(x, router, gate, up, down, 2, choice=ops.MoeChoice(None, 3, 1)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(K):
            call()
            pytest.fail(f"call {i} was not refused")
    assert ops.mxfp4_linear(x[:0], w).shape == (0, 100)
    assert ops.mxfp4_moe(x[:0], router, gate, up, down, 2).shape == (0, 200)
