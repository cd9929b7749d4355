"""What the adapters' stack and the new kernels' C entries refuse, without a GPU: nothing is launched."""

import ctypes

import pytest
import torch

from prism_b200 import ops


def _parts(L=2, G=2, r=16, kp=24, rows=(8, 4), dtype=torch.bfloat16):
    return torch.zeros(L, G, r, kp, dtype=dtype), torch.zeros(L, sum(rows), r, dtype=dtype), torch.ones(L)


def test_stack_checks():
    a, b, s = _parts()
    low = ops.LowRank(a, b, s, rows=(8, 4), k=20)
    assert (low.k, low.n, low.rank, low.count) == (20, 12, 16, 2)
    assert ops.LowRank(a, b, s, rows=(8, 4)).k == 24
    E = ops.KernelError
    bad = [((a, b, s, (8, 5)), {}), ((a, b, s, (12,)), {}), ((a, b, s, (12, 0)), {}), ((a, b, s, ()), {}), ((a, b, s, (8, 4), 25), {}), ((a, b, s, (8, 4), 0), {}),
           ((a.float(), b, s, (8, 4)), {}), ((a.half(), b.half(), s, (8, 4)), {}), ((a, b, s.double(), (8, 4)), {}), ((a, b, s[:1], (8, 4)), {}),
           ((a[0], b, s, (8, 4)), {}), ((a.transpose(2, 3), b, s, (8, 4)), {})]
    for args, kw in bad:
        with pytest.raises(E):
            ops.LowRank(*args, **kw)
    for r, kp in ((8, 24), (144, 24), (16, 20), (0, 24)):
        with pytest.raises(E):
            ops.LowRank(*_parts(r=r, kp=kp), rows=(8, 4))
    with pytest.raises(E):
        ops.LowRank(*_parts(G=9, rows=(1,) * 9), rows=(1,) * 9)
    flat = torch.zeros(a.numel() + 1, dtype=torch.bfloat16)
    with pytest.raises(E):
        ops.LowRank(flat[1:].view(a.shape), b, s, rows=(8, 4))


def test_put():
    low = ops.LowRank.empty(3, 5, (8, 4), 21, torch.float32, "cpu")
    assert low.a.shape == (3, 2, 16, 24) and low.nbytes == 4 * (3 * 2 * 16 * 24 + 3 * 12 * 16 + 3)
    A, B = torch.randn(5, 21), torch.randn(4, 5)
    low.put(1, [None, (A, B)], 2.0)
    assert torch.equal(low.a[1, 1, :5, :21], A) and torch.equal(low.b[1, 8:, :5], B) and low.scale.tolist() == [0, 2, 0]
    assert low.a.count_nonzero() == A.numel() and low.b.count_nonzero() == B.numel()
    low.put(1, [None, None], 0.0)
    assert low.a.abs().sum() == 0 and low.b.abs().sum() == 0
    for index, slices in ((3, [None, None]), (-1, [None, None]), (0, [None]), (0, [(A, B), None]), (0, [None, (A[:, :20], B)]), (0, [None, (A, B[:, :4])]),
                          (0, [None, (torch.zeros(17, 21), torch.zeros(4, 17))])):
        with pytest.raises(ops.KernelError):
            low.put(index, slices, 1.0)


def test_rows_on_the_host_are_refused():
    low = ops.LowRank.empty(1, 4, (8,), 16, torch.float32, "cpu")
    with pytest.raises(ops.KernelError):
        ops.low_rank(torch.zeros(2, 16), low, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ops.KernelError):
        ops.sample_filtered(torch.zeros(2, 16), None, torch.zeros(2), torch.zeros(2, dtype=torch.int32))


def test_the_library_refuses_sizes():
    lib = ops.lib()
    first = (ctypes.c_int * 3)(0, 8, 12)
    p = ctypes.addressof(first)

    def low_rank(T=4, K=20, Kp=24, r=16, L=2, G=2, first=p, hidden=None, sms=148):
        return lib.prism_low_rank(p, 24, 0, p, p, p, p, p, 12, p, 12, 0, T, K, Kp, r, L, G, first, hidden, sms, p, None)
    assert low_rank(T=0) == 0
    back = (ctypes.c_int * 3)(0, 8, 8)
    for change in (dict(G=0), dict(G=9), dict(r=8), dict(r=0), dict(r=144), dict(r=24), dict(K=0), dict(Kp=16), dict(Kp=20, K=20), dict(L=0), dict(sms=0),
                   dict(first=ctypes.addressof(back))):
        assert low_rank(**change) == 1, change

    def draw(n=2, R=2, V=100, u=p, out=p):
        return lib.prism_sample_filtered(p, 100, n, R, V, p, u, p, p, p, p, out, p, p, p, None)
    assert draw(n=0) == 0
    for change in (dict(V=0), dict(n=70000, R=80000), dict(n=3), dict(u=None), dict(out=None)):
        assert draw(**change) == 1, change
