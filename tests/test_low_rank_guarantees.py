"""The adapters' stack on the host (CPU)."""

import copy
import ctypes
import gc
import pickle

import pytest
import torch

from prism_b200 import ops


def test_put_says_what_rank_an_adapter_has_in_each_slice():
    low = ops.LowRank.empty(3, 20, (8, 4), 24, torch.float32, "cpu")
    assert low.ranks.dtype is torch.int32 and low.ranks.tolist() == [[32, 32]] * 3           # nothing is said yet: all rows count
    low.put(1, [(torch.ones(5, 24), torch.ones(8, 5)), None], 1.0)
    assert low.ranks.tolist() == [[32, 32], [5, 0], [32, 32]]
    low.put(1, [None, (torch.ones(20, 24), torch.ones(4, 20))], 1.0)
    assert low.ranks.tolist() == [[32, 32], [0, 20], [32, 32]]
    with pytest.raises(ops.KernelError):
        low.put(1, [None, (torch.ones(20, 23), torch.ones(4, 20))], 1.0)
    assert low.ranks.tolist() == [[32, 32], [0, 20], [32, 32]]


def test_ranks_are_checked():
    a, b, s = torch.zeros(2, 2, 16, 24), torch.zeros(2, 12, 16), torch.ones(2)
    assert ops.LowRank(a, b, s, (8, 4)).ranks is None
    assert ops.LowRank(a, b, s, (8, 4), ranks=torch.ones(2, 2, dtype=torch.int32)).ranks.tolist() == [[1, 1]] * 2
    for ranks in (torch.ones(2, 2), torch.ones(2, dtype=torch.int32), torch.ones(2, 3, dtype=torch.int32), torch.ones(2, 4, dtype=torch.int32)[:, ::2]):
        with pytest.raises(ops.KernelError):
            ops.LowRank(a, b, s, (8, 4), ranks=ranks)


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda low: pickle.loads(pickle.dumps(low))], ids=["copy", "deepcopy", "pickle"])
@pytest.mark.parametrize("filled", [True, False])
def test_a_copy_has_borders_of_its_own(how, filled):
    """The slices' borders go to the kernels' launchers by their address in host memory: a copy outlives what it was made from."""
    low = ops.LowRank.empty(2, 4, (8, 4), 21, torch.float32, "cpu")
    if not filled:
        low = ops.LowRank(low.a, low.b, low.scale, (8, 4), 21)
    else:
        low.put(1, [(torch.ones(3, 21), torch.ones(8, 3)), None], 2.0)
    other = how(low)
    assert other._sizes[-1] == ctypes.addressof(other._first) and other._sizes[:-1] == low._sizes[:-1]
    want = low.a.clone(), low.b.clone(), None if low.ranks is None else low.ranks.tolist()
    del low
    gc.collect()
    assert list((ctypes.c_int * 3).from_address(other._sizes[-1])) == [0, 8, 12]
    assert (other.rows, other.k, other.rank, other.count, other.n) == ((8, 4), 21, 16, 2, 12)
    assert torch.equal(other.a, want[0]) and torch.equal(other.b, want[1]) and (None if other.ranks is None else other.ranks.tolist()) == want[2]


def test_matrices_that_want_gradients_leave_nothing_behind():
    """An adapter as a training loop has it: its values are taken, its graph is not."""
    low = ops.LowRank.empty(2, 4, (8,), 24, torch.float32, "cpu")
    a, b = torch.nn.Parameter(torch.randn(3, 24)), torch.nn.Parameter(torch.randn(8, 3))
    low.put(1, [(a * 2, b)], 1.0)
    assert torch.equal(low.a[1, 0, :3, :24], a.detach() * 2) and torch.equal(low.b[1, :, :3], b.detach())
    for t in (low.a, low.b, low.scale, low.ranks):
        assert not t.requires_grad and t.grad_fn is None


def test_the_library_refuses_sizes_with_ranks_and_in_tiles():
    lib = ops.lib()
    first, back = (ctypes.c_int * 3)(0, 8, 12), (ctypes.c_int * 3)(0, 8, 8)
    p, q = ctypes.addressof(first), ctypes.addressof(back)

    def ranked(T=4, K=20, Kp=24, r=16, L=2, G=2, first=p, hidden=None, sms=148):
        return lib.prism_low_rank_ranked(p, 24, 0, p, p, p, p, p, p, 12, p, 12, 0, T, K, Kp, r, L, G, first, hidden, sms, p, None)

    def tile(T=4, K=20, Kp=24, r=16, L=2, G=2, first=p, hidden=p, sms=148):
        return lib.prism_low_rank_tile(p, 24, p, p, p, p, p, p, 12, p, 12, 0, T, K, Kp, r, L, G, first, hidden, sms, p, None)
    assert ranked(T=0) == 0 and tile(T=0) == 0
    for change in (dict(G=0), dict(G=9), dict(r=8), dict(r=0), dict(r=144), dict(r=24), dict(K=0), dict(Kp=16), dict(Kp=20, K=20), dict(L=0), dict(sms=0), dict(first=q)):
        for T in (4, 70000):
            assert ranked(T=T, **change) == 1, change
        for T in (4, 65535 * 128 + 5):
            assert tile(T=T, **change) == 1, change
