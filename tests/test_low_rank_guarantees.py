"""The adapters' stack on the host (CPU)."""

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
