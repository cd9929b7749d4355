"""Uniform numbers beyond the ends of [0, 1), where many tokens are kept (GPU)."""

import math

import numpy as np
import pytest
import torch

from test_sample_filtered_gpu import DEV, check, draw, plain_row

pytestmark = pytest.mark.gpu
LAST = 1 - 2.0 ** -24                                    # the largest float32 below 1
KINDS = [("equal", 152064, None, None, None), ("equal", 9001, None, None, None), ("equal", 9001, 300, None, None), ("equal", 520, 400, None, None),
         ("equal", 152064, 5000, None, None), ("equal", 152064, None, 0.9, None), ("flat", 152064, None, None, None), ("flat", 40000, 300, 0.99, 0.001),
         ("flat", 400000, None, 0.999, None)]


@pytest.mark.parametrize("kind,V,k,p,m", KINDS)
def test_what_is_not_below_1_is_the_last_number_that_is(kind, V, k, p, m):
    """The weight of all kept tokens is a whole number of up to 63 bits here: more than a 64-bit float tells from the next one."""
    ends = [1.0, math.nan, 2.0, math.inf, 1 + 2.0 ** -23]
    R = len(ends)
    x = torch.zeros(R, V) if kind == "equal" else torch.randn(1, V, generator=torch.Generator().manual_seed(V)).expand(R, V) * 0.5
    x = x.contiguous().to(DEV)
    every = lambda v: None if v is None else [v] * R     # noqa: E731
    got = draw(x, [1.0] * R, ends, every(k), every(p), every(m))
    want = draw(x, [1.0] * R, [LAST] * R, every(k), every(p), every(m))
    assert got == want
    row = x[0].cpu().numpy()
    f = np.float32
    tok, kept, lp = plain_row(row, f(1.0), f(LAST), k or 0, f(1.0 if p is None else p), f(m or 0))
    for i in range(R):
        assert got[0][i] == tok and got[1][i] == kept and abs(got[2][i] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -40


@pytest.mark.parametrize("V,k", [(152064, None), (520, 400)])
def test_what_is_below_0_is_0(V, k):
    ends = [-0.0, -1.0, -math.inf, -1e-30]
    x = torch.zeros(4, V, device=DEV)
    k = None if k is None else [k] * 4
    assert draw(x, [1.0] * 4, ends, k) == draw(x, [1.0] * 4, [0.0] * 4, k)


@pytest.mark.parametrize("V", [300, 9001, 50257, 152064])
@pytest.mark.parametrize("scale", [3e-42, 2e-40, 4e-39, 1e-37])
def test_logits_and_temperatures_that_are_nearly_nothing(V, scale):
    """Below 2^-126 float32 has steps of 2^-149, whatever the value: borders between bins are values too."""
    R = 12
    g = torch.Generator().manual_seed(V)
    rng = np.random.RandomState(V % 1000)
    x = (torch.randn(R, V, generator=g, dtype=torch.float64) * scale).float().to(DEV)
    t = (scale * (0.1 + rng.rand(R))).astype(np.float32)
    check(x, t, 0.02 + 0.96 * rng.rand(R), k=[0, 0, 0, V // 2, 0, V // 3, 0, 300, 0, 0, V // 4, 0],
          p=[0.3, 0.6, 0.9, 0.99, 0.9999994, 0.5, 0.04, 0.97, 0.8, 0.25, 0.9, 0.75], m=[0, 0, 0, 0, 0, 1e-6, 0, 0, 1e-4, 0, 0, 0.01])


@pytest.mark.parametrize("V", [6, 700, 40000])
def test_what_is_too_unlikely_is_kept_and_never_drawn(V):
    """A token's weight counts in steps of 2^-46 of the largest one's: 2^-48 of it is none, 2^-45 is two."""
    x = torch.full((2, V), -math.inf)
    x[:, 0], x[:, V // 2], x[:, V - 1] = -48 * math.log(2), -45 * math.log(2), 0.0
    tok, kept, lp = draw(x.to(DEV), [1.0, 1.0], [0.0, 0.5])
    assert tok == [V // 2, V - 1] and kept == [3, 3]
    assert abs(lp[0] + 45 * math.log(2)) < 1e-5 and abs(lp[1]) < 2.0 ** -40
