"""Low-rank adapters of many requests at once, beside a projection that they
share: ``out[t] = base[t] + s_l (x[t] A_l^T) B_l^T`` with l the adapter of
token t's request.  andre-fu/prism has no adapters: a model with one of its own
is a model of its own there (engine/weight_manager.py:45).

``LowRank``     the adapters of one projection, stacked
``low_rank``    their part of the projection's result, added to the shared part
``Adapted``     a projection's matrix with its adapters: what ``linear`` and its kin take in place of the matrix
"""

from __future__ import annotations

import ctypes
import itertools
from typing import Optional, Sequence

import torch

from .. import ops

MOST_RANK, MOST_SLICES = 128, 8      # csrc/low_rank.cu
RANK_UNIT, WIDTH_UNIT = 16, 8        # an adapter's rank in memory, and its A's rows, are whole numbers of these


def low_rank_limits():
    """``(largest rank, most slices)`` of a stack of adapters."""
    return MOST_RANK, MOST_SLICES


def _up(n: int, unit: int) -> int:
    return -(-n // unit) * unit


class LowRank:
    """Adapters of one projection ``[N, K]``.  ``a [L, G, r, Kp]``: the A of each of the L adapters for each of the G slices of the
    projection's rows (the matrices that it stacks: q, k and v, say), r rows each.  ``b [L, N, r]``: the rows of their B, all slices'
    below each other.  ``rows``: how many of the N rows each slice has.  r is a multiple of 16 up to 128, with zeros beyond an adapter's
    own rank; Kp is K rounded up to a multiple of 8 at least, with zeros beyond K.  ``scale``: float32 ``[L]``.  ``ranks``: int32 ``[L, G]``, the rank that
    each adapter has in each slice (0: it has none there); what lies beyond is no part of the formula, and an infinite x meets none of its zeros.
    None: all r rows of every A count."""

    __slots__ = ("a", "b", "scale", "ranks", "rows", "k", "rank", "count", "n", "_first", "_sizes")

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor, rows: Sequence[int], k: Optional[int] = None,
                 ranks: Optional[torch.Tensor] = None):
        rows = tuple(map(int, rows))
        sa, sb, dt = a.shape, b.shape, a.dtype
        if len(sa) != 4 or len(sb) != 3 or not rows or min(rows) < 1 or len(rows) > MOST_SLICES:
            raise ops.KernelError(f"adapters: A is [adapters, slices, rank, width] and B [adapters, rows, rank], of 1 to {MOST_SLICES} slices: got "
                                  f"{tuple(sa)}, {tuple(sb)} and rows {rows}")
        L, G, r, kp = sa
        k, n = kp if k is None else int(k), sum(rows)
        if G != len(rows) or sb != (L, n, r) or L < 1:
            raise ops.KernelError(f"adapters: A {tuple(sa)}, B {tuple(sb)} and rows {rows} do not belong together")
        if r % RANK_UNIT or not RANK_UNIT <= r <= MOST_RANK or kp % WIDTH_UNIT or not 1 <= k <= kp:
            raise ops.KernelError(f"adapters: a rank in memory is a multiple of {RANK_UNIT} up to {MOST_RANK} and a row of A a multiple of {WIDTH_UNIT} "
                                  f"that holds its {k} entries: got rank {r}, rows of {kp}")
        if (dt is not torch.bfloat16 and dt is not torch.float32) or b.dtype is not dt or scale.dtype is not torch.float32 or scale.shape != sa[:1]:
            raise ops.KernelError(f"adapters: A and B are both bfloat16 or both float32 and the scales float32 [{L}]: got {dt}, {b.dtype}, "
                                  f"{scale.dtype} {tuple(scale.shape)}")
        if not (a.is_contiguous() and b.is_contiguous() and scale.is_contiguous()) or a.data_ptr() % 16 or b.data_ptr() % 16 \
                or not a.get_device() == b.get_device() == scale.get_device():
            raise ops.KernelError("adapters: A, B and the scales lie contiguous on one device, A and B from a 16-byte border on")
        if ranks is not None and (ranks.dtype is not torch.int32 or ranks.shape != sa[:2] or not ranks.is_contiguous() or ranks.get_device() != a.get_device()):
            raise ops.KernelError(f"adapters: ranks are int32 [{L}, {G}], contiguous on {a.device}: got {ranks.dtype} {tuple(ranks.shape)} on {ranks.device}")
        self.ranks = ranks
        self.a, self.b, self.scale, self.rows, self.k, self.rank, self.count, self.n = a, b, scale, rows, k, r, L, n
        self._first = (ctypes.c_int * (G + 1))(0, *itertools.accumulate(rows))
        self._sizes = (k, kp, r, L, G, ctypes.addressof(self._first))

    def __reduce__(self):
        # copies and what is read back are made anew: the launchers follow the address of the borders, which are this object's
        return LowRank, (self.a, self.b, self.scale, self.rows, self.k, self.ranks)

    @classmethod
    def empty(cls, count: int, rank: int, rows: Sequence[int], k: int, dtype: torch.dtype, device) -> "LowRank":
        """Room for ``count`` adapters of ranks up to ``rank``, all zero (an adapter of zeros adds nothing).  All rows count until ``put`` says how many
        an adapter has."""
        r, kp = _up(int(rank), RANK_UNIT), _up(int(k), WIDTH_UNIT)
        return cls(torch.zeros((count, len(rows), r, kp), dtype=dtype, device=device), torch.zeros((count, sum(rows), r), dtype=dtype, device=device),
                   torch.zeros(count, dtype=torch.float32, device=device), rows, k, torch.full((count, len(rows)), r, dtype=torch.int32, device=device))

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.a, self.b, self.scale))

    @torch.no_grad()
    def put(self, index: int, slices, scale: float) -> None:
        """Adapter ``index``: per slice its ``(A [rank, K], B [rows, rank])``, or None where it has none."""
        if not 0 <= index < self.count or len(slices) != len(self.rows):
            raise ops.KernelError(f"adapter {index} of {self.count} with {len(slices)} of {len(self.rows)} slices")
        for g, ab in enumerate(slices):
            if ab is not None and not (ab[0].dim() == 2 and ab[0].shape[0] <= self.rank and ab[0].shape[1] == self.k
                                       and ab[1].shape == (self.rows[g], ab[0].shape[0])):
                raise ops.KernelError(f"adapter {index}: A {tuple(ab[0].shape)} and B {tuple(ab[1].shape)} for a matrix [{self.rows[g]}, {self.k}] and "
                                      f"ranks up to {self.rank}")
        self.a[index].zero_()
        self.b[index].zero_()
        self.scale[index] = float(scale)
        if self.ranks is not None:
            self.ranks[index].copy_(torch.tensor([0 if ab is None else ab[0].shape[0] for ab in slices], dtype=torch.int32))
        for g, ab in enumerate(slices):
            if ab is not None:
                rank, at = ab[0].shape[0], self._first[g]
                self.a[index, g, :rank, :self.k].copy_(ab[0])
                self.b[index, at:at + self.rows[g], :rank].copy_(ab[1])


class AdapterStep:
    """What the adapters of a model are told of a step before it runs: ``ids``, each token's adapter (int32 on the device), or None where no
    token has one; and ``low_rank``'s ``singles``."""

    __slots__ = ("ids", "singles")

    def __init__(self):
        self.ids, self.singles = None, 0


class Adapted:
    """A projection's matrix ``base`` (or an ``Mxfp4``) with its adapters: ``linear`` and what is built on it take it in the matrix's place.  In a
    step without adapters the matrix alone is used, by whichever kernel it would be used by; else the shared product runs as it does for a
    matrix by itself and the adapters' part is added to its result."""

    __slots__ = ("base", "low", "step")
    dtype = "adapted"                        # no kernel's: products that look for a dtype leave it to ``linear``

    def __init__(self, base, low: LowRank, step: AdapterStep):
        if tuple(base.shape) != (low.n, low.k):
            raise ops.KernelError(f"adapters for a matrix [{low.n}, {low.k}] beside one {tuple(base.shape)}")
        self.base, self.low, self.step = base, low, step

    @property
    def shape(self):
        return self.base.shape

    def dim(self) -> int:
        return 2

    def add_to(self, x: torch.Tensor, result: torch.Tensor) -> torch.Tensor:
        """The step's adapters' part, added to the shared product's result in place."""
        x = x if x.dtype is self.low.a.dtype else x.to(self.low.a.dtype)
        return low_rank(x, self.low, self.step.ids, result, result, self.step.singles)


def in_use(w):
    """``w`` itself, or the matrix alone of an ``Adapted`` whose adapters the step does not use."""
    return w.base if type(w) is Adapted and w.step.ids is None else w


SINGLES = 64                 # without a word from the caller, so many tokens are taken one by one
# So many tokens of portions, and they are taken in tiles: of 128 on tensor cores, or of 32 on CUDA cores (32-bit floats, sizes that TMA does not
# take); fewer one by one.  Microseconds one by one and in tiles, all tokens of one adapter, for gate and up, q k v and down of the 7B shape.
# bfloat16, rank 16: 64 tokens 15.5/18.6, 7.7/17.3, 10.4/28.1; 96 tokens 19.6/18.9, 10.6/17.6, 12.1/28.2; 128 tokens 32/19, 15.1/17.8, 16.5/28.4 (two adapters a
# tile cost the tiles a fifth more).  Rank 64: 64 tokens 68/20, 22/21, 27/29; 96 tokens 77/21, 34/22, 35/29.  Rank 128: 64 tokens 121/26, 43/27, 51/31.
# float32, rank 16: 192 tokens 110/62, 28/75, 51/178; 256 tokens 115/105, 42/76, 68/179; 384 tokens 170/122, 65/115, 127/181.  Rank 64: 128 tokens 220/81,
# 78/48, 85/185; 256 tokens 417/156, 147/84, 263/189.
# One border for all ranks and widths: it is near where the two meet for rank 16 and for the narrower matrices of rank 64; wide matrices of larger ranks would
# go in tiles from 32 tokens on (gate and up of rank 64: 35/19), q k v and down of rank 16 stay one by one longer.
TILE_FROM = 96
PLAIN_TILE_FROM = 256


def low_rank(x: torch.Tensor, low: LowRank, ids: torch.Tensor, base: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
             singles: Optional[int] = None) -> torch.Tensor:
    """``out[t] = base[t] + scale[l] (x[t] A_l^T) B_l^T`` with ``l = ids[t]`` (int32 ``[T]`` on the device; negative: ``out[t] = base[t]``).
    ``x [T, K]`` in the adapters' dtype; ``base`` and ``out [T, N]`` both bfloat16 or both float32, rows may have strides of their own;
    ``base`` None: zeros; ``out`` may be ``base`` itself, else it shares no memory with the others.  Adapters are finite.  Sums in float32, one rounding; portions in
    bfloat16 that go by tensor cores keep a hidden value (``x A^T``) as two bfloat16 terms, off by 2^-16 of it at most.  ``singles``: so many tokens from the first on
    are each a request of its own, and the others stand in runs of one adapter (as in a step: decoding requests, then portions of
    prompts); this says how the work is laid out and changes no result's meaning, though with the layout, and with how many tokens there are, the
    order of additions changes: a token's last bits may (among as many tokens in the same layout its neighbours change none).  An id outside the stack adds
    nothing and is reported by ``check_tc_errors``."""
    d, xs, dt = x.get_device(), x.shape, x.dtype
    if d < 0 or len(xs) != 2 or xs[1] != low.k or dt is not low.a.dtype or (x.stride(1) != 1 and low.k > 1) or low.a.get_device() != d:
        raise ops.KernelError(f"adapters in {low.a.dtype} on {low.a.device} for rows of {low.k} side by side in that CUDA device's memory: got {tuple(xs)} "
                              f"{dt}, strides {x.stride()} on {x.device}")
    T, N = xs[0], low.n
    if ids.dtype is not torch.int32 or ids.shape != xs[:1] or ids.get_device() != d or not ids.is_contiguous():
        raise ops.KernelError(f"adapters' numbers are int32 [{T}], contiguous on {x.device}: got {ids.dtype} {tuple(ids.shape)} on {ids.device}")
    if out is None:
        out = torch.empty((T, N), dtype=dt if base is None else base.dtype, device=x.device)
    odt = out.dtype
    for t in (out,) if base is None or base is out else (out, base):
        if t.shape != (T, N) or t.dtype is not odt or (odt is not torch.bfloat16 and odt is not torch.float32) or t.get_device() != d \
                or (t.stride(1) != 1 and N > 1) or (T > 1 and t.stride(0) < N):
            raise ops.KernelError(f"base and out are {T} rows of {N} side by side, both bfloat16 or both float32, on {x.device}: got {tuple(t.shape)} {t.dtype}, "
                                  f"strides {t.stride()} on {t.device}")
    ops._here(x, "low_rank")
    if T == 0:
        return out
    singles = (T if T <= SINGLES else 0) if singles is None else max(0, min(int(singles), T))
    L, stream, err = ops.lib(), ops._stream(), ops.mxfp4._err_word(x.device)
    sms = ops._num_sms.get(d) or ops.num_sms(x.device)
    ap, bp, sp, sizes, ranks = low.a.data_ptr(), low.b.data_ptr(), low.scale.data_ptr(), low._sizes, low.ranks
    bf16, out16 = dt is torch.bfloat16, odt is torch.bfloat16
    xp, x_row, ip, op, o_row = x.data_ptr(), x.stride(0), ids.data_ptr(), out.data_ptr(), out.stride(0)
    basep, b_row = (None, 0) if base is None else (base.data_ptr(), base.stride(0))
    if singles < T:
        G = len(low.rows)
        tiles = bf16 and xp % 16 == 0 and x_row % 8 == 0 and x_row >= low.k and L.prism_low_rank_tile_supported(low.k, low.rank, G, True)
        if T - singles < (TILE_FROM if tiles else PLAIN_TILE_FROM):
            singles = T
    if singles:
        ops._check(L.prism_low_rank(xp, x_row, bf16, ap, bp, sp, ip, basep, b_row, op, o_row, out16, singles, *sizes, None, sms, err, stream)
                   if ranks is None else
                   L.prism_low_rank_ranked(xp, x_row, bf16, ap, bp, sp, ranks.data_ptr(), ip, basep, b_row, op, o_row, out16, singles, *sizes, None, sms, err, stream),
                   "low_rank")
        if singles == T:
            return out
    rest, size = T - singles, 2 if out16 else 4
    xp, op, basep = xp + singles * x_row * (2 if bf16 else 4), op + singles * o_row * size, basep and basep + singles * b_row * size
    args = (ops._ptr(ranks), ip + 4 * singles, basep, b_row, op, o_row, out16, rest, *sizes)
    if tiles:
        hidden = torch.empty(2 * rest * G * low.rank + 2 * (-(-rest // 128)), dtype=torch.bfloat16, device=x.device)
        ops._check(L.prism_low_rank_tile(xp, x_row, ap, bp, sp, *args, hidden.data_ptr(), sms, err, stream), "low_rank_tile")
    else:
        hidden = torch.empty(rest * G * low.rank, dtype=torch.float32, device=x.device)
        ops._check(L.prism_low_rank_ranked(xp, x_row, bf16, ap, bp, sp, *args, hidden.data_ptr(), sms, err, stream), "low_rank")
    ops.launch_count += 1                    # two kernels
    return out
