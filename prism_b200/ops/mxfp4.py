"""Weights (and activations) in microscaled 4-bit floating point: elements of 4
bits (E2M1), one power of two (E8M0) for every 32 of them along a row - 17/32
of a byte an element, against 2 in bfloat16.  ``csrc/mxfp4.cuh`` has the format
bit by bit.  andre-fu/prism has no such path (its weights are those of the
file, engine/weight_pool.py:46-70).

``mxfp4_quantize``    rows to 4 bits; ``Mxfp4.dequantize`` gives the values back
``mxfp4_linear``      ``x @ w.T + bias`` with ``w`` in 4 bits, x as it is or brought to 4 bits too
``mxfp4_moe``         a whole mixture-of-experts layer for a few tokens, its experts in 4 bits
"""

from __future__ import annotations

import ctypes
import operator
import threading
from typing import Optional

import torch

from .. import ops

BLOCK, GROUP, TILE_ROWS, TILE_BYTES = 32, 128, 128, 512      # csrc/mxfp4.cuh
MOE_TOKENS, MOE_EXPERTS, MOE_TOP = 64, 256, 16               # the most of an ``mxfp4_moe`` call
DTYPE = "mxfp4"
MOE_CTAS = 0                # at most so many blocks share an ``mxfp4_moe`` call; 0: one an SM


class Mxfp4:
    """A matrix ``[N, K]`` (or a stack ``[E, N, K]`` of them) in 4 bits.  ``codes``: uint8 ``[..., N, Kp / 2]`` with ``Kp``
    the K rounded up to 128, element 2i in the low half of a byte, zero beyond K.  ``scales``: uint8 ``[..., ceil(N / 128),
    Kp / 128, 512]``: the scale of row r and block b of a tile of 128 rows by four blocks is byte ``(r % 32) * 16 + r % 128
    // 32 * 4 + b % 4``; zero for blocks beyond K, anything for rows beyond N.  ``act_bits``: what ``ops.linear`` does with the
    activations (``mxfp4_linear``); ``mxfp4_moe`` takes them as they are, so a stack's is 16."""

    __slots__ = ("codes", "scales", "shape", "act_bits")
    dtype = DTYPE

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, K: int):
        cs, ss = codes.shape, scales.shape
        groups, d = -(-K // GROUP), len(cs)
        if not (K > 0 and (d == 2 or d == 3) and len(ss) == d + 1 and cs[-1] == groups * (GROUP // 2) and cs[-2] > 0
                and ss[-1] == TILE_BYTES and ss[-2] == groups and ss[-3] == -(-cs[-2] // TILE_ROWS) and ss[0] == (cs[0] if d == 3 else ss[-3])
                and codes.dtype is torch.uint8 and scales.dtype is torch.uint8 and codes.is_contiguous() and scales.is_contiguous()
                and codes.device == scales.device):
            raise ops.KernelError(f"4-bit matrix of K = {K}: codes {tuple(cs)} {codes.dtype} and scales {tuple(ss)} {scales.dtype} do not belong together")
        self.codes, self.scales, self.shape, self.act_bits = codes, scales, (cs[0], K) if d == 2 else (cs[0], cs[1], K), 16

    @classmethod
    def _of(cls, codes, scales, shape) -> "Mxfp4":
        q = object.__new__(cls)
        q.codes, q.scales, q.shape, q.act_bits = codes, scales, shape, 16
        return q

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def dim(self) -> int:
        return len(self.shape)

    def __getitem__(self, e: int) -> "Mxfp4":
        """One matrix of a stack."""
        if len(self.shape) != 3 or not hasattr(e, "__index__"):
            raise ops.KernelError("only a stack of 4-bit matrices can be indexed, by the number of one of them")
        e = operator.index(e)
        one = Mxfp4._of(self.codes[e], self.scales[e], self.shape[1:])
        one.act_bits = self.act_bits
        return one

    def dequantize(self, dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The values that the codes stand for, exact in bfloat16 (default) and float32; NaN where the scale is 255.  ``out``:
        a place of this shape for them; a stack's matrices may lie apart in it."""
        dtype = dtype or (torch.bfloat16 if out is None else out.dtype)
        if dtype not in (torch.bfloat16, torch.float32):
            raise ops.KernelError(f"4-bit values come back as bfloat16 or float32, not {dtype}")
        codes, shape = self.codes, self.shape
        if not codes.is_cuda:
            ops._cuda(codes)
        K = shape[-1]
        if out is None:
            out = codes.new_empty(shape, dtype=dtype)
        elif out.shape != shape or out.dtype is not dtype or not out[0:1].is_contiguous() or not out.is_cuda or (
                len(shape) == 2 and not out.is_contiguous()) or (len(shape) == 3 and shape[0] > 1 and out.stride(0) < shape[1] * K) or (K % 8 == 0 and (out.data_ptr() % 16 or (len(shape) == 3 and out.stride(0) % 8))):
            raise ops.KernelError(f"4-bit values of {shape} do not go into {tuple(out.shape)} {out.dtype} with strides {out.stride()}")
        ops._check(ops.lib().prism_mxfp4_dequantize(codes.data_ptr(), self.scales.data_ptr(), shape[0] if len(shape) == 3 else 1, shape[-2], shape[-1],
                                                    out.data_ptr(), out.stride(0), ops.F32 if dtype is torch.float32 else ops.BF16, ops._stream()),
                   "mxfp4_dequantize")
        return out


def mxfp4_quantize(x: torch.Tensor) -> Mxfp4:
    """``x [N, K]`` (rows may have a stride of their own) or a contiguous stack ``[E, N, K]``, bfloat16 or float32, to 4
    bits: a block's exponent is that of its largest magnitude less two, elements round to nearest (ties to the even code) and
    saturate at 6.  A block that holds an infinity or NaN becomes NaN as a whole."""
    if not x.is_cuda:
        ops._cuda(x)
    xs = x.shape
    d = len(xs)
    N, K = (xs[-2], xs[-1]) if d == 2 or d == 3 else (0, 0)
    if not (N and K and xs[0] and (x.stride(-1) == 1 or K == 1) and (d == 2 or x.is_contiguous())):
        raise ops.KernelError(f"rows to quantise: a matrix whose rows lie side by side in memory or a contiguous stack of them, got {tuple(x.shape)} "
                              f"with strides {x.stride()}")
    groups, tiles = -(-K // GROUP), -(-N // TILE_ROWS)
    if d == 2:
        shape, matrices = (N, K), 1
        codes, scales = x.new_empty((N, groups * 64), dtype=torch.uint8), x.new_empty((tiles, groups, TILE_BYTES), dtype=torch.uint8)
    else:
        shape, matrices = (xs[0], N, K), xs[0]
        codes = x.new_empty((matrices, N, groups * 64), dtype=torch.uint8)
        scales = x.new_empty((matrices, tiles, groups, TILE_BYTES), dtype=torch.uint8)
    ops._check(ops.lib().prism_mxfp4_quantize(x.data_ptr(), ops._dt(x), x.stride(-2) if N > 1 else K, matrices, N, K, codes.data_ptr(),
                                              scales.data_ptr(), ops._stream()), "mxfp4_quantize")
    return Mxfp4._of(codes, scales, shape)


def _workspace(size_of: str, sizes):
    """``(bytes of workspace, counters)`` of a call."""
    b = (ctypes.c_longlong * 2)()
    if getattr(ops.lib(), size_of)(*sizes, ctypes.addressof(b)) != 0:
        raise ops.KernelError(f"{size_of}: sizes {sizes} are not supported")
    return b[0], b[1]


_err_words = {}


def _err_word(device: torch.device) -> int:
    """Address of the device's error word of bounded waits (``ops.check_tc_errors`` reads it)."""
    p = _err_words.get(device.index)
    if p is None:
        p = _err_words[device.index] = ops._tc_err_word(device).data_ptr()
    return p


_COUNTERS = 4096             # of a stream, the most of a call: tiles of a product in one launch (csrc/mxfp4_linear.cu), an experts' layer's control words
_TOO_SMALL = -1              # csrc/mxfp4.cuh: WORKSPACE_TOO_SMALL
_SCRATCH = 16 << 20          # a larger workspace is the call's own
_ARENA = 1 << 20
_streams = {}                # (device, stream) -> _Own: launches of one stream follow each other
_memory = threading.Lock()   # held from the choice of a call's memory until its last launch is on its way: threads share streams
_arenas = {}                 # device -> [counters for captured calls, how many are given away]


class _Own:
    """A stream's counters and workspace, and where they are."""

    __slots__ = ("counters", "work", "at")

    def __init__(self, counters: torch.Tensor, work: torch.Tensor):
        self.counters = counters
        self.use(work)

    def use(self, work: torch.Tensor) -> None:
        self.work, self.at = work, (work.data_ptr(), work.numel(), self.counters.data_ptr())


def _with_memory(run, args, size_of: str, sizes, stream: int, device: torch.device) -> int:
    """``run(workspace, its bytes, counters, *args)`` with memory that no other thread's call has meanwhile; its answer.  It is asked to
    run in the stream's workspace at once and says, before it launches anything, where that is too small: how much a call needs is
    for the device that it runs on to say.  Counters are zero before a launch and left so.  Under graph capture a call gets
    counters of its own for good, as graphs may run on any stream, and a workspace of the graph's."""
    with _memory:
        if torch._C._cuda_isCurrentStreamCapturing():
            arena = _arenas.get(device.index)
            nbytes, counters = _workspace(size_of, sizes)
            counters = (counters + 63) // 64 * 64
            if counters == 0:                                        # its first kernel clears those in its workspace
                at = 0
            elif arena is None or arena[1] + counters > _ARENA:
                block = torch.zeros(counters, dtype=torch.int32, device=device)            # cleared by the graph
                at = block.data_ptr()
            else:
                at = arena[0].data_ptr() + 4 * arena[1]
                arena[1] += counters
            work = torch.empty(nbytes, dtype=torch.uint8, device=device)
            return run(work.data_ptr(), work.numel(), at, *args)
        own = _streams.get((device.index, stream))
        if own is None:
            if device.index not in _arenas:
                _arenas[device.index] = [torch.zeros(_ARENA, dtype=torch.int32, device=device), 0]
                torch.cuda.current_stream(device).synchronize()      # captured calls of any stream find it cleared
            own = _streams[(device.index, stream)] = _Own(torch.zeros(_COUNTERS, dtype=torch.int32, device=device),
                                                          torch.empty(4 << 20, dtype=torch.uint8, device=device))
        code = run(*own.at, *args)
        if code == _TOO_SMALL:
            work = torch.empty(_workspace(size_of, sizes)[0], dtype=torch.uint8, device=device)
            if work.numel() <= _SCRATCH:
                own.use(work)
            code = run(work.data_ptr(), work.numel(), own.at[2], *args)
        return code


def _clear_counters():
    """After a launch that gave up (``ops.check_tc_errors``) its counters may be anything, and launches on other streams may still be
    counting: each device is waited for as a whole, then its counters are cleared."""
    with _memory:
        devices = sorted({key[0] for key in _streams} | set(_arenas), key=str)
        for device in devices:
            torch.cuda.synchronize(device)
        for block in [own.counters for own in _streams.values()] + [arena[0] for arena in _arenas.values()]:
            block.zero_()
        for device in devices:
            torch.cuda.synchronize(device)


def mxfp4_linear(x: torch.Tensor, w: Mxfp4, bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None, act_bits: int = 16) -> torch.Tensor:
    """``x @ w.T + bias`` for ``x [M, K]`` in bfloat16 (rows may have a stride of their own) and ``w [N, K]`` in 4 bits, sums
    in float32.  ``act_bits`` 16: x as it is; 4: each row of x is brought to 4 bits first, as ``mxfp4_quantize`` does it.
    ``out`` (row stride of its own) or ``out_dtype``: bfloat16 (default) or float32.  A row of x with an infinity or NaN in it
    gives NaN."""
    if not (x.is_cuda and w.codes.is_cuda and (bias is None or bias.is_cuda) and (out is None or out.is_cuda)):
        ops._cuda(x, w.codes, bias, out)
    xs, ws = x.shape, w.shape
    if len(xs) != 2 or len(ws) != 2 or xs[1] != ws[1]:
        raise ops.KernelError(f"product of {tuple(xs)} and {tuple(ws)}")
    M, K = xs
    N = ws[0]
    if x.dtype is not torch.bfloat16 or (x.stride(1) != 1 and K > 1) or act_bits not in (4, 16):
        raise ops.KernelError(f"activations are bfloat16 rows side by side in memory, used with 4 or 16 bits: got {x.dtype}, strides {x.stride()}, {act_bits}")
    if bias is not None and (bias.shape != (N,) or not bias.is_contiguous()):
        raise ops.KernelError(f"a bias has one entry per row of the weight, got {tuple(bias.shape)}")
    if out is None:
        out = x.new_empty((M, N), dtype=out_dtype)
    elif out.shape != (M, N) or (out.stride(1) != 1 and N > 1) or (M > 1 and out.stride(0) < N) or out_dtype not in (None, out.dtype):
        raise ops.KernelError(f"the result of {tuple(xs)} and {tuple(ws)} does not go into {tuple(out.shape)} {out.dtype} with strides {out.stride()}")
    if M == 0:
        return out
    stream = ops._stream()
    args = (x.data_ptr(), x.stride(0), w.codes.data_ptr(), w.scales.data_ptr(), None if bias is None else bias.data_ptr(),
            0 if bias is None else ops._dt(bias), out.data_ptr(), ops._dt(out), out.stride(0), M, N, K, act_bits, _err_word(x.device), stream)
    ops._check(_with_memory(ops.lib().prism_mxfp4_linear, args, "prism_mxfp4_linear_workspace", (M, N, K, act_bits), stream, x.device),
               "mxfp4_linear")
    return out


_ANY_CHOICE = ops.MoeChoice()


def mxfp4_moe(x: torch.Tensor, router: torch.Tensor, gate: Mxfp4, up: Mxfp4, down: Mxfp4, top: int, softmax: bool = False,
              renorm: bool = False, scale_input: bool = True, act: str = "silu", limit: float = 0.0,
              router_bias: Optional[torch.Tensor] = None, choice: Optional["ops.MoeChoice"] = None, out: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """A mixture-of-experts layer for up to 64 tokens, up to 256 experts and up to 16 of them a token, in one launch: ``x [T, H]``
    bfloat16, ``router [E, H]`` (logits in float32), ``gate``, ``up`` ``[E, F, H]`` and ``down`` ``[E, H, F]`` in 4 bits.  Each
    token takes the ``top`` experts with the largest scores (sigmoid of the logits, or their softmax; the lower index of equal ones); a choice's weight is its score
    (``renorm``: over the sum of the chosen) and multiplies the expert's input (``scale_input``) or its output.  ``act``:
    silu, gelu_tanh or clamped (with ``limit``, as in ``ops.glu``).  ``choice``: an ``ops.MoeChoice``.  Returns the sum over a
    token's choices, ``[T, H]`` bfloat16 or float32 (``out`` or ``out_dtype``).  Activations are taken as they are, hidden values are
    held to 2^-14 of themselves; a row of x, or 32 neighbouring hidden values, with an infinity or NaN among them are NaN as a whole."""
    for t in (x, router, gate.codes, up.codes, down.codes, router_bias, out):
        if t is not None and not t.is_cuda:
            ops._cuda(t)
    if x.dim() != 2 or x.dtype is not torch.bfloat16 or x.stride(1) != 1:
        raise ops.KernelError(f"activations are bfloat16 rows side by side in memory, got {tuple(x.shape)} {x.dtype}")
    T, H = x.shape
    E, F, _ = gate.shape if len(gate.shape) == 3 else (0, 0, 0)
    if not E or gate.shape != (E, F, H) or up.shape != gate.shape or down.shape != (E, H, F):
        raise ops.KernelError(f"experts {tuple(gate.shape)}, {tuple(up.shape)}, {tuple(down.shape)} do not belong together or to rows of {H}")
    if T > MOE_TOKENS or E > MOE_EXPERTS or not 1 <= top <= min(E, MOE_TOP):
        raise ops.KernelError(f"{T} tokens that use {top} of {E} experts: this layer is for up to {MOE_TOKENS} tokens, {MOE_EXPERTS} experts and "
                              f"{MOE_TOP} of them a token")
    if router.shape != (E, H) or not router.is_contiguous() or (router_bias is not None and (router_bias.shape != (E,) or not router_bias.is_contiguous())):
        raise ops.KernelError("the router has one row (and one bias) per expert")
    if act not in ops.GATED:
        raise ops.KernelError(f"a gated feed-forward's activation is one of {ops.GATED}, got {act!r}")
    ch = choice or _ANY_CHOICE
    corr = ch.correction
    if corr is not None and (corr.shape != (E,) or not corr.is_contiguous() or not corr.is_cuda):
        raise ops.KernelError("the correction has one entry per expert, on the device")
    if ch.groups < 1 or E % ch.groups or not 1 <= ch.keep <= ch.groups or ch.keep * (E // ch.groups) < top:
        raise ops.KernelError(f"{E} experts in {ch.groups} groups of which {ch.keep} are kept, {top} a token")
    if out is None:
        out = x.new_empty((T, H), dtype=out_dtype)
    elif out.shape != (T, H) or out.stride(1) != 1 or (T > 1 and out.stride(0) < H) or out_dtype not in (None, out.dtype):
        raise ops.KernelError(f"the result of {T} rows of {H} does not go into {tuple(out.shape)} {out.dtype} with strides {out.stride()}")
    if T == 0:
        return out
    stream = ops._stream()
    args = (x.data_ptr(), x.stride(0), router.data_ptr(), ops._dt(router), None if router_bias is None else router_bias.data_ptr(),
            0 if router_bias is None else ops._dt(router_bias), gate.codes.data_ptr(), gate.scales.data_ptr(), up.codes.data_ptr(), up.scales.data_ptr(),
            down.codes.data_ptr(), down.scales.data_ptr(), T, H, F, E, top, softmax, renorm, scale_input, ops.MOE_ACTS[act], limit,
            None if corr is None else corr.data_ptr(), 0 if corr is None else ops._dt(corr), ch.groups, ch.keep, ch.scale, ch.sum_eps, out.data_ptr(),
            ops._dt(out), out.stride(0), MOE_CTAS, _err_word(x.device), stream)
    ops._check(_with_memory(ops.lib().prism_mxfp4_moe, args, "prism_mxfp4_moe_workspace", (T, H, F, E, top, MOE_CTAS), stream, x.device),
               "mxfp4_moe")
    return out
