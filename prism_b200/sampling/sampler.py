"""Sampling parameters and the device sampler.

andre-fu/prism samples greedily when ``temperature <= 0`` and otherwise with
``softmax(logits / temperature)`` + ``torch.multinomial``
(engine/scheduler.py:266-272, engine/executor.py:423-427); it has no top-k,
top-p, min-p or penalties; this has the first three.  Differences: logits are float32,
the first token is sampled like every other (the reference always takes the
argmax there, scheduler.py:219), and the draw is the inverse CDF at a seeded
uniform number (``rng.uniform``) instead of an unseeded multinomial.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch

from .. import ops


@dataclass
class SamplingParams:
    """``max_new_tokens`` default 100 as ``Request.max_new_tokens``
    (engine/request_manager.py:24); ``temperature`` 0.0 = greedy (:25).  With a temperature, ``top_k`` (0: off), ``top_p`` (1:
    off) and ``min_p`` (0: off) say which tokens are drawn from (``ops.sample_filtered``).  ``logprobs``: the result lists the
    logarithm of the probability with which each token was drawn - after temperature and filters; 0 for a greedy one."""
    max_new_tokens: int = 100
    temperature: float = 0.0
    seed: Optional[int] = None
    eos_token_id: Optional[object] = None     # one id or several; None: the model's own
    ignore_eos: bool = False
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    logprobs: bool = False

    def __post_init__(self):
        if int(self.top_k) != self.top_k or not 0 <= self.top_k < 2 ** 31:
            raise ValueError(f"top_k {self.top_k!r}: a number of tokens, or 0 for all")
        if not 0 < self.top_p <= 1:
            raise ValueError(f"top_p {self.top_p!r}: a share of the probability above 0, up to 1 for all")
        if not 0 <= self.min_p <= 1:
            raise ValueError(f"min_p {self.min_p!r}: a share of the likeliest token's probability from 0 to 1")

    @property
    def by_filters(self) -> bool:
        """Whether its tokens are drawn by ``ops.sample_filtered``."""
        return self.logprobs or (self.temperature > 0 and (self.top_k > 0 or self.top_p < 1 or self.min_p > 0))


@dataclass
class SampleHandle:
    event: object
    host_tokens: torch.Tensor
    device_tokens: torch.Tensor
    host_logprobs: Optional[torch.Tensor] = None      # where the rows' parameters were given


class Sampler:
    """One kernel launch per step for all rows, two where some of them have filters and some draw without; token ids
    come back through a pinned buffer."""

    def __init__(self, device, max_rows: int = 256):
        self.device = torch.device(device)
        self.max_rows = max_rows
        # two sets of buffers: a step's tokens can still be read while the next step's are written
        self._outs = [torch.empty(max_rows, dtype=torch.int32, device=self.device) for _ in range(2)]
        self._hosts = [torch.empty(max_rows, dtype=torch.int32, pin_memory=True) for _ in range(2)]
        self._logprobs = [(torch.empty(max_rows, device=self.device), torch.empty(max_rows, pin_memory=True)) for _ in range(2)]
        self._turn = 0

    def sample(self, logits: torch.Tensor, temperatures: Sequence[float], us: Sequence[float]) -> List[int]:
        return self.read(self.sample_async(logits, temperatures, us))

    def sample_async(self, logits: torch.Tensor, temperatures: Sequence[float], us: Sequence[float],
                     params: Optional[Sequence[SamplingParams]] = None):
        """Launch the sampling kernel and the copy of the token ids to pinned host
        memory without waiting.  Returns a handle for ``read``; ``handle.device_tokens``
        (int32 ``[R]``) can feed the next step's token ids on the device.  ``params``: the rows' filters; a row that has none (and wants
        no logprobs) is drawn as it is without them, whatever rows it shares the step with."""
        R = logits.shape[0]
        if R > self.max_rows:
            self.__init__(self.device, max(R, 2 * self.max_rows))
        self._turn ^= 1
        out, host = self._outs[self._turn][:R], self._hosts[self._turn][:R]
        logprobs = None
        if params is not None:
            logprobs = self._sample_filtered(logits, temperatures, us, params, out)
        elif any(t > 0 for t in temperatures):
            tu = torch.tensor([list(temperatures), list(us)], dtype=torch.float32, pin_memory=True)
            tu = tu.to(self.device, non_blocking=True)
            ops.sample(logits, tu[0], tu[1], out)
        else:
            ops.sample(logits, None, None, out)
        host.copy_(out, non_blocking=True)
        ev = torch.cuda.Event()
        ev.record(torch.cuda.current_stream(self.device))
        return SampleHandle(ev, host, out, logprobs)

    def _sample_filtered(self, logits, temperatures, us, params, out) -> torch.Tensor:
        R = logits.shape[0]
        which = [i for i, p in enumerate(params) if p.by_filters]
        settings = torch.empty((7, R), dtype=torch.float32, pin_memory=True)
        s, whole = settings.numpy(), settings.view(torch.int32).numpy()
        s[0], s[1] = temperatures, us
        s[2], s[3] = [p.top_p for p in params], [p.min_p for p in params]
        whole[4] = [p.top_k for p in params]
        whole[5, :len(which)] = which
        # without filters: as ever; the others' draws are made after it
        s[6] = [0.0 if p.by_filters else t for p, t in zip(params, temperatures)]
        d = settings.to(self.device, non_blocking=True)
        i = d.view(torch.int32)
        if len(which) < R:
            drawn = bool((s[6] > 0).any())
            ops.sample(logits, d[6] if drawn else None, d[1] if drawn else None, out)
        lp, host = (t[:R] for t in self._logprobs[self._turn])
        ops.sample_filtered(logits, d[0], d[1], out, top_k=i[4], top_p=d[2], min_p=d[3], rows=i[5, :len(which)] if len(which) < R else None, logprob=lp)
        host.copy_(lp, non_blocking=True)
        return host

    def read(self, handle) -> List[int]:
        handle.event.synchronize()
        return handle.host_tokens.tolist()
