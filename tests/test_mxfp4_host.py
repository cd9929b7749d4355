"""The host side of the 4-bit operators, without a GPU: who gets which memory, and when."""

import threading
import time

import pytest
import torch


@pytest.fixture
def mx(monkeypatch):
    """``ops.mxfp4`` with one stream's memory in place, on the CPU."""
    from prism_b200.ops import mxfp4
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)
    monkeypatch.setattr(mxfp4, "_streams", {(None, 7): mxfp4._Own(torch.zeros(64, dtype=torch.int32), torch.empty(1024, dtype=torch.uint8))})
    monkeypatch.setattr(mxfp4, "_arenas", {None: [torch.zeros(1 << 12, dtype=torch.int32), 0]})
    monkeypatch.setattr(mxfp4, "_workspace", lambda size_of, sizes: (sizes[0], 8))
    return mxfp4


def in_threads(n, f):
    threads = [threading.Thread(target=f, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert not any(t.is_alive() for t in threads)


def test_calls_of_two_threads_do_not_share_a_stream_s_memory_at_once(mx):
    """A call of several launches has the stream's workspace and counters to itself until the last of them is on its way."""
    inside, most = [], []

    def launch(work, nbytes, counters):
        inside.append(work)
        most.append(len(inside))
        time.sleep(0.02)                                     # between a call's first launch and its second
        inside.remove(work)
        return 0

    in_threads(4, lambda i: [mx._with_memory(launch, (), "f", (100,), 7, torch.device("cpu")) for _ in range(3)])
    assert len(most) == 12 and max(most) == 1


def test_captures_of_two_threads_get_counters_of_their_own(mx, monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True, raising=False)
    given = []

    class Arena(list):                                       # a thread may be interrupted between reading the place and moving it on
        def __getitem__(self, i):
            v = super().__getitem__(i)
            if i == 1:
                time.sleep(0.002)
            return v
    mx._arenas[None] = Arena(mx._arenas[None])
    in_threads(4, lambda i: [mx._with_memory(lambda w, n, c: given.append(c) or 0, (), "f", (100,), 7, torch.device("cpu")) for _ in range(5)])
    assert len(given) == 20 == len(set(given))


def test_counters_are_cleared_behind_all_streams_work(mx, monkeypatch):
    """After a wait that ran out a launch on another stream may still be counting: the whole device is waited for first."""
    done = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: done.append(("wait", device)))

    class Counters(torch.Tensor):
        def zero_(self):
            done.append(("clear", None))
            return super().zero_()
    for own in mx._streams.values():
        own.counters = own.counters.add(3).as_subclass(Counters)
    mx._clear_counters()
    assert done[0] == ("wait", None) and ("clear", None) in done and done[-1][0] == "wait"
    assert not any(own.counters.any() for own in mx._streams.values())


def test_one_matrix_of_a_stack_and_nothing_else():
    from prism_b200 import ops
    w = ops.Mxfp4(torch.arange(3 * 5 * 64, dtype=torch.int64).remainder(251).to(torch.uint8).view(3, 5, 64), torch.zeros(3, 1, 1, 512, dtype=torch.uint8), 100)
    w.act_bits = 4
    for e in (0, 2, -1, torch.tensor(1)):
        one = w[e]
        assert one.shape == (5, 100) and one.act_bits == 4 and torch.equal(one.codes, w.codes[int(e)])
    for bad in (slice(0, 2), (0, 1), [0, 1], None, Ellipsis, 1.0):
        with pytest.raises(ops.KernelError):
            w[bad]
    for far in (3, -4):
        with pytest.raises(IndexError):
            w[far]
    assert [one.shape for one in w] == [(5, 100)] * 3


def test_captured_calls_take_the_counters_that_they_use(mx, monkeypatch):
    """A call whose first kernel clears counters in its workspace takes none; behind the last ones a graph clears its own."""
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True, raising=False)
    given = []

    def call():
        assert mx._with_memory(lambda w, n, c: given.append(c) or 0, (), "f", (100,), 7, torch.device("cpu")) == 0
    arena = mx._arenas[None]
    monkeypatch.setattr(mx, "_workspace", lambda size_of, sizes: (100, 0))
    call()
    assert arena[1] == 0 and not given[-1]
    monkeypatch.setattr(mx, "_workspace", lambda size_of, sizes: (100, 70))
    call()
    assert arena[1] == 128 and given[-1] == arena[0].data_ptr()
    monkeypatch.setattr(mx, "_ARENA", 250)
    call()
    assert arena[1] == 128 and given[-1] and not arena[0].data_ptr() <= given[-1] < arena[0].data_ptr() + 4 * arena[0].numel()


def test_threads_share_one_error_word(monkeypatch):
    """The word whose address is kept is the word that is read."""
    from prism_b200 import ops
    zeros = torch.zeros
    monkeypatch.setattr(ops, "_tc_err", {})

    def slow(*a, **k):
        time.sleep(0.02)
        return zeros(*a, **k)
    monkeypatch.setattr(torch, "zeros", slow)
    words = []
    in_threads(4, lambda i: words.append(ops._tc_err_word(torch.device("cpu"))))
    assert len(words) == 4 and all(w is ops._tc_err[0] for w in words)
