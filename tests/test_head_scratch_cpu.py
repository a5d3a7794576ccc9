"""Scratch of the head's operators, on the host with a library that only notes what it is given."""
import threading

import pytest
import torch

from llmc_b200.ops import kernels as KN


class OnDevice(torch.Tensor):
    """A host tensor that says it lies on a GPU."""
    index = 0

    @property
    def device(self):
        return torch.device("cuda", self.index)


class Library:
    def __init__(self, words, call):
        self.llmc_linear_ce_fwd_scratch = lambda N, V: words(N, V)
        self.llmc_linear_ce_fwd = lambda losses, lse, scratch, *rest: call(scratch) or 0


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(KN, "_stream_of", lambda op, device: 0)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)
    empty, made = torch.empty, []

    def on_host(n, dtype=None, device=None):
        made.append(empty(n, dtype=dtype))
        return made[-1]

    monkeypatch.setattr(torch, "empty", on_host)
    monkeypatch.setattr(KN, "_scratch", KN._Scratch())
    KN._head_words.clear()
    yield monkeypatch, made
    KN._head_words.clear()


def _call(N=3, index=0):
    kind = type("OnDevice%d" % index, (OnDevice,), {"index": index})
    on = lambda t: t.as_subclass(kind)
    x, w = torch.zeros(N, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16)
    KN.linear_cross_entropy_forward(on(torch.zeros(N)), None, on(x), on(w), on(torch.zeros(N, dtype=torch.int32)), 5)


def test_threads_that_call_on_one_stream_have_scratch_of_their_own(host):
    """A call is several launches, between which another thread's may fall: what the first has left for the second must not be written meanwhile."""
    monkeypatch, _ = host
    both, seen = threading.Barrier(2, timeout=20), []

    def native(scratch):
        seen.append(scratch)
        both.wait()                          # the two calls are in the library at the same time

    lib = Library(lambda N, V: 1000, native)
    monkeypatch.setattr(KN._lib, "cuda", lambda: lib)
    threads = [threading.Thread(target=_call) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(seen) == 2 and seen[0] != seen[1]


def test_sizes_are_those_of_the_device_that_is_called(host):
    """What a call needs depends on the number of SMs: another GPU of the process may need more."""
    monkeypatch, made = host
    words = {"now": 100}
    lib = Library(lambda N, V: words["now"], lambda scratch: None)
    monkeypatch.setattr(KN._lib, "cuda", lambda: lib)
    _call(index=0)
    words["now"] = 300
    _call(index=1)
    assert [t.numel() for t in made] == [100, 300]
