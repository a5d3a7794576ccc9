"""What a clipping plan keeps on the GPU, on the host with a library that only notes what it is given."""
import pytest
import torch

from llmc_b200.ops import kernels as KN


class OnDevice(torch.Tensor):
    """A host tensor that says it lies on a GPU."""
    @property
    def device(self):
        return torch.device("cuda", 0)


class Library:
    llmc_clip_chunk_bytes = staticmethod(lambda: 16384)
    llmc_clip_scratch = staticmethod(lambda: 593)
    llmc_clip = staticmethod(lambda *a: 0)


@pytest.fixture
def plan(monkeypatch):
    uploads, fills, used = [], [], []
    zeros = torch.zeros

    def on_host(*a, **k):
        if k.get("device") is not None:
            fills.append(a)
        k.pop("device", None)
        return zeros(*a, **k)

    def upload(t, *a, **k):
        uploads.append((t.numel(), a, k))
        return t.as_subclass(OnDevice)

    monkeypatch.setattr(KN._lib, "cuda", lambda: Library)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch, "zeros", on_host)
    monkeypatch.setattr(torch.Tensor, "to", upload)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: used.append((t.data_ptr(), s)))
    stream = {"now": 11}
    monkeypatch.setattr(KN, "_stream_of", lambda op, device: stream["now"])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream["now"])
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)

    def make(*sizes):
        return KN.clip_plan(None, [zeros(n).as_subclass(OnDevice) for n in sizes])

    return make, uploads, fills, used, stream


@pytest.mark.parametrize("sizes", [(5000, 3), (0,)])
def test_a_plan_is_ready_for_every_stream_when_it_has_been_made(plan, sizes):
    """Its table and its scratch are copies from host memory, each of which has arrived when it returns; a fill on the device would be ordered with the stream of the plan's making alone."""
    make, uploads, fills, _, _ = plan
    p = make(*sizes)
    assert not fills and len(uploads) == 2
    assert all(not any(isinstance(v, bool) and v for v in list(a) + list(k.values())) for _, a, k in uploads)        # none of them non-blocking
    assert p.scratch.numel() == 593 and not p.scratch.any()


def test_memory_of_a_plan_outlasts_its_calls_in_other_streams(plan):
    """Dropped behind a call in another stream: the allocator has to know that this stream reads the table still."""
    make, _, _, used, stream = plan
    p, norm = make(5000, 3), torch.ones(1).as_subclass(OnDevice)
    KN.clip_grad_norm(norm, p, 1.0)
    assert not used                                            # the stream that it was made in
    stream["now"] = 12
    KN.clip_grad_norm(norm, p, 1.0)
    KN.clip_grad_norm(norm, p, 1.0)
    assert used == [(p.table.data_ptr(), 12), (p.scratch.data_ptr(), 12)]
