"""The cache of bf16 weight operands, its bookkeeping on CPU tensors (the kernels' calls are replaced)."""
import pytest
import torch

from deep_vision_amd.ops import wcache


class Kernels:
    WPREP_CHUNK, WPREP_DESC_BYTES = 4096, 56

    def __init__(self):
        self.refreshed = 0

    def wprep_batched(self, *args):
        self.refreshed += 1


@pytest.fixture
def kernels(monkeypatch):
    k = Kernels()
    monkeypatch.setattr(wcache, "lib", lambda: k)
    monkeypatch.setattr(wcache, "stream_handle", lambda: 1)
    monkeypatch.setattr(wcache, "_entries", {})
    monkeypatch.setattr(wcache, "_tables", {})
    return k


def layout(param, done):
    def compute(out):
        done.append(param.data_ptr())
        return torch.empty(param.numel(), dtype=torch.bfloat16) if out is None else out
    return wcache.get(param, 1, 8, 0, compute)


def test_a_step_refreshes_parameters_that_moved_since_their_last_use(kernels):
    """An optimizer made after a first forward pass moves the parameters into its buffer; a step (of any
    optimizer) may come before the next forward pass."""
    p, done = torch.nn.Parameter(torch.zeros(4, 8)), []
    buf = layout(p, done)
    p.data = torch.ones(4, 8)
    wcache.after_step(torch.device("cpu"))
    assert kernels.refreshed == 1
    assert layout(p, done) is buf and len(done) == 1  # laid out by the step
    wcache.after_step(torch.device("cpu"))
    assert kernels.refreshed == 2
    p.data = torch.full((4, 8), 2.0)
    assert layout(p, done) is buf and len(done) == 2
