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


def test_other_streams_wait_for_the_layout_once(kernels, monkeypatch):
    now, waits = {"stream": 1, "capturing": False}, []

    class Event:
        def record(self):
            self.stream = now["stream"]

    class Current:
        def wait_event(self, event):
            waits.append((now["stream"], event.stream))

    class OnGpu:
        """A buffer as the cache looks at it."""

        is_cuda, device = True, torch.device("cuda", 0)

    monkeypatch.setattr(wcache, "stream_handle", lambda: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "current_stream", Current)
    p = torch.nn.Parameter(torch.zeros(4, 8))

    def use(stream, capturing=False):
        now.update(stream=stream, capturing=capturing)
        wcache.get(p, 1, 8, 0, lambda out: OnGpu())

    for s in (1, 1, 2, 2, 3, 1):
        use(s)
    use(4, capturing=True)
    assert waits == [(2, 1), (3, 1)]
    with torch.no_grad():
        p.add_(1)
    use(2)  # lays it out again
    for s in (1, 2, 3):
        use(s)
    assert waits == [(2, 1), (3, 1), (1, 2), (3, 2)]
