"""The cache of bf16 weight operands, its bookkeeping on CPU tensors (the kernels' calls are replaced)."""
import pytest
import torch

from deep_vision_amd.ops import wcache


class Kernels:
    WPREP_CHUNK, WPREP_DESC_BYTES = 4096, 56

    def __init__(self):
        self.refreshed, self.table, self.single = 0, None, []

    def wprep_batched(self, *args):
        self.refreshed += 1
        self.table = args[0]

    def wprep(self, *args):
        self.single.append(args)


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

    class Stream:
        def __init__(self, handle):
            self.handle = handle

        def wait_stream(self, other):
            waits.append((self.handle, other.handle))

    monkeypatch.setattr(wcache, "stream_handle", lambda: now["stream"])
    monkeypatch.setattr(wcache, "_capturing", lambda: now["capturing"])
    monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda: Stream(0))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: Stream(now["stream"]))
    p = torch.nn.Parameter(torch.zeros(4, 8))

    def use(stream, capturing=False):
        now.update(stream=stream, capturing=capturing)
        wcache.get(p, 1, 8, 0, lambda out: torch.empty(4, 8))

    for s in (1, 1, 2, 2, 3, 1):
        use(s)
    use(4, capturing=True)
    assert waits == [(2, 1), (3, 1)]
    with torch.no_grad():
        p.add_(1)
    use(0)  # the default stream lays it out again
    for s in (1, 2, 0, 1):
        use(s)
    assert waits == [(2, 1), (3, 1), (1, 0), (2, 0)]


class Capture:
    """Says that the current stream captures, from inside ``with``."""

    on = False

    def __enter__(self):
        Capture.on = True

    def __exit__(self, *exc):
        Capture.on = False


@pytest.fixture
def capture(kernels, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: Capture.on)
    return Capture()


class Cuda(torch.Tensor):
    """A CPU buffer that the cache takes for one on the GPU."""

    is_cuda = True


def lay(param, mode=0, log=None):
    def compute(out):
        if log is not None:
            log.append(mode)
        return torch.empty(param.numel(), dtype=torch.bfloat16).as_subclass(Cuda) if out is None else out
    return wcache.get(param, 1, 8, mode, compute)


CPU = torch.device("cpu")


def test_a_captured_step_copies_nothing_from_the_host_and_keeps_what_it_touches(kernels, capture, monkeypatch):
    """A parameter of some other model dies between the last eager step and the captured one: the table of eager
    steps is out of date, and one made inside the capture would be a copy from memory that is gone at the replay."""
    import gc
    import weakref

    mine, other = torch.nn.Parameter(torch.zeros(4, 8)), torch.nn.Parameter(torch.zeros(4, 8))
    buf = lay(mine)
    lay(other)
    wcache.after_step(CPU)
    made = []
    real = wcache._make_table
    monkeypatch.setattr(wcache, "_make_table", lambda *a: made.append(Capture.on) or real(*a))
    step = wcache.step_capture([mine])
    with step, capture:
        del other
        gc.collect()
        assert lay(mine) is buf
        wcache.after_step(CPU)
    assert made == [False] and kernels.refreshed == 2
    assert kernels.table == step.table[0].data_ptr()  # its own, of its own parameters
    assert step.table[0].numel() == Kernels.WPREP_DESC_BYTES
    alive = weakref.ref(mine)
    wcache.clear()
    del mine
    gc.collect()
    assert alive() is not None and step.laid and next(iter(step.laid.values()))[0] is buf


def test_entries_after_replays(kernels, capture):
    p, q, log = torch.nn.Parameter(torch.zeros(4, 8)), torch.nn.Parameter(torch.zeros(4, 8)), []
    lay(p, 0, log), lay(q, 0, log)
    step = wcache.step_capture([p])
    with step, capture:
        lay(p, 0, log)
        lay(p, 1, log)  # not seen before the capture: the graph's own
        wcache.after_step(CPU)
    assert log == [0, 0, 1] and len(wcache._entries) == 2
    lay(p, 0, log), lay(p, 1, log), lay(q, 0, log)
    assert log == [0, 0, 1, 1]
    step.replayed()
    lay(p, 0, log), lay(q, 0, log)  # refreshed by the replay, not touched by it
    assert log == [0, 0, 1, 1]
    lay(p, 1, log), lay(p, 1, log)  # laid out between the capture and the replay
    assert log == [0, 0, 1, 1, 1]
    step.replayed()
    with torch.no_grad():
        p.add_(1)  # behind the replay
    lay(p, 0, log)
    assert log == [0, 0, 1, 1, 1, 0]
    step.replayed()
    p.data = torch.ones(4, 8)  # the graph goes on with the old address
    lay(p, 0, log)
    assert log == [0, 0, 1, 1, 1, 0, 0]


def test_two_captured_steps_with_different_operands(kernels, capture):
    p, log = torch.nn.Parameter(torch.zeros(4, 8)), []
    lay(p, 0, log)
    a = wcache.step_capture([p])
    with a, capture:
        wcache.after_step(CPU)
    lay(p, 1, log)
    b = wcache.step_capture([p])
    with b, capture:
        wcache.after_step(CPU)
    for order in ((a, b), (b, a)):
        del log[:]
        for c in order:
            c.replayed()
        lay(p, 0, log), lay(p, 1, log)
        assert log == [1]  # the first graph leaves that one as it was


def test_a_step_captured_by_hand(kernels, capture):
    class Owner:
        def __init__(self, *params):
            self.param_groups = [{"params": list(params)}]

    p, q = torch.nn.Parameter(torch.zeros(4, 8)), torch.nn.Parameter(torch.zeros(4, 8))
    buf = lay(p)
    lay(q)
    owner = Owner(p)
    with capture:
        wcache.after_step(CPU, owner)
    assert kernels.refreshed == 0 and [c[:2] for c in kernels.single] == [(p.data_ptr(), buf.data_ptr())]
    assert kernels.single[0][2:10] == (1, 4, 8, 1, 1, 8, 0, 0) and owner._captured_operands[0] is buf
    with wcache.step_capture([q]), capture:  # a second optimizer in a captured step
        wcache.after_step(CPU, owner)
    assert kernels.refreshed == 1 and len(kernels.single) == 2


def test_parameters_changed_between_replays_are_laid_out_before_the_next(kernels, capture):
    p = torch.nn.Parameter(torch.zeros(4, 8))
    lay(p)
    step = wcache.step_capture([p])
    with step, capture:
        wcache.after_step(CPU)
    assert kernels.refreshed == 1
    for change, launches in ((False, 1), (True, 2), (False, 2), (True, 3)):
        if change:
            with torch.no_grad():
                p.mul_(0.5)
        step.catch_up()
        step.replayed()
        assert kernels.refreshed == launches
