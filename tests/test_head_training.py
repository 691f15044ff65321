"""What a training loop does around layer norm and linear cross entropy: steps between the passes, several
captured signatures, forward-mode derivatives, traces, streams and threads. The CPU tests run the ops' Python
with the kernels' calls replaced."""
import pytest
import torch

from deep_vision_amd import nn as dnn
from deep_vision_amd import ops as F
from deep_vision_amd.ops import common, loss, norm
from deep_vision_amd.train.optim import FusedAdamW, FusedSGD

DEV = "cuda"
gpu = pytest.mark.gpu


class Kernels:
    """Stands in for the extension: every launch is counted and does nothing."""

    XENT_MAX_ROWS, XENT_MAX_CLASSES = 1 << 22, 1 << 30

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 64  # bytes of a workspace, rows of a slab
        return call


@pytest.fixture
def on_cpu(monkeypatch):
    """The ops' GPU path on CPU tensors; ``now`` says which stream is current and whether it captures."""
    now, kernels = {"stream": 1, "capturing": False}, Kernels()
    for m in (common, norm, loss):
        monkeypatch.setattr(m, "stream_handle", lambda: now["stream"])
        monkeypatch.setattr(m, "lib", lambda: kernels)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    for m in (norm, loss):
        monkeypatch.setattr(m, "native", lambda x: True)
    monkeypatch.setattr(loss, "_operand", lambda w, Dp: torch.zeros(w.shape[0], Dp, dtype=torch.bfloat16))
    now["kernels"] = kernels
    return now


def head(width=8, classes=5, dev="cpu"):
    torch.manual_seed(0)
    return dnn.LayerNorm(width).to(dev), dnn.Linear(width, classes).to(dev)


def call(op, norm_layer, fc, x, y):
    if op == "layer_norm":
        return norm_layer(x)
    return F.linear_cross_entropy(x, fc.weight, y, fc.bias, reduction="none")


# ---------------------------------------------------------------- an optimizer step between the passes
@pytest.mark.parametrize("op", ["layer_norm", "linear_cross_entropy"])
@pytest.mark.parametrize("make", [lambda p: FusedAdamW(p, lr=0.1), lambda p: FusedSGD(p, lr=0.1)])
def test_a_step_between_the_passes_is_refused(on_cpu, op, make):
    norm_layer, fc = head()
    opt = make([*norm_layer.parameters(), *fc.parameters()])
    other = make([torch.nn.Parameter(torch.ones(3))])
    x, y = torch.randn(4, 8).bfloat16().requires_grad_(), torch.zeros(4, dtype=torch.int64)
    out = call(op, norm_layer, fc, x, y)
    other.step()  # of other parameters
    out.sum().backward()
    for move in (opt.step, opt.graph_tick):
        opt.use_device_hparams(move == opt.graph_tick)
        out = call(op, norm_layer, fc, x, y)
        move()
        with pytest.raises(RuntimeError, match="updated the weight since the forward pass"):
            out.sum().backward()
        call(op, norm_layer, fc, x, y).sum().backward()


def test_a_step_of_the_bias_alone_or_of_neither(on_cpu):
    norm_layer, fc = head()
    x, y = torch.randn(4, 8).bfloat16().requires_grad_(), torch.zeros(4, dtype=torch.int64)
    opt = FusedSGD(fc.parameters(), lr=0.1)
    for skip, text in (("weight", "updated the bias"), ("bias", "updated the weight")):
        out = call("linear_cross_entropy", None, fc, x, y)
        getattr(fc, skip).grad = None  # it stays
        opt.step()
        with pytest.raises(RuntimeError, match=text):
            out.sum().backward()
    out = call("layer_norm", norm_layer, fc, x, y)
    fc.weight.grad = fc.bias.grad = None
    opt.step()
    out.sum().backward()
    shaped = torch.nn.Parameter(torch.ones(2, 4))  # read through a reshaped view
    opt = FusedSGD([shaped], lr=0.1)
    out = F.layer_norm(x.view(4, 2, 4), (2, 4), shaped)
    opt.step()
    with pytest.raises(RuntimeError, match="updated the weight"):
        out.sum().backward()


@pytest.mark.parametrize("move", ["again", "split", "joined"])
def test_a_step_of_an_optimizer_made_between_the_passes(on_cpu, move):
    """The parameters move from one optimizer's buffer to others' between the passes; what steps then counts, and
    what does not step does not."""
    norm_layer, fc = head()
    x, y = torch.randn(4, 8).bfloat16().requires_grad_(), torch.zeros(4, dtype=torch.int64)
    params = [*fc.parameters(), *norm_layer.parameters()]
    if move == "joined":
        FusedSGD(fc.parameters(), lr=0.1), FusedSGD(norm_layer.parameters(), lr=0.1)
    else:
        FusedSGD(params, lr=0.1)
    for stepped in (True, False):
        out = call("linear_cross_entropy", None, fc, x, y)
        if move == "split":
            opt, other = FusedSGD(fc.parameters(), lr=0.1), FusedSGD(norm_layer.parameters(), lr=0.1)
        else:
            opt, other = FusedSGD(params, lr=0.1), FusedSGD([torch.nn.Parameter(torch.ones(2))], lr=0.1)
        other.step()
        if stepped:
            FusedSGD(opt.param_groups[0]["params"], lr=0.1).step()  # the same parameters once more
            with pytest.raises(RuntimeError, match="an optimizer has updated"):
                out.sum().backward()
        else:
            out.sum().backward()


@gpu
@pytest.mark.parametrize("op", ["layer_norm", "linear_cross_entropy"])
def test_a_step_between_the_passes_is_refused_on_the_gpu(op):
    norm_layer, fc = head(64, 90, DEV)
    opt = FusedAdamW([*norm_layer.parameters(), *fc.parameters()], lr=0.1)
    x, y = torch.randn(20, 64, device=DEV).bfloat16().requires_grad_(), torch.randint(0, 90, (20,), device=DEV)
    out = call(op, norm_layer, fc, x, y)
    want = torch.autograd.grad(out.sum(), x, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(out.sum(), x, retain_graph=True)[0], want)
    with torch.autograd.graph.save_on_cpu():
        kept = call(op, norm_layer, fc, x, y)
    out.sum().backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="updated the weight since"):
        out.sum().backward()
    if op == "layer_norm":  # what was saved elsewhere is what the forward pass saw
        assert torch.equal(torch.autograd.grad(kept.sum(), x)[0], want)
    call(op, norm_layer, fc, x, y).sum().backward()


# ---------------------------------------------------------------- what watches a call beside autograd
def tensors_of(op):
    x = torch.randn(4, 8)
    if op == "layer_norm":
        return [x, torch.ones(8), torch.zeros(8)], lambda x, w, b: F.layer_norm(x, 8, w, b)
    y = torch.zeros(4, dtype=torch.int64)
    return [x, torch.randn(5, 8).bfloat16(), torch.zeros(5)], lambda x, w, b: F.linear_cross_entropy(x, w, y, b)


@pytest.mark.parametrize("op", ["layer_norm", "linear_cross_entropy"])
@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_is_refused(on_cpu, op, no_grad):
    from torch.autograd import forward_ad

    args, f = tensors_of(op)
    for i in range(3):
        with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(NotImplementedError, match="forward mode"):
                f(*dual)
    assert not f(*args).requires_grad


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("op", ["layer_norm", "linear_cross_entropy"])
@pytest.mark.parametrize("no_grad", [False, True])
def test_a_trace_records_the_operator(on_cpu, op, no_grad):
    args, f = tensors_of(op)
    with torch.set_grad_enabled(not no_grad):
        traced = torch.jit.trace(lambda x, w, b: f(x, w, b), args, check_trace=False)
    nodes = [n.kind() for n in traced.graph.nodes()]
    assert "prim::PythonOp" in nodes and "aten::empty" not in nodes
    before = len(on_cpu["kernels"].calls)
    traced(*args)
    assert len(on_cpu["kernels"].calls) > before


@gpu
@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("op", ["layer_norm", "linear_cross_entropy"])
def test_a_traced_call_gives_the_operators_results(op):
    args, f = tensors_of(op)
    args = [t.to(DEV) for t in args]
    if op == "linear_cross_entropy":
        y = torch.tensor([0, 4, 2, 1], device=DEV)
        f = lambda x, w, b: F.linear_cross_entropy(x, w, y, b)  # noqa: E731
    traced = torch.jit.trace(f, args, check_trace=False)
    for k in range(3):
        now = [t + k if t.dtype == torch.float32 else t for t in args]
        torch.empty(1 << 20, device=DEV).fill_(float("nan"))
        assert torch.equal(traced(*now), f(*now))


# ---------------------------------------------------------------- several captured signatures
class Fake:
    """Stands in for a stream or a graph."""

    handles = 100

    def __init__(self, *args, **kw):
        Fake.handles += 1
        self.handle = Fake.handles

    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture
def captures(on_cpu, monkeypatch):
    """CapturedStep on CPU tensors; the list of what it does to the device, in order."""
    import contextlib

    from deep_vision_amd.ops import act

    done = []

    @contextlib.contextmanager
    def within(stream, capturing=False):
        old = dict(on_cpu)
        on_cpu.update(stream=stream.handle, capturing=capturing)
        done.append("capture" if capturing else "warm-up")
        yield
        on_cpu.update(old)

    for name, to in (("Stream", Fake), ("CUDAGraph", Fake), ("current_stream", Fake),
                     ("synchronize", lambda: done.append("synchronize")), ("current_device", lambda: 0),
                     ("stream", within), ("graph", lambda g, stream: within(stream, True))):
        monkeypatch.setattr(torch.cuda, name, to)
    monkeypatch.setattr(act, "step_counter", lambda dev: None)
    return done


@pytest.mark.parametrize("backend", ["nccl", None])
def test_a_capture_begins_when_the_collectives_before_it_are_off_the_watchdogs_list(captures, monkeypatch, backend):
    import time

    from deep_vision_amd.train.graph import CapturedStep

    monkeypatch.setenv("TORCH_NCCL_ASYNC_ERROR_HANDLING", "0")
    monkeypatch.setattr(torch.distributed, "is_initialized", lambda: backend is not None)
    monkeypatch.setattr(torch.distributed, "get_backend", lambda: backend)
    monkeypatch.setattr(time, "sleep", lambda s: captures.append(s))
    opt = FusedSGD([torch.nn.Parameter(torch.zeros(3))], lr=0.1)
    CapturedStep(lambda: None, opt)
    waits = [x for x in captures if isinstance(x, float)]
    assert captures == ["warm-up", "synchronize", *waits, "capture"]
    assert (sum(waits) > 0.2) if backend else not waits  # the watchdog's period is 0.1 s


def test_every_signature_is_captured_beside_the_outputs_of_the_others(captures):
    """Each capture has a stream of its own; a step that returns its loss as it is leaves no graph behind, once released."""
    from deep_vision_amd.train.graph import CapturedStep

    norm_layer, fc = head()
    opt = FusedSGD([*norm_layer.parameters(), *fc.parameters()], lr=0.1)

    def step(x, y):
        opt.zero_grad()
        loss = call("linear_cross_entropy", None, fc, norm_layer(x), y).sum()
        loss.backward()
        opt.step()
        return loss, {"again": [loss, 3]}

    kept = []
    for rows in (4, 3, 2):
        kept.append(CapturedStep(step, opt, (torch.randn(rows, 8).bfloat16(), torch.zeros(rows, dtype=torch.int64)), warmup=1))
        kept[-1].release()
    for cap in kept:
        assert cap.outputs[0].grad_fn is None and cap.warmup_outputs[1]["again"][0].grad_fn is None
        assert cap.outputs[1]["again"][1] == 3


@gpu
def test_two_batch_sizes_through_the_trainers_captured_step():
    """Replays of either signature, in turn, against eager steps: losses and parameters as in eager training, but
    for the bias corrections (in 32 bits on the device, 64 on the host)."""
    from deep_vision_amd.train.graph import GraphedTrainStep

    def make():
        norm_layer, fc = head(128, 300, DEV)
        model = torch.nn.Sequential(norm_layer, fc)
        opt = FusedAdamW(model.parameters(), lr=1e-3)

        def forward_loss(x, y):
            z = norm_layer(x)
            return F.linear_cross_entropy(z, fc.weight, y, fc.bias), z

        def eager(x, y):
            opt.zero_grad()
            loss, z = forward_loss(x, y)
            loss.backward()
            opt.step()
            return loss.detach(), z.detach()

        return model, opt, forward_loss, eager

    model, opt, forward_loss, eager = make()
    graphed = GraphedTrainStep(model, opt, forward_loss, eager)
    twin, _, _, plain = make()
    g = torch.Generator(device=DEV).manual_seed(0)
    for k, rows in enumerate((64, 64, 24, 64, 24, 24, 64)):
        x = torch.randn(rows, 128, generator=g, device=DEV).bfloat16()
        y = torch.randint(0, 300, (rows,), generator=g, device=DEV)
        a, b = graphed(x, y), plain(x, y)
        torch.cuda.synchronize()
        torch.testing.assert_close(a[0], b[0], rtol=2e-3, atol=2e-3)
        for p, q in zip(model.parameters(), twin.parameters()):
            assert (p - q).norm() <= 1e-3 * q.norm(), k
    assert len(graphed.graphs) == 2


# ---------------------------------------------------------------- the record of live graphs
class Track(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *leaves):
        common.track_leaves(ctx, *leaves)
        return sum(t.sum() for t in leaves)

    @staticmethod
    def backward(ctx, g):
        raise NotImplementedError


def test_two_threads_lose_no_live_graph(on_cpu, monkeypatch):
    import threading
    import time
    import weakref

    class Slow:
        @staticmethod
        def ref(t):
            time.sleep(0.05)  # both threads are here at once, unless one waits for the other
            return weakref.ref(t)

    monkeypatch.setattr(common, "weakref", Slow)
    for last in range(2):
        on_cpu.update(stream=1, capturing=False)
        x = torch.zeros(2, requires_grad=True)
        out = [None, None]

        def forward(i):
            out[i] = Track.apply(x)

        threads = [threading.Thread(target=forward, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        on_cpu.update(stream=2, capturing=True)
        out[1 - last] = None
        with pytest.raises(RuntimeError, match="still alive"):
            Track.apply(x)
        out[last] = None
        Track.apply(x)


def test_the_record_stays_small_and_is_not_searched_on_every_call(on_cpu, monkeypatch):
    monkeypatch.setattr(common, "_GRAPHS", {})
    monkeypatch.setattr(common, "_GRAPHS_KEEP", 8)
    monkeypatch.setattr(common, "_graphs_limit", 8)
    for _ in range(100):
        Track.apply(torch.zeros(1, requires_grad=True))
    assert len(common._GRAPHS) <= 9
    leaves = [torch.zeros(1, requires_grad=True) for _ in range(100)]
    alive = [Track.apply(t) for t in leaves]
    assert len(common._GRAPHS) >= 100 and common._graphs_limit >= 100
    del alive


# ---------------------------------------------------------------- the parameter's operand
@gpu
@pytest.mark.parametrize("warm", [True, False])
def test_replays_follow_a_parameter_that_changes(warm):
    """A graph of the loss and its gradients, no optimizer in it. Parameters change between the replays: by torch
    operations, by another optimizer, by this package's. Without eager passes before the capture too."""
    torch.manual_seed(0)
    fc = dnn.Linear(72, 130).to(DEV)
    x, y = torch.randn(40, 72, device=DEV).bfloat16().requires_grad_(), torch.randint(0, 130, (40,), device=DEV)
    leaves = [x, fc.weight, fc.bias]

    def passes(weight=fc.weight):
        out = F.linear_cross_entropy(x, weight, y, fc.bias)
        return [out.detach(), *torch.autograd.grad(out, [x, weight, fc.bias])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    if warm:
        with torch.cuda.stream(s):
            passes()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = passes()
        with torch.no_grad():
            got.append(F.linear_cross_entropy(x, fc.weight, y, fc.bias))
    eager = passes()  # before any replay
    assert all(torch.equal(a, b) for a, b in zip(eager, passes(fc.weight.detach().clone().requires_grad_())))
    fused = FusedSGD(fc.parameters(), lr=0.5)  # the parameters move into its buffer: a new capture below
    if warm:
        with torch.cuda.stream(s):
            passes()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = passes()
        with torch.no_grad():
            got.append(F.linear_cross_entropy(x, fc.weight, y, fc.bias))
    other = torch.optim.SGD(leaves[1:], lr=0.5)
    for k in range(6):
        if k % 3 == 0:
            with torch.no_grad():
                fc.weight.add_(0.1 * torch.randn_like(fc.weight))
        else:
            for p in leaves[1:]:
                p.grad.normal_()
            (other if k % 3 == 1 else fused).step()
        graph.replay()
        torch.cuda.synchronize()
        want = passes(fc.weight.detach().clone().requires_grad_())  # no cached operand
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k
        assert torch.equal(got[-1], want[0])


@gpu
def test_a_parameter_shared_by_two_streams():
    """Both streams only read the parameter: the second finds an operand that the first, held up, has yet to lay out."""
    torch.manual_seed(0)
    fc = dnn.Linear(256, 1000).to(DEV)
    x, y = torch.randn(64, 256, device=DEV).bfloat16(), torch.randint(0, 1000, (64,), device=DEV)
    want = F.linear_cross_entropy(x, fc.weight.detach().clone(), y, fc.bias)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for change in (False, True):
        if change:
            with torch.no_grad():
                fc.weight.mul_(0.5)
            want = F.linear_cross_entropy(x, fc.weight.detach().clone(), y, fc.bias)
        torch.cuda.synchronize()
        with torch.cuda.stream(a), torch.no_grad():
            torch.cuda._sleep(200_000_000)  # clock ticks: tens of milliseconds, then the stream goes on
            first = F.linear_cross_entropy(x, fc.weight, y, fc.bias)
        with torch.cuda.stream(b), torch.no_grad():
            second = [F.linear_cross_entropy(x, fc.weight, y, fc.bias) for _ in range(2)]
        torch.cuda.synchronize()
        assert torch.equal(first, want) and all(torch.equal(t, want) for t in second)


# ---------------------------------------------------------------- sizes
def test_more_logits_than_a_launch_holds_are_refused(on_cpu):
    on_cpu["kernels"].linear_xent_fwd_bytes = lambda *args: -1
    _, fc = head()
    with pytest.raises(ValueError, match="more than a call takes"):
        call("linear_cross_entropy", None, fc, torch.randn(4, 8).bfloat16(), torch.zeros(4, dtype=torch.int64))
    assert "linear_xent_fwd" not in on_cpu["kernels"].calls


@gpu
@pytest.mark.parametrize("rows,classes,fits", [(1 << 22, 1 << 16, True), (1 << 20, 1 << 18, True), (1 << 22, 1 << 18, False),
                                               (1 << 20, 1 << 20, False), (1 << 22, 3, True), (1, 1 << 30, True), (256, 1 << 30, True),
                                               (1 << 8, 1 << 29, True), (300, 1 << 30, False)])
def test_which_sizes_a_launch_holds(rows, classes, fits):
    """The sizes alone, nothing is launched: 2^32 threads are more than a launch takes, and the largest tile, 256 x 256,
    has 512 of them. Few rows take larger tiles than they otherwise would."""
    from deep_vision_amd._ext import lib

    for D in (64, 2048):
        assert (lib().linear_xent_fwd_bytes(0, D, 0, D, 0, 0, rows, classes, D, D, -100, 0.0, 1) >= 0) == fits


@gpu
def test_a_checkpoint_loaded_between_replays_of_a_training_step():
    """The next replay starts from the loaded parameters, as an eager step does."""
    from deep_vision_amd.train.graph import CapturedStep

    def make():
        norm_layer, fc = head(64, 200, DEV)
        model = torch.nn.Sequential(norm_layer, fc)
        opt = FusedSGD(model.parameters(), lr=0.1)

        def step(x, y):
            opt.zero_grad()
            loss = F.linear_cross_entropy(norm_layer(x), fc.weight, y, fc.bias)
            loss.backward()
            opt.step()
            return loss.detach()

        return model, opt, step

    g = torch.Generator(device=DEV).manual_seed(0)
    x, y = torch.randn(48, 64, generator=g, device=DEV).bfloat16(), torch.randint(0, 200, (48,), generator=g, device=DEV)
    model, opt, step = make()
    twin, _, eager = make()
    saved = {k: v + 0.5 * torch.randn(v.shape, generator=g, device=DEV) for k, v in model.state_dict().items()}
    cap = CapturedStep(step, opt, (x, y), warmup=1)
    eager(x, y)
    for k in range(4):
        if k % 2 == 0:
            model.load_state_dict(saved), twin.load_state_dict(saved)
        a, b = cap(x, y), eager(x, y)
        torch.cuda.synchronize()
        assert torch.equal(a, b), k
        assert all(torch.equal(p, q) for p, q in zip(model.parameters(), twin.parameters())), k
