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
