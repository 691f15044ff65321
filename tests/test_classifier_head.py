"""The training end of a classifier as one run: layer norm, linear cross entropy, AdamW.

Bounds of the gradients against 64 bits, relative to their norms, with h = 2^-8 (half a step of bf16): the
normalised rows are rounded to bf16 (h each, and w x + b of them again through every logit), the
gradient of the logits is rounded (h), the gradient of the rows is rounded (h), and rounded products
meet in sums of independent terms: 4 h of the norm covers the four roundings in a row.
"""
import math

import pytest
import torch

from deep_vision_amd import nn as dnn
from deep_vision_amd import ops as F
from deep_vision_amd.train.optim import OPTIMIZERS

DEV = "cuda"
H, U = 2.0 ** -8, 2.0 ** -24
KW = dict(lr=3e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.02)


class Head(torch.nn.Module):
    def __init__(self, width, classes):
        super().__init__()
        self.norm = dnn.LayerNorm(width)
        self.fc = dnn.Linear(width, classes)

    def forward(self, x, labels):
        return F.linear_cross_entropy(self.norm(x), self.fc.weight, labels, self.fc.bias, label_smoothing=0.1)


def batch(rows, width, classes, seed, dev):
    g = torch.Generator().manual_seed(seed)
    y = torch.randint(0, classes, (rows,), generator=g)
    x = torch.randn(rows, width, generator=g) + torch.randn(classes, width, generator=torch.Generator().manual_seed(1))[y]
    # a padded batch; what its rows hold is finite (the loss would drop a NaN, but layer norm's weight
    # gradient is a sum over every row, and 0 * NaN is NaN by its formula)
    y[-rows // 8:] = -100
    x[-rows // 8:] = 1000.0 * torch.arange(width)
    return x.to(dev, torch.bfloat16), y.to(dev)


def make(width, classes, bits, dev):
    torch.manual_seed(0)
    head = Head(width, classes).to(dev)
    return head, OPTIMIZERS["AdamW"](head.parameters(), **KW, state_bits=bits, seed=3)


def exact_gradients(head, x, y):
    w, b, fw, fb = (p.detach().double().requires_grad_() for p in head.parameters())
    keep = y >= 0
    z = torch.nn.functional.layer_norm(x[keep].double(), (x.shape[1],), w, b)
    loss = torch.nn.functional.cross_entropy(z @ fw.t() + fb, y[keep], label_smoothing=0.1)
    return loss, torch.autograd.grad(loss, (w, b, fw, fb))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
def test_steps_against_64_bits(bits, dev):
    head, opt = make(96, 203, bits, dev)
    for step in range(1, 6):
        x, y = batch(64, 96, 203, step, dev)
        want_loss, want = exact_gradients(head, x, y)
        opt.zero_grad()
        loss = head(x, y)
        loss.backward()
        assert abs(loss.item() - want_loss.item()) <= 4 * H * 2  # logits of size 2
        before = [p.detach().double().clone() for p in head.parameters()]
        for p, g in zip(head.parameters(), want):
            assert p.grad.isfinite().all()
            assert (p.grad.double() - g).norm() <= 4 * H * g.norm()
        m0 = [{k: v.double() for k, v in s.items() if k != "step"} for s in opt.state_dict()["state"].values()]
        opt.step()
        for i, (p, q) in enumerate(zip(head.parameters(), before)):
            g = p.grad.double().reshape(-1)
            if not m0:
                m, v = torch.zeros_like(g), torch.zeros_like(g)
            elif bits == 32:
                m, v = m0[i]["exp_avg"].reshape(-1), m0[i]["exp_avg_sq"].reshape(-1)
            else:
                m, v = ((m0[i][k].view(-1, 256) * m0[i][k + "_scale"][:, None]).reshape(-1)[:g.numel()]
                        for k in ("exp_avg", "exp_avg_root"))
                v = v * v
            # m is a sum of two rounded products: off by up to 2^-24 of each and of the sum, whatever cancels
            terms = 0.9 * m.abs() + 0.1 * g.abs()
            m, v = 0.9 * m + 0.1 * g, 0.98 * v + 0.02 * g * g
            per = KW["lr"] / (1 - 0.9 ** step) / ((v / (1 - 0.98 ** step)).sqrt() + KW["eps"])
            move = per * m
            want_p = (q * (1 - KW["lr"] * KW["weight_decay"])).reshape(-1) - move
            bound = 4 * U * want_p.abs() + 32 * U * per * terms + 1e-12
            assert ((p.detach().double().reshape(-1) - want_p).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_are_the_eager_ones(bits):
    """The whole step replayed from a graph: losses and parameters of the eager run, bit for bit but for the
    bias corrections (in 32 bits on the device, 64 on the host)."""
    from deep_vision_amd.train.graph import CapturedStep

    def step_of(head, opt):
        def step(x, y):
            opt.zero_grad()
            loss = head(x, y)
            loss.backward()
            opt.step()
            return loss.detach()
        return step

    a, oa = make(256, 1000, bits, DEV)
    b, ob = make(256, 1000, bits, DEV)
    x, y = batch(128, 256, 1000, 0, DEV)
    cap = CapturedStep(step_of(a, oa), oa, (x.clone(), y.clone()))
    eager = step_of(b, ob)
    for _ in range(2):  # the capture's warm-up steps
        eager(x, y)
    for k in range(1, 5):
        x, y = batch(128, 256, 1000, k, DEV)
        la, lb = cap(x, y).clone(), eager(x, y)
        torch.cuda.synchronize()
        torch.testing.assert_close(la, lb, rtol=2e-3, atol=2e-3)
        for p, q in zip(a.parameters(), b.parameters()):
            assert (p - q).norm() <= 1e-3 * q.norm()


@pytest.mark.gpu
def test_two_graphs_of_one_head():
    """Two captured passes over the same parameters, replayed in turn and with eager passes between them:
    neither leaves anything in the other's way."""
    head, _ = make(128, 500, 32, DEV)
    inputs = [batch(64, 128, 500, k, DEV) for k in range(2)] + [batch(96, 128, 500, 7, DEV)]
    params = list(head.parameters())

    def grads(x, y):
        loss = head(x, y)
        return [loss.detach()] + list(torch.autograd.grad(loss, params))

    want = [grads(x, y) for x, y in inputs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for x, y in inputs:
            grads(x, y)
    torch.cuda.synchronize()
    graphs = []
    for x, y in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = grads(x, y)
        graphs.append((g, out))
    for order in ((0, 1, 2), (2, 0, 1, 0), (1, 1, 2)):
        for i in order:
            graphs[i][0].replay()
        eager = grads(*inputs[0])
        torch.cuda.synchronize()
        for i in set(order):
            assert all(torch.equal(p, q) for p, q in zip(graphs[i][1], want[i]))
        assert all(torch.equal(p, q) for p, q in zip(eager, want[0]))
        del eager
