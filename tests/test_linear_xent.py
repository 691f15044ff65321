"""Linear + cross entropy without the logits, against its formula in 64 bits.

Bounds, with u = 2^-24 and h = 2^-8 (half a step of bf16): a logit is a sum of D products in fp32, 16 at a
time: off by at most e = (D / 16 + 32) 2u sum|x w|. Exponentials and their sums add 64u for each power of
two of their argument's size and depth u for a sum of that depth. d = p - target is then off by
p (2e + ...) and rounded once to bf16 (h |d|); dx and dw sum d against w or x in fp32 and are rounded
to their own type once.
"""
import pytest
import torch

from deep_vision_amd import ops as F

DEV = "cuda"
U, H = 2.0 ** -24, 2.0 ** -8
BF16, F32 = torch.bfloat16, torch.float32
gpu = pytest.mark.gpu


def make(N, D, V, bias=True, ignored=0.0, seed=0, dev=DEV, logit=1.5, wdtype=BF16):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(N, D, generator=g, device=dev).to(BF16)
    w = (torch.randn(V, D, generator=g, device=dev) * (logit / D ** 0.5)).to(wdtype)
    b = 0.3 * torch.randn(V, generator=g, device=dev) if bias else None
    y = torch.randint(0, V, (N,), generator=g, device=dev)
    if ignored:
        y[torch.rand(N, generator=g, device=dev) < ignored] = -100
    return x, w, b, y


def oracle(x, w, b, y, smooth=0.0, ignore=-100, reduction="mean", go=None):
    """(loss, dx, dw, db) in 64 bits and the bound of each."""
    V, D, N = w.shape[0], w.shape[1], x.shape[0]
    keep = (y != ignore) & (y >= 0) & (y < V)
    x = torch.where(keep[:, None], x.double(), 0.0)
    w = w.to(BF16).double()  # the operand that the products use
    l = x @ w.t()
    size = x.abs() @ w.abs().t()
    if b is not None:
        l, size = l + b.double(), size + b.double().abs()
    lse = torch.logsumexp(l, 1)
    at = y.clamp(0, V - 1)[:, None]
    chosen = l.gather(1, at)[:, 0]
    fin = torch.where(l.isfinite(), l, 0.0)
    rows = lse - (1 - smooth) * chosen - (smooth * l.mean(1) if smooth else 0.0)
    rows = torch.where(keep, rows, 0.0)
    count = max(int(keep.sum()), 1)
    scale = keep.double() / (count if reduction == "mean" else 1)
    go = torch.ones(N if reduction == "none" else 1, dtype=torch.float64, device=x.device) if go is None else go.double()
    scale = scale * go
    p = torch.exp(l - lse[:, None])
    d = p - smooth / V
    d.scatter_add_(1, at, torch.full_like(d[:, :1], smooth - 1))
    d = torch.where(keep[:, None], d, 0.0)
    sd = scale[:, None] * d

    e_l = (D / 16 + 32) * 2 * U * torch.where(l.isfinite(), size, 0.0)
    depth = 128 + V / 128 + 64
    e_exp = 4 * U * (lse[:, None] - fin).abs().clamp(max=200) + 8 * U
    e_lse = (p * (e_l + e_exp)).sum(1) + depth * U + 4 * U * lse.abs()
    e_rows = e_lse + e_l.gather(1, at)[:, 0] + 4 * U * (lse.abs() + chosen.abs()) + 4 * U * rows.abs()
    if smooth:
        e_rows = e_rows + smooth * ((e_l + U * fin.abs()).mean(1) + depth * U * fin.abs().mean(1))
    e_d = p * (e_l + e_exp + e_lse[:, None]) + 4 * U * d.abs() + U * (1 + smooth / V)
    e_d = torch.where(keep[:, None], e_d, 0.0)
    a = scale.abs()[:, None]
    round_d = a * (e_d + H * (d.abs() + e_d))
    aw, ax, asd = w.abs(), x.abs(), sd.abs()
    tol_dx = round_d @ aw + (V / 16 + 96) * 2 * U * (asd @ aw)
    tol_dw = round_d.t() @ ax + (N / 16 + 96) * 2 * U * (asd.t() @ ax)
    tol_db = (a * e_d).sum(0) + (N / 32 + 64) * U * asd.sum(0)
    if reduction == "none":
        loss, tol = rows, e_rows
    else:
        k = count if reduction == "mean" else 1
        loss, tol = rows.sum() / k, (e_rows.sum() + (N / 64 + 64) * U * rows.abs().sum()) / k
    return (loss, sd @ w, sd.t() @ x, sd.sum(0)), (tol, tol_dx, tol_dw, tol_db)


def check(name, got, want, tol, dtype):
    got = got.double()
    half = torch.finfo(dtype).eps / 2
    bound = 1.01 * tol + half * (want.abs() + tol) + 1e-30
    assert got.shape == want.shape, name
    assert torch.equal(got.isfinite(), want.isfinite()), name
    ok = want.isfinite()
    worst = ((got - want).abs()[ok] / bound[ok]).max().item() if ok.any() else 0.0
    assert worst <= 1, f"{name}: {worst:.3g} times its bound"


def run_and_check(x, w, b, y, smooth=0.0, ignore=-100, reduction="mean", go=None):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    b = b.detach().requires_grad_() if b is not None else None
    loss = F.linear_cross_entropy(x, w, y, b, label_smoothing=smooth, ignore_index=ignore, reduction=reduction)
    leaves = [x, w] + ([b] if b is not None else [])
    grads = torch.autograd.grad(loss, leaves, go if go is not None or reduction != "none" else torch.ones_like(loss))
    want, tol = oracle(x.detach(), w.detach(), b.detach() if b is not None else None, y, smooth, ignore, reduction, go)
    assert loss.dtype == F32 and grads[0].dtype == x.dtype and grads[1].dtype == w.dtype
    check("loss", loss.detach(), want[0], tol[0], F32)
    check("dx", grads[0], want[1], tol[1], BF16)
    check("dweight", grads[1], want[2], tol[2], w.dtype)
    if b is not None:
        check("dbias", grads[2], want[3], tol[3], F32)
    with torch.no_grad():
        assert torch.equal(loss, F.linear_cross_entropy(x, w, y, b, smooth, ignore, reduction))
    return loss, grads


# ---------------------------------------------------------------- refusals and the CPU form
def test_refusals():
    x, w, b, y = make(4, 6, 9, dev="cpu")
    f = F.linear_cross_entropy
    for args, kw, kind, text in (
            ((x, w[:, :5], y), {}, ValueError, "does not match weight"), ((x, w[0], y), {}, ValueError, "does not match weight"),
            ((x, w[:0], y), {}, ValueError, "does not match weight"), ((x[:, :0], w[:, :0], y), {}, ValueError, "does not match"),
            ((x, w, y[:3]), {}, ValueError, "labels"), ((x, w, y[:, None]), {}, ValueError, "labels"),
            ((x, w, y.float()), {}, TypeError, "integers"), ((x, w, y > 0), {}, TypeError, "integers"),
            ((x, w, y, b[:8]), {}, ValueError, "bias has shape"), ((x, w, y, b[:, None]), {}, ValueError, "bias has shape"),
            ((x, w, y, b), dict(reduction="max"), ValueError, "reduction"),
            ((x, w, y, b), dict(label_smoothing=1.5), ValueError, "label_smoothing"),
            ((x, w, y, b), dict(label_smoothing=float("nan")), ValueError, "label_smoothing"),
            ((x, w.to("meta"), y), {}, ValueError, "all tensors must be on"),
            ((x, w, y, b.to("meta")), {}, ValueError, "all tensors must be on")):
        with pytest.raises(kind, match=text):
            f(*args, **kw)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cpu_form(reduction):
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((7, 5), (11, 5), (11,)))
    y = torch.tensor([0, 3, -100, 10, 2, 5, 5])
    a = F.linear_cross_entropy(x, w, y, b, 0.1, reduction=reduction)
    c = torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, w, b), y, label_smoothing=0.1, reduction=reduction)
    torch.testing.assert_close(a, c)
    for p, q in zip(torch.autograd.grad(a.sum(), (x, w, b)), torch.autograd.grad(c.sum(), (x, w, b))):
        torch.testing.assert_close(p, q)
    y2 = torch.where(y == -100, torch.tensor(11), y)  # outside the classes: left out as well
    with torch.no_grad():
        x[2] = float("nan")
    a = F.linear_cross_entropy(x, w, y2, b, 0.1, reduction=reduction)
    torch.testing.assert_close(a, c)
    dx, dw = torch.autograd.grad(a.sum(), (x, w))
    assert not dx[2].any() and dw.isfinite().all()
    assert F.linear_cross_entropy(x, w, torch.full_like(y, -1), b).item() == 0.0


# ---------------------------------------------------------------- numerics
SHAPES = [(1, 8, 1), (1, 64, 2), (2, 65, 10), (3, 100, 257), (8, 2048, 1000), (63, 128, 255), (64, 64, 256), (65, 1021, 64),
          (130, 192, 1001), (257, 256, 513), (256, 2048, 1000), (300, 72, 4999), (771, 1021, 2011), (1024, 128, 8192),
          (2500, 64, 7), (5000, 40, 130), (16, 4096, 12000)]


@gpu
@pytest.mark.parametrize("N,D,V", SHAPES)
def test_shapes(N, D, V):
    run_and_check(*make(N, D, V, bias=True, ignored=0.15))
    run_and_check(*make(N, D, V, bias=False, seed=1), smooth=0.1)


@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smooth", [0.0, 0.1, 1.0])
def test_reductions(reduction, smooth):
    x, w, b, y = make(150, 96, 333, ignored=0.2)
    go = torch.randn(150 if reduction == "none" else 1, device=DEV)
    run_and_check(x, w, b, y, smooth, reduction=reduction, go=go if reduction == "none" else go[0])


@gpu
def test_several_pieces_of_the_vocabulary():
    run_and_check(*make(4096, 64, 70000, bias=True, ignored=0.1))


# enough work that the products read the weight and the logits' gradient k by k
@gpu
@pytest.mark.parametrize("N,D,V,reduction", [(999, 2045, 8191, "none"), (2001, 1021, 16381, "mean"), (8101, 1500, 1999, "sum"),
                                             (2001, 2048, 8190, "none")])
def test_large_shapes_with_odd_ends(N, D, V, reduction):
    x, w, b, y = make(N, D, V, bias=True, ignored=0.15)
    go = torch.randn(N, device=DEV) if reduction == "none" else None
    run_and_check(x, w, b, y, 0.1, reduction=reduction, go=go)
    clean = F.linear_cross_entropy(x.requires_grad_(), w.requires_grad_(), y, reduction=reduction)
    want = torch.autograd.grad(clean, (x, w), go)
    x = x.detach().clone()
    x[(y == -100).nonzero()[::2, 0]] = float("nan")  # whatever the rows hold that do not count
    # a weight in the middle of a buffer of NaN: nothing beside it takes part
    Dp = (D + 7) // 8 * 8
    hold = torch.full((V + 70, Dp + 64), float("nan"), dtype=BF16, device=DEV)
    inner = hold[3:V + 3, 8:8 + D]
    inner.copy_(w.detach())
    inner.requires_grad_()
    got = torch.autograd.grad(F.linear_cross_entropy(x.requires_grad_(), inner, y, reduction=reduction), (x, inner), go)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    p = torch.nn.Parameter(w.detach().float())
    got = torch.autograd.grad(F.linear_cross_entropy(x.nan_to_num(), p, y, reduction=reduction), p, go)[0]
    assert torch.equal(got.to(BF16), want[1])


@gpu
def test_several_large_pieces_with_odd_ends():
    run_and_check(*make(12001, 1021, 45007, bias=True, ignored=0.1))


@gpu
def test_wide_logits_and_classes_that_are_ruled_out():
    x, w, b, y = make(70, 64, 900, logit=40.0)
    run_and_check(x, w, b, y)
    b = b.clone()
    y = y % 300 + 600
    b[:512] = float("-inf")  # whole tiles of the vocabulary
    loss, grads = run_and_check(x, w, b, y)
    assert not grads[1][:512].any() and not grads[2][:512].any()
    b[:512] = torch.finfo(F32).min
    run_and_check(x, w, b, y)
    b[:] = torch.finfo(F32).min  # every class: all logits round to the same value
    loss = F.linear_cross_entropy(x, w, y, b, reduction="none")
    torch.testing.assert_close(loss, torch.full_like(loss, torch.finfo(F32).min).sub(torch.finfo(F32).min).add(900.0).log())
    wr = w.detach().clone().requires_grad_()
    g = torch.autograd.grad(F.linear_cross_entropy(x, wr, y, b), wr)[0]
    assert g.isfinite().all()


@gpu
def test_rows_that_do_not_count():
    x, w, b, y = make(200, 128, 500, ignored=0.3)
    keep = y >= 0
    clean = run_and_check(x, w, b, y)
    dirty = x.clone()
    dirty[~keep] = float("nan")
    dirty[(~keep).nonzero()[0]] = float("inf")
    for ignore, lab in ((-100, y), (7, torch.where(keep, torch.where(y == 7, 8, y), 7)), (-100, torch.where(keep, y, 500)),
                        (-100, torch.where(keep, y, 2 ** 40))):
        got = run_and_check(dirty, w, b, lab, ignore=ignore)
        assert not got[1][0][~keep].any()
        if ignore == -100:
            assert torch.equal(got[0], clean[0]) and all(torch.equal(p, q) for p, q in zip(got[1], clean[1]))
    none = torch.full_like(y, -100)
    for reduction in ("mean", "sum", "none"):
        loss, grads = run_and_check(dirty, w, b, none, reduction=reduction)
        assert not loss.any() and not any(g.any() for g in grads)
    rows = F.linear_cross_entropy(dirty, w, y, b, reduction="none")
    assert rows.isfinite().all() and not rows[~keep].any()
    bad = x.clone()
    bad[5] = float("nan")
    y5 = y.clone()
    y5[5] = 3
    assert F.linear_cross_entropy(bad, w, y5, b).isnan()


@gpu
def test_layouts_and_types():
    x, w, b, y = make(90, 256, 600)
    want = run_and_check(x, w, b, y)
    wide = torch.randn(90, 300, device=DEV).to(BF16)
    for off in (0, 8, 3):
        wide[:, off:off + 256] = x
        got = run_and_check(wide[:, off:off + 256], w, b, y)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1][0], want[1][0])
    got = run_and_check(x.t().contiguous().t(), w.t().contiguous().t(), b, y.int())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1][1], want[1][1])
    run_and_check(x[:1].expand(90, 256), w, b, y)
    # several leading dimensions, fp32 inputs
    loss = F.linear_cross_entropy(x.view(9, 10, 256), w, y.view(9, 10), b, reduction="none")
    assert loss.shape == (9, 10) and torch.equal(loss.view(-1), F.linear_cross_entropy(x, w, y, b, reduction="none"))
    xf = x.float().requires_grad_()
    g = torch.autograd.grad(F.linear_cross_entropy(xf, w, y, b), xf)[0]
    assert g.dtype == F32 and torch.equal(g.to(BF16), want[1][0])
    run_and_check(x, w.float(), b, y)  # an fp32 weight that is no parameter
    p = torch.nn.Parameter(make(90, 256, 600, wdtype=F32)[1])
    run_and_check(x, p.detach(), b, y)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        F.linear_cross_entropy(x.half(), w, y)
    with pytest.raises(TypeError, match="weight must be"):
        F.linear_cross_entropy(x, w.half(), y)
    with pytest.raises(TypeError, match="bias must be"):
        F.linear_cross_entropy(x, w, y, b.to(BF16))


@gpu
def test_no_rows():
    x, w, b, y = make(0, 64, 30)
    for t in (x, w, b):
        t.requires_grad_()
    for reduction in ("mean", "sum", "none"):
        loss = F.linear_cross_entropy(x, w, y, b, reduction=reduction)
        assert not loss.any() and loss.numel() == (0 if reduction == "none" else 1)
        grads = torch.autograd.grad(loss.sum(), (x, w, b))
        assert not any(g.any() for g in grads)


@gpu
def test_gradient_against_differences():
    """x and w on a grid of 1/64 below 2, so that a step of 1/64 stays exact in bf16: the central
    difference of the fp32 loss is the derivative up to t^2 / 6 of the third one (some 1e-4 here) and
    the loss's own 1e-6 over t."""
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randint(-64, 65, (32, 64), generator=g, device=DEV).float() / 64
    w = torch.randint(-32, 33, (100, 64), generator=g, device=DEV).float() / 64
    y = torch.randint(0, 100, (32,), generator=g, device=DEV)
    b = torch.zeros(100, device=DEV)
    _, grads = run_and_check(x.to(BF16), w.to(BF16), b, y, smooth=0.1)
    t = 1 / 64
    for i, leaf in enumerate((x, w, b)):
        for s in range(4):
            d = torch.randint(-1, 2, leaf.shape, generator=g, device=DEV).float()

            def f(k):
                a = [v + k * t * d if j == i else v for j, v in enumerate((x, w, b))]
                return F.linear_cross_entropy(a[0].to(BF16), a[1].to(BF16), y, a[2], 0.1).double()

            diff, inner = (f(1) - f(-1)) / (2 * t), (grads[i].double() * d.double()).sum()
            size = grads[i].double().norm() * d.double().norm()
            assert (diff - inner).abs() < 1e-2 * size + 1e-4, (i, s)


@gpu
def test_a_weight_past_32_bits_of_elements():
    V, D = (1 << 20) + 5, 2112
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.empty(V, D, dtype=BF16, device=DEV)
    for i in range(0, V, 1 << 16):
        n = min(1 << 16, V - i)
        w[i:i + n] = torch.randn(n, D, generator=g, device=DEV) * 0.03
    x = torch.randn(5, D, generator=g, device=DEV).to(BF16).requires_grad_()
    y = torch.tensor([0, V - 1, V - 2, 7, -100], device=DEV)
    w.requires_grad_()
    loss = F.linear_cross_entropy(x, w, y)
    dx, dw = torch.autograd.grad(loss, (x, w))
    with torch.no_grad():
        l = torch.cat([x.float() @ w[i:i + (1 << 16)].float().t() for i in range(0, V, 1 << 16)], 1).double()[:4]
        lse = torch.logsumexp(l, 1)
        want = (lse - l.gather(1, y[:4, None])[:, 0]).mean()
        assert abs(loss.item() - want.item()) < 1e-4
        d = torch.exp(l - lse[:, None])
        d.scatter_add_(1, y[:4, None], torch.full((4, 1), -1.0, dtype=torch.float64, device=DEV))
        tail = (d[:, -9:] / 4).t() @ x[:4].double()
        assert (dw[-9:].double() - tail).norm() < 1e-2 * tail.norm()
        wdx = sum((d[:, i:i + (1 << 16)] / 4) @ w[i:i + (1 << 16)].double() for i in range(0, V, 1 << 16))
        assert (dx[:4].double() - wdx).norm() < 1e-2 * wdx.norm() and not dx[4].any()


# ---------------------------------------------------------------- as a program uses it
@gpu
def test_parameters_of_a_layer_and_their_gradient_buffers():
    from deep_vision_amd import nn as dnn
    from deep_vision_amd.train.optim import FusedSGD

    torch.manual_seed(0)
    head = dnn.Linear(200, 300).to(DEV)
    x, _, _, y = make(128, 200, 300)
    opt = FusedSGD(head.parameters(), lr=0.1)  # flat buffers: .grad is live from here on
    opt.zero_grad()
    x.requires_grad_()
    ref = torch.autograd.grad(F.linear_cross_entropy(x, head.weight, y, head.bias), (x, head.weight, head.bias))
    assert not head.weight.grad.any()  # autograd.grad leaves the buffers alone
    want, tol = oracle(x.detach(), head.weight.detach(), head.bias.detach(), y)
    for n, g, i, t in (("dx", ref[0], 1, BF16), ("dweight", ref[1], 2, F32), ("dbias", ref[2], 3, F32)):
        check(n, g, want[i], tol[i], t)
    buf = head.weight.grad
    F.linear_cross_entropy(x, head.weight, y, head.bias).backward()
    assert head.weight.grad is buf and torch.equal(buf, ref[1]) and torch.equal(head.bias.grad, ref[2])
    (2 * F.linear_cross_entropy(x, head.weight, y, head.bias)).backward()
    torch.testing.assert_close(buf, 3 * ref[1])
    before = head.weight.detach().clone()
    opt.step()  # the cached operands follow the parameters
    assert not torch.equal(before, head.weight)
    a = F.linear_cross_entropy(x, head.weight, y, head.bias)
    b = F.linear_cross_entropy(x, head.weight.detach().clone(), y, head.bias)
    assert torch.equal(a, b)


@gpu
def test_some_gradients_only_and_a_retained_graph():
    x, w, b, y = make(100, 128, 400, ignored=0.1)
    full = run_and_check(x, w, b, y)[1]
    for which in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        leaves = [t.detach().clone().requires_grad_(i in which) for i, t in enumerate((x, w, b))]
        loss = F.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2])
        got = torch.autograd.grad(loss, [leaves[i] for i in which], retain_graph=True)
        again = torch.autograd.grad(loss, [leaves[i] for i in which])
        for i, g, h in zip(which, got, again):
            assert torch.equal(g, full[i]) and torch.equal(g, h)


@gpu
def test_saved_tensors_kept_elsewhere_and_recomputation():
    from torch.utils.checkpoint import checkpoint

    wide, w, b, y = make(50, 200, 300)
    for x in (wide[:, :128], wide[:, 3:103]):  # used in place, and packed
        x = x.detach().requires_grad_()
        wx, bx = w[:, :x.shape[1]].detach().clone().requires_grad_(), b.clone().requires_grad_()
        want = torch.autograd.grad(F.linear_cross_entropy(x, wx, y, bx), (x, wx, bx))
        with torch.autograd.graph.save_on_cpu():
            loss = F.linear_cross_entropy(x, wx, y, bx)
        got = torch.autograd.grad(loss, (x, wx, bx))
        again = torch.autograd.grad(checkpoint(lambda t: F.linear_cross_entropy(t, wx, y, bx), x, use_reentrant=False),
                                    (x, wx, bx))
        assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, got, again))


@gpu
def test_what_changes_between_the_passes_is_refused():
    x, w, b, y = make(20, 64, 90)
    w.requires_grad_()
    loss = F.linear_cross_entropy(x, w, y, b)
    y[0] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    loss = F.linear_cross_entropy(x, w, y, b)
    g = torch.autograd.grad(loss, w, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivative"):
        g.sum().backward()


@gpu
def test_shared_weight_and_broadcast_rows():
    """One weight as classifier twice and in an elementwise term, one row broadcast to a batch: autograd
    adds what each use gives (sums of bf16 gradients: h of the largest partial sum each)."""
    x, w, b, y = make(40, 128, 200)
    row = x[:1].detach().clone().requires_grad_()
    w = w.requires_grad_()
    one = torch.autograd.grad(F.linear_cross_entropy(row.expand(40, 128), w, y, b), (row, w))
    two = torch.autograd.grad(F.linear_cross_entropy(x, w, y, b), w)[0]
    loss = F.linear_cross_entropy(row.expand(40, 128), w, y, b) + F.linear_cross_entropy(x, w, y, b) + w.float().sum()
    got = torch.autograd.grad(loss, (row, w))
    assert torch.equal(got[0], one[0])
    want = one[1].double() + two.double() + 1
    assert ((got[1].double() - want).abs() <= 2 * H * (one[1].double().abs() + two.double().abs() + 1)).all()


@gpu
def test_two_streams_and_a_replayed_graph():
    x, w, b, y = make(512, 256, 3000, ignored=0.1)
    want = run_and_check(x, w, b, y)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]

    def step():
        loss = F.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2])
        return loss.detach(), torch.autograd.grad(loss, leaves)

    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for loss, grads in got:
        assert torch.equal(loss, want[0]) and all(torch.equal(p, q) for p, q in zip(grads, want[1]))
    del got, loss, grads
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        out = step()
    for k in range(3):
        nx, _, _, ny = make(512, 256, 3000, ignored=0.1, seed=k)
        with torch.no_grad():
            leaves[0].copy_(nx)
        y.copy_(ny)
        graph.replay()
        torch.cuda.synchronize()
        loss, grads = run_and_check(nx, w, b, ny)
        assert torch.equal(loss, out[0]) and all(torch.equal(p, q) for p, q in zip(out[1], grads))


@gpu
def test_more_classes_than_a_launch_of_the_smallest_tiles_holds():
    """2^28 classes in tiles of 32 x 32 would be 2^32 threads. A logit is off by (64 / 16 + 32) 2u sum|x w| (the module's
    bound), some 1e-4; the gradients are held to 1 % of their norms (d is rounded to bf16, h = 0.4 %)."""
    V, D, N = (1 << 28) + 5, 64, 3
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.empty(V, D, dtype=BF16, device=DEV)
    step = 1 << 24
    for i in range(0, V, step):
        n = min(step, V - i)
        w[i:i + n] = torch.randn(n, D, generator=g, device=DEV).mul_(0.2)
    x = torch.randn(N, D, generator=g, device=DEV).to(BF16).requires_grad_()
    y = torch.tensor([V - 1, 0, 1 << 27], device=DEV)
    w.requires_grad_()
    loss = F.linear_cross_entropy(x, w, y, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    with torch.no_grad():
        lse, chosen = torch.full((N,), -float("inf"), dtype=torch.float64, device=DEV), torch.zeros(N, dtype=torch.float64, device=DEV)
        for i in range(0, V, step):
            l = (x.float() @ w[i:i + step].float().t()).double()
            lse = torch.logaddexp(lse, torch.logsumexp(l, 1))
            for n in range(N):
                if i <= y[n] < i + step:
                    chosen[n] = l[n, y[n] - i]
        assert abs(loss.item() - (lse - chosen).sum().item()) < 1e-3
        want = torch.zeros(N, D, dtype=torch.float64, device=DEV)
        for i in range(0, V, step):
            part = w[i:i + step].float()
            d = torch.exp((x.float() @ part.t()).double() - lse[:, None])
            for n in range(N):
                if i <= y[n] < i + step:
                    d[n, y[n] - i] -= 1
            want += (d.float() @ part).double()
            if i + step >= V or i == 0:
                rows = d.t() @ x.double()
                assert (dw[i:i + step].double() - rows).norm() < 1e-2 * rows.norm()
        assert (dx.double() - want).norm() < 1e-2 * want.norm()
