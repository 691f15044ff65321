"""Layer norm against its formula in 64 bits.

Bounds, with u = 2^-24: a mean over D columns is summed in at most 80 rounded additions one after
another (32 per lane and 9 across lanes, or 20 per lane of the widest rows tested), so it is off by
at most 80 u mean|x|; a product or quotient by u. The output's own rounding is half a step of its type.
"""
import pytest
import torch

from deep_vision_amd import nn as dnn
from deep_vision_amd import ops as F

DEV = "cuda"
U = 2.0 ** -24
DEPTH = 80
gpu = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def oracle(x, w, b, dy, eps=1e-5):
    """y, dx, dw, db in 64 bits, and the bound of each one's error in 32."""
    D = x.shape[-1]
    x, dy = x.double().reshape(-1, D), dy.double().reshape(-1, D)
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(D, dtype=torch.float64, device=x.device) if b is None else b.double()
    mu = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mu).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (x - mu) * rstd
    y = xh * w + b
    h = dy * w
    dx = rstd * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
    e_mu = DEPTH * U * x.abs().mean(1, keepdim=True)
    e_xh = rstd * (e_mu + U * (x - mu).abs()) + xh.abs() * (DEPTH + 4) * U  # (x - mu) and rstd
    # the mean's error shifts (x - mu) as a whole: it enters the variance squared, and by cross terms it is cancelled from
    e_xh = e_xh + xh.abs() * rstd * rstd * e_mu * e_mu
    tol_y = w.abs() * e_xh + 3 * U * (y.abs() + b.abs())
    s1, s2 = h.abs().mean(1, keepdim=True), (h * xh).abs().mean(1, keepdim=True)
    e_q = (DEPTH + 2) * U * s2 + (h.abs() * e_xh).mean(1, keepdim=True)
    q = (h * xh).mean(1, keepdim=True).abs()
    tol_dx = rstd * (4 * U * h.abs() + DEPTH * U * s1 + xh.abs() * e_q + q * e_xh) + (DEPTH + 8) * U * dx.abs() \
        + 4 * U * rstd * (s1 + xh.abs() * s2)
    depth = x.shape[0] / 64 + 128  # rows of a block, the block's groups, the slab
    tol_dw = (dy.abs() * e_xh).sum(0) + depth * U * (dy * xh).abs().sum(0)
    tol_db = depth * U * dy.abs().sum(0)
    return (y, dx, (dy * xh).sum(0), dy.sum(0)), (tol_y, tol_dx, tol_dw, tol_db)


def check(name, got, want, tol, dtype=torch.float32):
    got = got.double().reshape(want.shape)
    bound = tol * 1.01 + half_step(dtype) * (want.abs() + tol) + 1e-30
    worst = ((got - want).abs() / bound).max().item() if want.numel() else 0.0
    assert worst <= 1, f"{name}: {worst:.3g} times its bound"


def run_and_check(x, w, b, dy, eps=1e-5):
    x = x.detach().requires_grad_()
    leaves = [x] + [t.requires_grad_() for t in (w, b) if t is not None]
    y = F.layer_norm(x, (x.shape[-1],), w, b, eps)
    grads = torch.autograd.grad(y, leaves, dy)
    want, tol = oracle(x.detach(), w.detach() if w is not None else None, b.detach() if b is not None else None, dy, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and grads[0].dtype == x.dtype
    check("y", y.detach(), want[0], tol[0], x.dtype)
    check("dx", grads[0], want[1], tol[1], x.dtype)
    if w is not None:
        check("dweight", grads[1], want[2], tol[2])
    if b is not None:
        check("dbias", grads[-1], want[3], tol[3])
    return y, grads


def make(rows, D, dtype, dev=DEV, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, D, generator=g, device=dev) * 2 + 0.5
    dy = torch.randn(rows, D, generator=g, device=dev)
    w = 1 + 0.3 * torch.randn(D, generator=g, device=dev)
    b = 0.3 * torch.randn(D, generator=g, device=dev)
    return x.to(dtype), w, b, dy.to(dtype)


# ---------------------------------------------------------------- refusals and the CPU form
def test_refusals():
    x, w = torch.randn(4, 6), torch.randn(6)
    with pytest.raises(ValueError, match="last dimensions"):
        F.layer_norm(x, (5,))
    with pytest.raises(ValueError, match="last dimensions"):
        F.layer_norm(x, (2, 4, 6))
    with pytest.raises(ValueError, match="last dimensions"):
        F.layer_norm(x, ())
    with pytest.raises(ValueError, match="weight has shape"):
        F.layer_norm(x, (6,), w[:5])
    with pytest.raises(ValueError, match="bias has shape"):
        F.layer_norm(x, (6,), w, w[:, None])
    for eps in (0.0, -1e-5, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            F.layer_norm(x, (6,), eps=eps)
    with pytest.raises(ValueError, match="all tensors must be on"):
        F.layer_norm(x, (6,), torch.empty(6, device="meta"))


def test_cpu_matches_torch():
    x, w, b, dy = make(5, 33, torch.float32, "cpu")
    torch.testing.assert_close(F.layer_norm(x, 33, w, b), torch.nn.functional.layer_norm(x, (33,), w, b))
    assert F.layer_norm(x.bfloat16(), 33, w, b).dtype == torch.bfloat16
    m = dnn.LayerNorm(33)
    torch.testing.assert_close(m(x), torch.nn.LayerNorm(33)(x))
    assert list(m.state_dict()) == ["weight", "bias"]


@pytest.mark.parametrize("op", ["layer_norm", "linear_cross_entropy"])
def test_capture_is_refused_for_leaves_behind_a_view_or_a_cast(monkeypatch, op):
    """The ops reshape and cast what they are given: the leaves that count are the caller's."""
    from deep_vision_amd.ops import common, loss, norm

    now = {"stream": 1, "capturing": False}
    monkeypatch.setattr(common, "stream_handle", lambda: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    for m in (norm, loss):
        monkeypatch.setattr(m, "native", lambda x: True)
    monkeypatch.setattr(norm, "_forward", lambda x, ld, w, b, eps, train: (x * 1, None))
    monkeypatch.setattr(loss, "_linear_xent_forward", lambda x, w, b, y, *a: (x.float().sum(), (y, x, w, b, None)))
    x = torch.randn(3, 2, 8)
    if op == "layer_norm":
        w, b = torch.ones(2, 8), torch.zeros(2, 8)
        leaves, call = (x, w, b), lambda: norm.layer_norm(x, (2, 8), w, b)
    else:
        w, y = torch.randn(5, 8).to(torch.bfloat16), torch.zeros(3, 2, dtype=torch.int64)
        leaves, call = (x, w), lambda: loss.linear_cross_entropy(x, w, y)
    for leaf in leaves:
        leaf.requires_grad_()
        now.update(stream=1, capturing=False)
        alive = call()
        now.update(stream=2, capturing=True)
        with pytest.raises(RuntimeError, match="still alive"):
            call()
        del alive
        call()
        leaf.requires_grad_(False)


def test_no_sink_while_a_graph_of_another_stream_lives(monkeypatch):
    """The accumulation node would belong to the other stream, which nothing orders behind an in-place sum."""
    from deep_vision_amd.ops import common

    now = {"stream": 1}
    monkeypatch.setattr(common, "stream_handle", lambda: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    sank = []

    class Fn(torch.autograd.Function):
        @staticmethod
        def forward(ctx, w):
            common.track_leaves(ctx, w)
            ctx.save_for_backward(w)
            return w * 2

        @staticmethod
        def backward(ctx, g):
            sink = common.accumulation_sink(ctx, 0, ctx.saved_tensors[0])
            sank.append(sink is not None)
            if sink is None:
                return g * 2
            sink.add_(g * 2)

    w = torch.nn.Parameter(torch.ones(3))
    w.grad = torch.zeros(3)
    Fn.apply(w).sum().backward()
    kept = Fn.apply(w)
    now["stream"] = 2
    Fn.apply(w).sum().backward()
    del kept
    Fn.apply(w).sum().backward()
    assert sank == [True, False, True] and torch.equal(w.grad, torch.full((3,), 6.0))


def test_capture_is_refused_while_an_eager_graph_lives(monkeypatch):
    """The bookkeeping of track_leaves on the CPU: another stream's live graph of the same leaf."""
    from deep_vision_amd.ops import common

    now = {"stream": 1, "capturing": False}
    monkeypatch.setattr(common, "stream_handle", lambda: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])

    class Fn(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            common.track_leaves(ctx, x)
            return x * 2

        @staticmethod
        def backward(ctx, g):
            return g * 2

    x = torch.randn(3, requires_grad=True)
    y = Fn.apply(x)
    now.update(stream=2, capturing=True)
    with pytest.raises(RuntimeError, match="still alive"):
        Fn.apply(x)
    Fn.apply(x * 1)  # not a leaf: nothing accumulates into it
    now["stream"] = 1
    z = Fn.apply(x)  # the eager graph's own stream
    now["stream"] = 2
    del y, z
    Fn.apply(x)


# ---------------------------------------------------------------- numerics
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [1, 2, 7, 8, 63, 64, 127, 128, 129, 255, 256, 257, 512, 1000, 1001, 1024, 2047, 2048, 2049,
                               4096, 4100, 8192, 8200, 16384, 16385, 20000])
def test_widths(D, dtype):
    for rows in (1, 3, 67):
        run_and_check(*make(rows, D, dtype))


@gpu
@pytest.mark.parametrize("rows,D,dtype", [(5000, 256, torch.bfloat16), (4099, 96, torch.float32), (3001, 2048, torch.bfloat16),
                                          (1500, 1024, torch.float32), (700, 4096, torch.bfloat16)])
def test_many_rows(rows, D, dtype):
    run_and_check(*make(rows, D, dtype))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(dtype):
    wide, w, b, dy = make(37, 1016, dtype)
    for x, g in ((wide[:, :1001], dy[:, :1001]), (wide[:, 1:1002], dy[:, 3:1004]), (wide[::2, 5:1006], dy[::2, 5:1006])):
        run_and_check(x, w[:1001].clone(), b[:1001].clone(), g)
    run_and_check(wide[:, ::2], w[:508].clone(), b[:508].clone(), dy[:, ::2])  # columns apart
    run_and_check(wide.t()[:64], w[:37].clone(), b[:37].clone(), dy.t()[:64])
    run_and_check(wide[:1].expand(9, 1016), w.clone(), b.clone(), dy[:1].expand(9, 1016))
    x4, _, _, g4 = make(2 * 5 * 6, 40, dtype)  # a channels-last feature map, normalised over its channels
    x4 = x4.view(2, 5, 6, 40).permute(0, 3, 1, 2)
    run_and_check(x4.permute(0, 2, 3, 1), w[:40].clone(), b[:40].clone(), g4.view(2, 5, 6, 40))
    run_and_check(x4.permute(0, 2, 3, 1)[..., :33], w[:33].clone(), b[:33].clone(), g4.view(2, 5, 6, 40)[..., :33])


@gpu
def test_parts_of_the_gradient_and_no_affine():
    x, w, b, dy = make(19, 100, torch.float32)
    full = run_and_check(x, w, b, dy)[1]
    run_and_check(x, None, None, dy)
    run_and_check(x, w.detach(), None, dy)
    run_and_check(x, None, b.detach(), dy)
    xs, ws, bs = x.clone().requires_grad_(), w.detach().clone().requires_grad_(), b.detach().clone().requires_grad_()
    for leaves, k in (((xs,), (0,)), ((ws,), (1,)), ((bs,), (2,)), ((xs, bs), (0, 2))):
        use = [t if any(t is leaf for leaf in leaves) else t.detach() for t in (xs, ws, bs)]
        got = torch.autograd.grad(F.layer_norm(use[0], (100,), use[1], use[2]), leaves, dy)
        for g, i in zip(got, k):
            assert torch.equal(g, full[i])
    with torch.no_grad():
        assert not F.layer_norm(xs, (100,), ws, bs).requires_grad
    y = F.layer_norm(xs, (100,), ws, bs)
    assert torch.equal(y, F.layer_norm(x, (100,), w.detach(), b.detach()))


@gpu
def test_several_dimensions_and_empty_inputs():
    x, w, b, dy = make(6, 60, torch.bfloat16)
    y = F.layer_norm(x.view(2, 3, 4, 15), (4, 15), w.view(4, 15), b.view(4, 15))
    assert torch.equal(y.view(6, 60), F.layer_norm(x, 60, w, b))
    wv = w.view(4, 15).clone().requires_grad_()
    g = torch.autograd.grad(F.layer_norm(x.view(2, 3, 4, 15), (4, 15), wv, None), wv, dy.view(2, 3, 4, 15))[0]
    assert g.shape == (4, 15)
    e = torch.empty(0, 60, device=DEV, requires_grad=True)
    w2 = w.clone().requires_grad_()
    y = F.layer_norm(e, 60, w2, b)
    dx, dw = torch.autograd.grad(y, (e, w2), torch.empty_like(y))
    assert y.shape == (0, 60) and dx.shape == (0, 60) and not dw.any()
    with pytest.raises(ValueError, match="empty"):
        F.layer_norm(torch.empty(3, 0, device=DEV), 0)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        F.layer_norm(x.half(), 60)
    with pytest.raises(TypeError, match="must be float32"):
        F.layer_norm(x, 60, w.bfloat16())


@gpu
def test_a_mean_far_from_zero_and_values_that_are_not_finite():
    x, w, b, dy = make(9, 777, torch.float32)
    run_and_check(x + 1000.0, w, b, dy)
    run_and_check(torch.full_like(x, 3.25), w, b, dy)  # no variance: eps alone
    w, b = w.detach(), b.detach()
    good = F.layer_norm(x, 777, w, b)
    x[4, 100], x[6, 5] = float("inf"), float("nan")
    bad = F.layer_norm(x, 777, w, b)
    keep = torch.tensor([i not in (4, 6) for i in range(9)], device=DEV)
    assert torch.equal(bad[keep], good[keep]) and bad[4].isnan().all() and bad[6].isnan().all()


@gpu
def test_gradient_against_differences():
    """<grad, d> against (f(x + t d) - f(x - t d)) / 2t, f = sum(y * dy) with y from the kernel in 32
    bits: f is off by about 2^-24 sqrt(n) * 16 (each y's few roundings), the quotient by that over t;
    the third derivative's term is t^2 of order one."""
    x, w, b, dy = make(8, 96, torch.float32)
    y, grads = run_and_check(x, w, b, dy)
    t = 1e-2
    for i, leaf in enumerate((x, w, b)):
        d = torch.randn(leaf.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i))

        def f(s):
            a = [v.detach() + s * d if j == i else v.detach() for j, v in enumerate((x, w, b))]
            return (F.layer_norm(a[0], 96, a[1], a[2]).double() * dy.double()).sum()

        diff, inner = (f(t) - f(-t)) / (2 * t), (grads[i].double() * d.double()).sum()
        size = grads[i].double().norm() * d.double().norm()
        assert (diff - inner).abs() < 2e-3 * size + 16 * U * (8 * 96) ** 0.5 * 4 / t


# ---------------------------------------------------------------- as a program uses it
@gpu
def test_gradients_accumulate_into_a_live_buffer():
    x, w, b, dy = make(33, 200, torch.bfloat16)
    m = dnn.LayerNorm(200).to(DEV)
    with torch.no_grad():
        m.weight.copy_(w), m.bias.copy_(b)
    gw, gb = torch.autograd.grad(m(x), (m.weight, m.bias), dy)
    m.weight.grad, m.bias.grad = torch.full_like(w, 2.0), torch.full_like(b, -1.0)
    buf = m.weight.grad
    m(x).backward(dy)
    assert m.weight.grad is buf
    assert torch.equal(m.weight.grad, gw + 2) and torch.equal(m.bias.grad, gb - 1)
    only = torch.full_like(b, 0.5).requires_grad_()  # a bias without a weight
    only.grad = torch.ones_like(only)
    F.layer_norm(x, 200, None, only).backward(dy)
    assert torch.equal(only.grad, gb + 1)
    again = torch.autograd.grad(m(x), (m.weight, m.bias), dy)  # leaves .grad alone
    assert torch.equal(again[0], gw) and torch.equal(again[1], gb) and torch.equal(m.weight.grad, gw + 2)
    y = m(x)
    (y + m(x)).backward(dy)  # the same parameters twice in one graph
    torch.testing.assert_close(m.weight.grad, 3 * gw + 2)


@gpu
def test_saved_tensors_kept_elsewhere_and_recomputation():
    from torch.utils.checkpoint import checkpoint

    wide, w, b, dy = make(21, 300, torch.bfloat16)
    x = wide[:, 4:204].detach().requires_grad_()  # strided: what comes back from the host is not
    w, b, dy = w[:200].clone().requires_grad_(), b[:200].clone().requires_grad_(), dy[:, :200]
    want = torch.autograd.grad(F.layer_norm(x, 200, w, b), (x, w, b), dy)
    with torch.autograd.graph.save_on_cpu():
        y = F.layer_norm(x, 200, w, b)
    got = torch.autograd.grad(y, (x, w, b), dy)
    again = torch.autograd.grad(checkpoint(lambda t: F.layer_norm(t, 200, w, b), x, use_reentrant=False), (x, w, b), dy)
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, got, again))


@gpu
def test_no_second_derivative():
    x, w, b, dy = make(4, 32, torch.float32)
    x.requires_grad_()
    g = torch.autograd.grad(F.layer_norm(x, 32, w, b), x, dy, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivative"):
        g.sum().backward()


@gpu
def test_another_stream_and_a_replayed_graph():
    x, w, b, dy = make(300, 512, torch.bfloat16)
    x.requires_grad_()
    want = run_and_check(x, w, b, dy)
    x, w, b = x.detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = F.layer_norm(x, 512, w, b)
        got = torch.autograd.grad(y, (x, w, b), dy)
        y = y.detach()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want[0]) and all(torch.equal(a, c) for a, c in zip(got, want[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        y = F.layer_norm(x, 512, w, b)
        got = torch.autograd.grad(y, (x, w, b), dy)
    for k in range(3):
        with torch.no_grad():
            x.copy_(make(300, 512, torch.bfloat16, seed=k)[0])
        graph.replay()
        torch.cuda.synchronize()
        a = x.detach().clone().requires_grad_()
        ye = F.layer_norm(a, 512, w.detach(), b.detach())
        assert torch.equal(y, ye) and torch.equal(got[0], torch.autograd.grad(ye, a, dy)[0])


@gpu
def test_rows_past_32_bits_of_elements():
    D, rows = 4096, (1 << 31) // 4096 + 3
    x = torch.zeros(rows, D, dtype=torch.bfloat16, device=DEV)
    tail, w, b, dy = make(5, D, torch.bfloat16)
    x[-5:] = tail
    y = F.layer_norm(x, D, w, b)
    assert torch.equal(y[-5:], F.layer_norm(tail, D, w, b))
    g = torch.zeros_like(x)
    g[-5:] = dy
    x.requires_grad_()
    t = tail.clone().requires_grad_()
    dx = torch.autograd.grad(F.layer_norm(x, D, w, b), x, g)[0]
    assert torch.equal(dx[-5:], torch.autograd.grad(F.layer_norm(t, D, w, b), t, dy)[0])
    assert not dx[:100].any()
