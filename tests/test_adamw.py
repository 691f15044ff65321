"""FusedAdamW with 32- and 8-bit moments against the update in 64 bits."""
import math

import pytest
import torch

from deep_vision_amd.train.optim import OPTIMIZERS, FusedAdamW

DEV = "cuda"
gpu = pytest.mark.gpu
SIZES = [1, 3, 255, 256, 257, 64, 4095, 4096, 4097, 10000, 2]
KW = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)
U = 2.0 ** -24


def tensors(sizes=SIZES, dev="cpu", seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale * 10 ** torch.empty(1).uniform_(-2, 1, generator=g)).to(dev) for n in sizes]


def make(dev, bits, sizes=SIZES, seed=7, **kw):
    params = [torch.nn.Parameter(t) for t in tensors(sizes, dev)]
    return params, FusedAdamW(params, **{**KW, **kw}, state_bits=bits, seed=seed)


def feed(params, step, skip=()):
    for i, (p, g) in enumerate(zip(params, tensors([p.numel() for p in params], params[0].device, 100 + step))):
        if i in skip:
            p.grad = None
        elif p.grad is None:
            p.grad = g.view(p.shape).clone()
        else:
            p.grad.copy_(g.view(p.shape))


def states(opt):
    return {k: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for k, t in opt.flat_states()[0].items()}


# ---------------------------------------------------------------- refusals, CPU
def test_refusals():
    p = [torch.nn.Parameter(torch.zeros(3))]
    for kw, text in ((dict(state_bits=16), "state_bits"), (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"),
                     (dict(lr=-1.0), "negative"), (dict(eps=-1.0), "negative"), (dict(weight_decay=-1.0), "negative")):
        with pytest.raises(ValueError, match=text):
            FusedAdamW(p, **kw)
    with pytest.raises(TypeError, match="fp32"):
        FusedAdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.bfloat16))])
    params, opt = make("cpu", 8)
    other, small = make("cpu", 8, sizes=[1, 3, 255, 256, 257, 64, 4095, 4096, 4097, 100, 2])
    feed(params, 0)
    opt.step()
    with pytest.raises(ValueError, match="saved 8-bit state"):
        small.load_state_dict(opt.state_dict())
    assert OPTIMIZERS["AdamW"] is FusedAdamW


def test_config_name_reaches_the_optimizer():
    from deep_vision_amd.train.engine import make_optimizer

    opt = make_optimizer("adamw", [torch.nn.Parameter(torch.zeros(5))], {"lr": 1e-3, "betas": [0.9, 0.95], "state_bits": 8})
    assert isinstance(opt, FusedAdamW) and opt.state_bits == 8


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
def test_32_bits_against_torch_in_64(dev):
    """Ten steps. A step moves p by at most lr (1 + wd |p|) (the moments' ratio stays under
    (1 - b1) / sqrt(1 - b2) in general, near 1 here) and rounds it once: ten times half a step of p,
    and of the update, whose own few roundings are 16 of 2^-24 of it at most; m and v as sums of ten
    rounded terms."""
    params, opt = make(dev, 32)
    ref = [torch.nn.Parameter(t.double()) for t in tensors(dev=dev)]
    topt = torch.optim.AdamW(ref, **KW)
    for step in range(10):
        feed(params, step)
        for p, r in zip(params, ref):
            r.grad = p.grad.double()
        opt.step()
        topt.step()
    for i, (p, r) in enumerate(zip(params, ref)):
        bound = 10 * (2 * U * r.abs().amax() + 32 * U * KW["lr"] * 4)
        assert ((p.double() - r).abs() <= bound).all(), i
        st = topt.state[r]
        sd = opt.state_dict()["state"][i]
        m_size, v_size = 10 * 8 * U * tensors_max(params[i].grad), 10 * 8 * U * tensors_max(params[i].grad) ** 2
        assert ((sd["exp_avg"].double() - st["exp_avg"]).abs() <= 4 * U * st["exp_avg"].abs() + m_size).all()
        assert ((sd["exp_avg_sq"].double() - st["exp_avg_sq"]).abs() <= 24 * U * st["exp_avg_sq"] + v_size * 1e-2).all()


def tensors_max(t):
    return 10 * t.abs().max().item()  # the scale of a tensor's gradients differs by up to 1000 between steps


def test_8_bit_codes_keep_the_moments_on_average():
    """One block, many seeds: each stored value lies on one of the two codes around the moment, and
    their mean is the moment: over 400 seeds within 5 standard deviations of at most half a step."""
    n, runs = 256, 400
    g = torch.randn(n, generator=torch.Generator().manual_seed(3))
    total_m, total_r = torch.zeros(n), torch.zeros(n)
    for seed in range(runs):
        p = torch.nn.Parameter(torch.zeros(n))
        opt = FusedAdamW([p], state_bits=8, seed=seed)
        p.grad.copy_(g)
        opt.step()
        s = opt.flat_states()[0]
        total_m += s["exp_avg"].float() * s["exp_avg_scale"]
        total_r += s["exp_avg_root"].float() * s["exp_avg_root_scale"]
    m, r = 0.1 * g, (0.001 ** 0.5) * g.abs()
    for mean, want in ((total_m / runs, m), (total_r / runs, r)):
        step = torch.maximum(want.abs() / 8, want.abs().max() / 448 * 2.0 ** -9)
        assert ((mean - want).abs() <= 5 * step / 2 / runs ** 0.5 + 1e-6 * want.abs().max()).all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
def test_8_bit_step_and_rounding(dev):
    """From known codes: p as the 64-bit update of the decoded moments gives it, and each new code one
    of the two around the new moment."""
    params, opt = make(dev, 8)
    for step in range(3):
        feed(params, step)
        opt.step()
    old = {k: v.clone() for k, v in opt.flat_states()[0].items()}
    before = [p.detach().double().clone() for p in params]
    feed(params, 3)
    opt.step()
    new, at = opt.flat_states()[0], 0

    def wide(s, name, i0, n):
        b = i0 // 256
        e = -(-n // 256)
        return (s[name][i0:i0 + e * 256].double().view(e, 256) * s[name + "_scale"][b:b + e].double()[:, None]).view(-1), e

    for p, q in zip(params, before):
        n = p.numel()
        m0, e = wide(old, "exp_avg", at, n)
        r0, _ = wide(old, "exp_avg_root", at, n)
        g = torch.zeros_like(m0)
        g[:n] = p.grad.double()
        m, v = 0.9 * m0 + 0.1 * g, 0.999 * r0 * r0 + 0.001 * g * g
        per = KW["lr"] / (1 - 0.9 ** 4) / (v.sqrt() / math.sqrt(1 - 0.999 ** 4) + KW["eps"])
        move, terms = per * m, per * (0.9 * m0.abs() + 0.1 * g.abs())  # m's products round whatever cancels
        want = q * (1 - KW["lr"] * KW["weight_decay"]) - move[:n]
        assert ((p.detach().double() - want).abs() <= 3 * U * want.abs() + 24 * U * terms[:n]).all()
        for name, t in (("exp_avg", m), ("exp_avg_root", v.sqrt())):
            got, _ = wide(new, name, at, n)
            top = t.abs().view(e, 256).amax(1, keepdim=True).expand(e, 256).reshape(-1)
            step = torch.maximum(torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=1e-30)))) / 8 / 1.0, top / 448 * 2.0 ** -9)
            # a code's exponent counts in units of the scale: the step is at most twice the value's own
            assert ((got - t).abs() <= 2 * step * (1 + 1e-5)).all()
            assert not got[n:].any()
        assert (wide(new, "exp_avg_root", at, n)[0][:n][v[:n] > 0] > 0).all()
        at += e * 256


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_without_a_gradient_stays(bits):
    params, opt = make("cpu", bits)
    feed(params, 0)
    opt.step()
    snap = [p.detach().clone() for p in params]
    kept = opt.state_dict()["state"]
    feed(params, 1, skip=(1, 4, 10))
    opt.step()
    now = opt.state_dict()["state"]
    for i, (p, q) in enumerate(zip(params, snap)):
        assert torch.equal(p, q) == (i in (1, 4, 10))
        if i in (1, 4, 10):
            assert all(torch.equal(now[i][k].float(), kept[i][k].float()) for k in kept[i] if k != "step")


@pytest.mark.parametrize("bits", [32, 8])
def test_resume_and_the_flat_order_do_not_change_a_run(bits, tmp_path):
    from deep_vision_amd.parallel.flat import flatten_parameters

    params, opt = make("cpu", bits)
    for step in range(4):
        feed(params, step)
        opt.step()
        if step == 1:
            torch.save(opt.state_dict(), tmp_path / "o.pt")
            saved = [p.detach().clone() for p in params]
    other = torch.nn.ParameterList([torch.nn.Parameter(t) for t in saved])
    flatten_parameters(other)  # the data-parallel layer's order: last parameter first
    again = FusedAdamW(list(other), **KW, state_bits=bits, seed=7)
    again.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
    for step in (2, 3):
        feed(list(other), step)
        again.step()
    assert all(torch.equal(a, b) for a, b in zip(params, other))


def test_rebinding_carries_the_8_bit_state():
    from deep_vision_amd.parallel.flat import flatten_parameters

    params, opt = make("cpu", 8)
    plist, ropt = make("cpu", 8)
    for step in range(3):
        if step == 1:
            flatten_parameters(torch.nn.ParameterList(plist))
        for ps, o in ((params, opt), (plist, ropt)):
            feed(ps, step)
            o.step()
    assert all(torch.equal(a, b) for a, b in zip(params, plist))


def test_checkpoints_of_either_width_load():
    """8 from 32 bits: rounded to nearest, off by half a step (a sixteenth, or half the least code);
    32 from 8: the values the codes stand for."""
    params, wide = make("cpu", 32)
    feed(params, 0)
    wide.step()
    _, narrow = make("cpu", 8)
    narrow.load_state_dict(wide.state_dict())
    _, back = make("cpu", 32)
    back.load_state_dict(narrow.state_dict())
    a, b = wide.state_dict()["state"], back.state_dict()["state"]
    for i in a:
        for k, root in (("exp_avg", False), ("exp_avg_sq", True)):
            x, y = (t[i][k].sqrt() if root else t[i][k] for t in (a, b))
            blocks = torch.zeros(-(-x.numel() // 256) * 256)
            blocks[:x.numel()] = x.abs()
            top = blocks.view(-1, 256).amax(1, keepdim=True).expand(-1, 256).reshape(-1)[:x.numel()]
            assert ((x - y).abs() <= x.abs() / 16 * (1 + 1e-5) + top / 448 * 2.0 ** -9).all()
    assert wide._flat[0]["step"] == back._flat[0]["step"] == 1


# ---------------------------------------------------------------- the kernels
@gpu
def test_8_bit_kernel_gives_the_hosts_codes():
    """The moments of both forms are rounded operation by operation: equal bits over several steps."""
    gp, gopt = make(DEV, 8)
    cp, copt = make("cpu", 8)
    for step in range(6):
        feed(cp, step)
        for a, b in zip(gp, cp):
            a.grad.copy_(b.grad)
        gopt.step()
        copt.step()
        for k, t in states(copt).items():
            assert torch.equal(states(gopt)[k].cpu(), t), (step, k)
        for a, b in zip(gp, cp):
            size = b.detach().abs() + KW["lr"] * 4
            assert ((a.detach().cpu() - b.detach()).abs() <= (step + 1) * 16 * U * size).all()


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_kernel_skips_what_has_no_gradient(bits):
    params, opt = make(DEV, bits)
    host, hopt = make("cpu", bits)
    for step, skip in ((0, ()), (1, (0, 3, 10)), (2, (9,))):
        feed(params, step, skip)
        feed(host, step, skip)
        for a, b in zip(params, host):
            if b.grad is not None:
                a.grad.copy_(b.grad)
        snap = [p.detach().clone() for p in params]
        opt.step()
        hopt.step()
        for i, (p, q) in enumerate(zip(params, snap)):
            assert torch.equal(p, q) == (i in skip)
    for a, b in zip(params, host):
        assert ((a.detach().cpu() - b.detach()).abs() <= 64 * U * (b.detach().abs() + KW["lr"] * 4)).all()


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_follow_eager_ones(bits):
    from deep_vision_amd.train.graph import CapturedStep

    a, oa = make(DEV, bits)
    b, ob = make(DEV, bits)
    src = [t.to(DEV) for t in tensors(seed=55)]

    def step_of(params, opt):
        def step():
            for p, t in zip(params, src):
                p.grad.copy_(t)
            opt.step()
            return params[0].detach()
        return step

    cap = CapturedStep(step_of(a, oa), oa, ())
    eager = step_of(b, ob)
    for _ in range(2):  # the capture's two warm-up steps
        eager()
    for k in range(4):
        for o in (oa, ob):
            o.param_groups[0]["lr"] = 1e-2 / (k + 1)
        for i, t in enumerate(src):
            t.copy_(tensors(seed=60 + k)[i])
        cap()
        eager()
        torch.cuda.synchronize()
        for x, y in zip(a, b):
            torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-7)
        if bits == 8:
            sa, sb = states(oa), states(ob)
            assert all(torch.equal(sa[n], sb[n]) for n in sa)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_device_guard_leaves_everything_as_it_was(bits):
    params, opt = make(DEV, bits)
    opt.use_device_guard(True)
    feed(params, 0)
    opt.step()
    snap, st = [p.detach().clone() for p in params], {k: v.clone() for k, v in states(opt).items()}
    feed(params, 1)
    params[3].grad[5] = float("inf")
    opt.step()
    assert opt.device_guard_counts()[0] == 1
    assert all(torch.equal(p, q) for p, q in zip(params, snap)) and all(torch.equal(states(opt)[k], v) for k, v in st.items())
    feed(params, 2)
    opt.step()
    assert not torch.equal(params[3], snap[3])


@gpu
def test_values_that_are_not_finite_show():
    params, opt = make(DEV, 8, sizes=[600])
    feed(params, 0)
    params[0].grad[300] = float("nan")
    opt.step()
    p, s = params[0].detach(), opt.flat_states()[0]
    assert p[300].isnan() and p.isnan().sum() == 1
    assert s["exp_avg"].float()[300].isnan() and s["exp_avg"].float().isnan().sum() == 1


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_two_groups_and_another_stream(bits):
    a = [torch.nn.Parameter(t) for t in tensors(dev=DEV)]
    b = [torch.nn.Parameter(t) for t in tensors(dev=DEV)]
    one = FusedAdamW([{"params": a[:4], "weight_decay": 0.0}, {"params": a[4:]}], **KW, state_bits=bits)
    two = FusedAdamW([{"params": b[:4], "weight_decay": 0.0}, {"params": b[4:]}], **KW, state_bits=bits)
    s = torch.cuda.Stream()
    for step in range(2):
        feed(a, step)
        feed(b, step)
        one.step()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            two.step()
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert len(one.flat_params()) == len(one.flat_states()) == 2


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_past_32_bits_of_values(bits):
    """2^31 zeros before a tensor (which stay: no gradient, no moments, no decay of zero): the tensor
    behind them moves as it does alone, its noise apart (another place)."""
    tail = tensors([5000], DEV)[0]
    big = torch.nn.Parameter(torch.zeros((1 << 31) + 13, device=DEV))
    far, near = torch.nn.Parameter(tail.clone()), torch.nn.Parameter(tail.clone())
    one = FusedAdamW([big, far], **KW, state_bits=bits)
    two = FusedAdamW([near], **KW, state_bits=bits)
    for step in range(2):
        feed([near], step)
        far.grad.copy_(near.grad)
        one.step()
        two.step()
        if bits == 32 or step == 0:
            assert torch.equal(far, near)
    assert not big[:1000].any() and not big[-1000:].any()
    a, b = one.state_dict()["state"][1], two.state_dict()["state"][0]
    for k in a:
        if k.endswith("_scale") or bits == 32:
            torch.testing.assert_close(a[k], b[k], rtol=0.3 if bits == 8 else 0, atol=0)


def poisoned(dev, bad, always=False, steps=3):
    """(parameters, states) of 8-bit runs whose first step's gradient (``always``: every step's) holds
    ``bad`` {(tensor, place): value}, step by step."""
    params, opt = make(dev, 8, sizes=[600, 300, 256])
    out = []
    for step in range(steps):
        grads = tensors([600, 300, 256], "cpu", 100 + step)
        if always or step == 0:
            for (i, at), v in bad.items():
                grads[i][at] = v
        for p, g in zip(params, grads):
            p.grad.copy_(g)
        opt.step()
        out.append(([p.detach().cpu().clone() for p in params], {k: t.cpu().clone() for k, t in states(opt).items()}))
    return out


INF, NAN = float("inf"), float("nan")
BAD = [{(0, 300): NAN}, {(0, 300): INF}, {(0, 5): -INF, (0, 300): 1e25}, {(0, 599): INF, (2, 0): NAN},
       {(1, k): NAN for k in range(300)}, {(1, k): INF for k in range(256)}]


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
def test_a_value_that_is_not_finite_stays_alone(dev, bad):
    """The others of its block go on as beside a zero; itself is NaN from the second step on. (A finite gradient
    whose square overflows leaves the first step's parameter finite, and its first moment sets its block's scale.)"""
    runs = poisoned(dev, bad), poisoned(dev, {k: 0.0 for k in bad}, always=True)
    starts = (0, 768, 1280)
    places = torch.tensor([starts[i] + at for i, at in bad])
    apart = torch.zeros(1536, dtype=torch.bool)  # places that are not those of the clean run
    apart[places] = True
    block = {starts[i] // 256 + at // 256 for (i, at), v in bad.items() if abs(v) < INF}
    for b in block:
        apart[b * 256:b * 256 + 256] = True
    for step, ((p, s), (cp, cs)) in enumerate(zip(*runs)):
        for name in ("exp_avg", "exp_avg_root"):
            scale, clean = s[name + "_scale"], cs[name + "_scale"]
            assert scale.isfinite().all()
            assert all(scale[b] == clean[b] for b in range(6) if b not in block)
            assert torch.equal(s[name][~apart], cs[name][~apart])
            codes = s[name].view(torch.float8_e4m3fn).float()
            assert codes.isfinite().sum() == 1536 - len(bad) + (len(block) if name == "exp_avg" else 0)
        for i, (a, b) in enumerate(zip(p, cp)):
            keep = ~apart[starts[i]:starts[i] + a.numel()]
            assert torch.equal(a[keep], b[keep])
            assert a.isnan().sum() == sum(j == i and (step > 0 or not abs(v) < INF) for (j, _), v in bad.items())


@gpu
@pytest.mark.parametrize("bad", BAD)
def test_host_and_kernel_agree_behind_a_value_that_is_not_finite(bad):
    for (gp, gs), (cp, cs) in zip(poisoned(DEV, bad), poisoned("cpu", bad)):
        assert all(torch.equal(gs[k], cs[k]) for k in cs)
        assert all(torch.equal(a.isnan(), b.isnan()) for a, b in zip(gp, cp))


@pytest.mark.parametrize("b2", [0.99, 0.997])
def test_8_bit_second_moment_settles_above_its_mean(b2):
    """What the documentation says of v. A step moves the root by at most (1 - b2) / 2 E|g^2 / v - 1| r = 0.49
    (1 - b2) r in the mean, and the block's scale by as much: rounding adds at most their product with a code's step,
    r / 8, to the root's square each step, which the decay forgets by 1 - b2: at most 2 * 0.49 / 8 = 12 % in balance."""
    n, steps = 8192, int(6 / (1 - b2))
    g = torch.Generator().manual_seed(0)
    v = torch.zeros(n)
    p = torch.nn.Parameter(torch.zeros(n))
    opt = FusedAdamW([p], lr=0.0, betas=(0.9, b2), state_bits=8)
    for _ in range(steps):
        p.grad.copy_(torch.randn(n, generator=g))
        v = b2 * v + (1 - b2) * p.grad ** 2
        opt.step()
    s = opt.flat_states()[0]
    r = s["exp_avg_root"].float().view(-1, 256) * s["exp_avg_root_scale"][:, None]
    assert 0.01 < (r ** 2).mean() / v.mean() - 1 < 0.13
    assert -0.01 < r.mean() / v.sqrt().mean() - 1 < 0.07  # the mean of roots moves by no more than half of that


@pytest.mark.parametrize("bits", [32, 8])
def test_a_saved_8_bit_state_of_another_size_is_refused(bits):
    """More or fewer blocks, and a longer tensor of as many blocks, whose codes go on behind the shorter one's end."""
    _, saved = make("cpu", 8, sizes=[600])
    feed(saved.param_groups[0]["params"], 0)
    saved.step()
    state = saved.state_dict()
    for n, text in ((500, "expected 512"), (800, "expected 1024"), (599, "of a larger one")):
        with pytest.raises(ValueError, match=text):
            make("cpu", bits, sizes=[n])[1].load_state_dict(state)
    opt = make("cpu", bits, sizes=[600])[1]
    state["state"][0]["exp_avg"].view(torch.uint8)[600:] = 0x80  # zeros with a sign
    opt.load_state_dict(state)
    assert opt._flat[0]["step"] == 1


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=gpu)])
@pytest.mark.parametrize("name,kw", [("AdamW", {}), ("AdamW", {"state_bits": 8}), ("Adam", {}), ("SGD", {"momentum": 0.9}),
                                     ("RMSprop", {})])
def test_a_group_added_later_moves_as_from_the_start(dev, name, kw):
    sizes = [300, 7]
    a, b = ([torch.nn.Parameter(t) for t in tensors(sizes, dev)] for _ in range(2))
    whole = OPTIMIZERS[name]([{"params": a[:1]}, {"params": a[1:], "lr": 0.05}], lr=0.01, **kw)
    added = OPTIMIZERS[name](b[:1], lr=0.01, **kw)
    added.add_param_group({"params": b[1:], "lr": 0.05})
    for step in range(3):
        for ps, opt in ((a, whole), (b, added)):
            feed(ps, step)
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and not torch.equal(a[1].cpu(), tensors(sizes)[1])
    again = OPTIMIZERS[name]([{"params": [torch.nn.Parameter(torch.zeros(300))]}, {"params": [torch.nn.Parameter(torch.zeros(7))]}],
                             lr=0.01, **kw)
    again.load_state_dict(added.state_dict())
    assert [f["step"] for f in again._flat] == [3, 3]
