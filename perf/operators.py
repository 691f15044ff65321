"""Layer norm, linear + softmax cross entropy, and AdamW with 32- or 8-bit moments: cases, plain forms, definitions.

The three operators of a classifier's training end: the normalisation of its features, the loss of a
linear classifier over many classes together with its gradient, and the optimizer step. ``run`` takes
one pass through an operator: in elementary torch operations, or (``own``) through this package.
"""
import math
import random

import torch

own = False

DEV = "cuda"
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256  # values that share a scale of the 8-bit moments; a block holds values of one tensor only


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one pooled feature vector of a served image, forward only: launch latency counts
        dict(name="layer norm, 1 row of 2048", op="layer_norm", rows=1, width=2048, pad=0, dtype="bf16", train=False),
        # odd sizes: rows that are a slice of a wider fp32 buffer
        dict(name="layer norm, 777 x 1001 fp32", op="layer_norm", rows=777, width=1001, pad=7, dtype="fp32", train=True),
        # the last feature map of a batch of 256 images, channels last: 256 x 7 x 7 positions
        dict(name="layer norm, 12544 x 2048", op="layer_norm", rows=12544, width=2048, pad=0, dtype="bf16", train=True),
        # a first-stage feature map of a batch of 128 images: 128 x 56 x 56 positions, narrow rows
        dict(name="layer norm, 401408 x 256", op="layer_norm", rows=401408, width=256, pad=0, dtype="bf16", train=True),
        # validation of a few images against 1000 classes: a loss for each image, no gradient
        dict(name="cross entropy, 8 x 1000 eval", op="xent", rows=8, width=2048, classes=1000, smoothing=0.0,
             ignored=0.0, bias=True, reduction="none", train=False),
        # the usual training step of a 1000-class classifier
        dict(name="cross entropy, 256 x 1000", op="xent", rows=256, width=2048, classes=1000, smoothing=0.0,
             ignored=0.0, bias=True, reduction="mean", train=True),
        # odd sizes, smoothed labels, a padded batch whose last rows carry no label
        dict(name="cross entropy, 771 x 20011", op="xent", rows=771, width=1021, classes=20011, smoothing=0.1,
             ignored=0.2, bias=True, reduction="mean", train=True),
        # many positions against a large label set: the logits would take 2 GiB in 32 bits
        dict(name="cross entropy, 8192 x 65536", op="xent", rows=8192, width=2048, classes=65536, smoothing=0.0,
             ignored=0.1, bias=False, reduction="mean", train=True),
        # LeNet-5: a step that is all latency
        dict(name="adamw 32, 61706 values", op="adamw", tensors=10, values=61706, bits=32),
        # ResNet-50: 161 tensors
        dict(name="adamw 32, 25557032 values", op="adamw", tensors=161, values=25557032, bits=32),
        dict(name="adamw 8, 25557032 values", op="adamw", tensors=161, values=25557032, bits=8),
        # VGG-16
        dict(name="adamw 8, 138357544 values", op="adamw", tensors=32, values=138357544, bits=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "xent", "adamw"])
    if op == "layer_norm":
        width = _log(rng, 16, 8192)
        rows = _log(rng, 1, min(401408, 100_000_000 // width))
        return dict(op=op, rows=rows, width=width, pad=rng.choice([0, 0, 8, 5]), dtype=rng.choice(["bf16", "fp32"]),
                    train=rng.random() < 0.75)
    if op == "xent":
        width, classes = _log(rng, 32, 4096), _log(rng, 10, 131072)
        rows = _log(rng, 1, min(16384, max(1, 1_000_000_000_000 // (width * classes)), 600_000_000 // classes))
        return dict(op=op, rows=rows, width=width, classes=classes, smoothing=rng.choice([0.0, 0.0, 0.1]),
                    ignored=rng.choice([0.0, 0.15]), bias=rng.random() < 0.5,
                    reduction=rng.choice(["mean", "mean", "sum", "none"]), train=rng.random() < 0.75)
    tensors = _log(rng, 1, 300)
    return dict(op=op, tensors=tensors, values=_log(rng, max(1000, 4 * tensors), 138_000_000), bits=rng.choice([32, 8]))


def _sizes(tensors, values):
    """Tensor sizes as a network has them: each matrix is followed by two short vectors."""
    rng = random.Random(tensors * 1000003 + values)
    most = max(1, values // (4 * tensors))
    sizes = [min(most, rng.choice([64, 128, 255, 256, 512, 1000, 1024, 2048])) for _ in range(tensors)]
    matrices = list(range(0, tensors, 3))
    weights = [math.exp(rng.uniform(0.0, 4.0)) for _ in matrices]
    left = values - sum(sizes)
    for i, w in zip(matrices, weights):
        sizes[i] += int(left * w / sum(weights))
    sizes[0] += values - sum(sizes)
    return sizes


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"layer_norm": _prepare_norm, "xent": _prepare_xent, "adamw": _prepare_adamw}[case["op"]](case, gen)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _inputs_norm(case, gen):
    rows, width, pad = case["rows"], case["width"], case["pad"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    # features with a mean and spread of their own in each row
    x = _randn(gen, rows, width + pad) * (0.5 + torch.rand(rows, 1, generator=gen, device=DEV)) + _randn(gen, rows, 1)
    return dict(x=x.to(dtype)[:, :width], dy=(_randn(gen, rows, width) * 1e-2).to(dtype),
                weight=1 + 0.2 * _randn(gen, width), bias=0.2 * _randn(gen, width))


def _prepare_norm(case, gen):
    s = dict(case=case, **_inputs_norm(case, gen))
    if case["train"]:
        for name in ("x", "weight", "bias"):
            s[name].requires_grad_()
    return s


def _inputs_xent(case, gen):
    rows, width, classes = case["rows"], case["width"], case["classes"]
    x = _randn(gen, rows, width).abs_().to(torch.bfloat16)  # pooled features behind a ReLU
    weight = (_randn(gen, classes, width) * (1.5 / math.sqrt(width))).to(torch.bfloat16)
    labels = torch.randint(0, classes, (rows,), generator=gen, device=DEV)
    labels[rows - int(rows * case["ignored"]):] = -100
    s = dict(x=x, weight=weight, labels=labels, bias=0.1 * _randn(gen, classes) if case["bias"] else None)
    if case["reduction"] == "none":
        s["upstream"] = torch.rand(rows, generator=gen, device=DEV)  # the caller's own weight of each row
    return s


def _prepare_xent(case, gen):
    s = dict(case=case, **_inputs_xent(case, gen))
    if case["train"]:
        for name in ("x", "weight", "bias"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def _inputs_adamw(case, gen):
    sizes = _sizes(case["tensors"], case["values"])
    n = case["values"]
    s = dict(sizes=sizes, param=_randn(gen, n) * 0.05, grad=_randn(gen, n) * 1e-3)
    # moments as a long run has them: v near the mean square of the gradient, m a fraction of its size
    if case["bits"] == 32:
        s["exp_avg"] = _randn(gen, n) * 3e-4
        s["exp_avg_sq"] = (1e-3 * (0.5 + torch.rand(n, generator=gen, device=DEV))) ** 2
        return s
    blocks = sum(-(-k // BLOCK) for k in sizes)
    m = _randn(gen, blocks, BLOCK)
    r = 0.5 + torch.rand(blocks, BLOCK, generator=gen, device=DEV)
    inside = _inside(sizes).view(blocks, BLOCK)
    for name, t, unit in (("exp_avg", m, 3e-4), ("exp_avg_root", r, 1e-3)):
        t = t * inside
        top = t.abs().amax(1)
        s[name] = (t * (448.0 / top)[:, None]).to(torch.float8_e4m3fn).view(-1)
        s[name + "_scale"] = top * (unit / 448.0)
    return s


def _starts(sizes):
    """(first value, first block) of each tensor."""
    at, block, out = 0, 0, []
    for n in sizes:
        out.append((at, block))
        at, block = at + n, block + -(-n // BLOCK)
    return out


def _inside(sizes):
    """1 where a place of the blocks holds a value, 0 behind a tensor's end."""
    return torch.cat([(torch.arange(-(-n // BLOCK) * BLOCK, device=DEV) < n).float() for n in sizes])


def _places(sizes):
    """The place in the blocks of each value of the flat buffers."""
    return torch.cat([torch.arange(n, device=DEV) + block * BLOCK for n, (_, block) in zip(sizes, _starts(sizes))])


STEP, SEED = 1000, 12345


def _prepare_adamw(case, gen):
    s = _inputs_adamw(case, gen)
    s["case"], s["step"] = case, STEP
    if not own:
        if case["bits"] == 8:
            s["places"] = _places(s["sizes"])
        return s
    from deep_vision_amd.train.optim import FusedAdamW

    params = [torch.nn.Parameter(p) for p in s["param"].split(s["sizes"])]
    opt = FusedAdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case["bits"], seed=SEED)
    for p, g in zip(params, s["grad"].split(s["sizes"])):
        p.grad.copy_(g)
    state = {}
    for i, (n, (at, block)) in enumerate(zip(s["sizes"], _starts(s["sizes"]))):
        e = -(-n // BLOCK)
        if case["bits"] == 32:
            state[i] = {k: s[k][at:at + n] for k in ("exp_avg", "exp_avg_sq")}
        else:
            state[i] = {k: s[k][block * BLOCK:(block + e) * BLOCK] for k in ("exp_avg", "exp_avg_root")}
            state[i].update({k + "_scale": s[k + "_scale"][block:block + e] for k in ("exp_avg", "exp_avg_root")})
        state[i]["step"] = torch.tensor(float(STEP))
    opt.load_state_dict({"state": state, "param_groups": opt.state_dict()["param_groups"]})
    return dict(case=case, opt=opt, params=params)


# --------------------------------------------------------------------------------------------- run
def run(s):
    op = s["case"]["op"]
    if own:
        return {"layer_norm": _own_norm, "xent": _own_xent, "adamw": _own_adamw}[op](s)
    with torch.no_grad():
        return {"layer_norm": _plain_norm, "xent": _plain_xent, "adamw": _plain_adamw}[op](s)


def _own_norm(s):
    from deep_vision_amd import ops as F

    y = F.layer_norm(s["x"], (s["case"]["width"],), s["weight"], s["bias"])
    if not s["case"]["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def _own_xent(s):
    from deep_vision_amd import ops as F

    c = s["case"]
    loss = F.linear_cross_entropy(s["x"], s["weight"], s["labels"], s["bias"], label_smoothing=c["smoothing"],
                                  reduction=c["reduction"])
    out = {"loss": loss.detach()}
    if c["train"]:
        names = [k for k in ("x", "weight", "bias") if s[k] is not None]
        grads = torch.autograd.grad(loss, [s[k] for k in names], s.get("upstream"))
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out


def _own_adamw(s):
    s["opt"].step()
    return {"param": s["opt"].flat_params()[0], **s["opt"].flat_states()[0]}


def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"], s["bias"]
    n = x.shape[1]
    d = x - x.sum(1, keepdim=True) / n
    rstd = 1.0 / torch.sqrt((d * d).sum(1, keepdim=True) / n + 1e-5)
    xhat = d * rstd
    y = (xhat * w + b).to(s["x"].dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    h = dy * w
    dx = (h - h.sum(1, keepdim=True) / n - xhat * ((h * xhat).sum(1, keepdim=True) / n)) * rstd
    return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}


def _plain_xent(s):
    c, labels = s["case"], s["labels"]
    x, w = s["x"].float(), s["weight"].float()
    logits = x @ w.t()
    if s["bias"] is not None:
        logits += s["bias"]
    counted = labels >= 0
    at = labels.clamp(min=0)[:, None]
    top = logits.amax(1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(1, keepdim=True)
    lse = (top + torch.log(total))[:, 0]
    eps = c["smoothing"]
    loss = lse - (1 - eps) * logits.gather(1, at)[:, 0] - eps * (logits.sum(1) / c["classes"])
    loss = loss * counted
    if c["reduction"] == "mean":
        scale = counted / counted.sum().clamp(min=1)
        out = {"loss": (loss * scale).sum()}
    else:
        scale = counted.float()
        out = {"loss": loss.sum() if c["reduction"] == "sum" else loss}
        if c["reduction"] == "none":
            scale = scale * s["upstream"]
    if c["train"]:
        p /= total
        p -= eps / c["classes"]
        p.scatter_add_(1, at, torch.full_like(p[:, :1], eps - 1))
        p *= scale[:, None]
        out["dx"], out["dweight"] = (p @ w).to(torch.bfloat16), (p.t() @ x).to(torch.bfloat16)
        if s["bias"] is not None:
            out["dbias"] = p.sum(0)
    return out


def _mix(h):
    """A 32-bit mixing of whole numbers, held in int64."""
    h = h ^ (h >> 16)
    h = (h * 0x6C8E9CF5) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x5D2A4B35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _noise(n, step):
    """32 bits for each place of the blocks, from its number, the step and the seed."""
    key = _mix(torch.tensor((SEED + step * 0x9E3779B1) & 0xFFFFFFFF, device=DEV))
    i = torch.arange(n, device=DEV)
    return _mix((i * 0x2545F491 + key) & 0xFFFFFFFF)


def _store_8_bits(s, name, t, noise):
    """Blocks of values as e4m3 codes times a scale for each block, rounded up with the probability that 20 bits of noise give."""
    top = t.abs().amax(1, keepdim=True)
    most, unit = torch.tensor(448.0, device=DEV), torch.tensor(1 / 448.0, device=DEV)
    up = torch.where(top >= 2.0 ** -100, most / top, torch.zeros_like(top))
    y = t.abs() * up * 2.0 ** -120  # the exponent field and fraction of the code are now those of the float
    code = ((y.view(torch.int32).long() + noise) >> 20).clamp_(max=126)
    if name == "exp_avg":
        code = code + 128 * (t < 0)
    else:
        code = torch.maximum(code, (t > 0).long())  # a root that is not zero stays so: it is divided by
    s[name].copy_(code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1))
    s[name + "_scale"].copy_((top * unit)[:, 0])


def _plain_adamw(s):
    s["step"] += 1
    step = s["step"]
    g = s["grad"]
    if s["case"]["bits"] == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
        m.copy_(m * BETA1 + g * (1 - BETA1))
        v.copy_(v * BETA2 + (g * g) * (1 - BETA2))
        root = torch.sqrt(v)
        out = {"exp_avg": m, "exp_avg_sq": v}
    else:
        at = s["places"]
        blocks = s["exp_avg_scale"].numel()
        pad = torch.zeros(blocks * BLOCK, device=DEV)
        pad[at] = g
        pad = pad.view(blocks, BLOCK)
        m = s["exp_avg"].float().view(blocks, BLOCK) * s["exp_avg_scale"][:, None]
        r = s["exp_avg_root"].float().view(blocks, BLOCK) * s["exp_avg_root_scale"][:, None]
        m = m * BETA1 + pad * (1 - BETA1)
        root = torch.sqrt((r * r) * BETA2 + (pad * pad) * (1 - BETA2))
        noise = _noise(blocks * BLOCK, step).view(blocks, BLOCK)
        _store_8_bits(s, "exp_avg", m, noise & 0xFFFFF)
        _store_8_bits(s, "exp_avg_root", root, noise >> 12)
        m, root = m.view(-1)[at], root.view(-1)[at]
        out = {k: s[k] for k in ("exp_avg", "exp_avg_scale", "exp_avg_root", "exp_avg_root_scale")}
    denom = root * (1 / math.sqrt(1 - BETA2 ** step)) + EPS
    p = s["param"]
    p.copy_(p * (1 - LR * DECAY) - (LR / (1 - BETA1 ** step)) * (m / denom))
    return {"param": p, **out}


# ---------------------------------------------------------------------------------------- the least
def work(case):
    if case["op"] == "layer_norm":
        n, e = case["rows"] * case["width"], 2 if case["dtype"] == "bf16" else 4
        if case["train"]:
            return {"bytes": 4 * n * e + 16 * case["width"], "flops": 18 * n}
        return {"bytes": 2 * n * e + 8 * case["width"], "flops": 7 * n}
    if case["op"] == "xent":
        n, d, v = case["rows"], case["width"], case["classes"]
        one = 2 * d * (n + v) + (4 * v if case["bias"] else 0) + 8 * n
        return {"bytes": one * (2 if case["train"] else 1), "flops": (6 if case["train"] else 2) * n * d * v}
    n = case["values"]
    if case["bits"] == 32:
        return {"bytes": 28 * n, "flops": 14 * n}
    return {"bytes": 16 * n + 16 * (n // BLOCK), "flops": 20 * n}


# ------------------------------------------------------------------------------- the definitions, 64 bits
def exact(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    with torch.no_grad():
        return {"layer_norm": _exact_norm, "xent": _exact_xent, "adamw": _exact_adamw}[case["op"]](case, gen)


def _exact_norm(case, gen):
    s = {k: t.double() for k, t in _inputs_norm(case, gen).items()}
    x, dy = s["x"], s["dy"]
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    std = (var + 1e-5).sqrt()
    out = {"y": s["weight"] * (x - mean) / std + s["bias"]}
    if case["train"]:
        xhat = (x - mean) / std
        part = dy * s["weight"]
        out["dx"] = (part - part.mean(1, keepdim=True) - xhat * (part * xhat).mean(1, keepdim=True)) / std
        out["dweight"], out["dbias"] = torch.einsum("nd,nd->d", dy, xhat), dy.sum(0)
    return out


def _exact_xent(case, gen):
    s = _inputs_xent(case, gen)
    x, w, labels = s["x"].double(), s["weight"].double(), s["labels"]
    rows = torch.nonzero(labels >= 0)[:, 0]
    n, v, eps = len(rows), case["classes"], case["smoothing"]
    logp = x[rows] @ w.t()
    if s["bias"] is not None:
        logp += s["bias"].double()
    logp -= torch.logsumexp(logp, 1, keepdim=True)
    chosen = logp[torch.arange(n, device=DEV), labels[rows]]
    each = torch.zeros(case["rows"], dtype=torch.float64, device=DEV)
    each[rows] = -(1 - eps) * chosen - eps * logp.mean(1)
    up = torch.full((n, 1), 1 / max(n, 1) if case["reduction"] == "mean" else 1.0, dtype=torch.float64, device=DEV)
    out = {"loss": each if case["reduction"] == "none" else each.sum() / (max(n, 1) if case["reduction"] == "mean" else 1)}
    if case["train"]:
        if case["reduction"] == "none":
            up = s["upstream"].double()[rows, None]
        d = logp.exp_().sub_(eps / v)
        d[torch.arange(n, device=DEV), labels[rows]] -= 1 - eps
        d *= up
        dx = torch.zeros_like(x)
        dx[rows] = d @ w
        out.update(dx=dx, dweight=d.t() @ x[rows])
        if s["bias"] is not None:
            out["dbias"] = d.sum(0)
    return out


def _exact_adamw(case, gen):
    s = _inputs_adamw(case, gen)
    step, g, p = STEP + 1, s["grad"].double(), s["param"].double()
    out = {}
    if case["bits"] == 32:
        m = BETA1 * s["exp_avg"].double() + (1 - BETA1) * g
        v = BETA2 * s["exp_avg_sq"].double() + (1 - BETA2) * g ** 2
        out.update(exp_avg=m, exp_avg_sq=v)
    else:
        at = _places(s["sizes"])
        wide = lambda k: s[k].double() * s[k + "_scale"].double().repeat_interleave(BLOCK)  # noqa: E731
        m, r = wide("exp_avg"), wide("exp_avg_root")
        full = torch.zeros_like(m)
        full[at] = g
        m = BETA1 * m + (1 - BETA1) * full
        v = BETA2 * r ** 2 + (1 - BETA2) * full ** 2
        h = _noise(m.numel(), step)
        for name, t, u in (("exp_avg", m, (h % 2 ** 20) / 2.0 ** 20), ("exp_avg_root", v.sqrt(), (h >> 12) / 2.0 ** 20)):
            unit = t.abs().view(-1, BLOCK).amax(1) / 448
            a = t.abs() / unit.repeat_interleave(BLOCK)
            # e4m3: steps of an eighth of the power of two below, of 2^-9 under the least normal value
            grid = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
            q = (torch.floor(a / grid + u) * grid).clamp(max=448)
            q = torch.where((t > 0) & (name == "exp_avg_root"), q.clamp(min=2.0 ** -9), q)
            out[name], out[name + "_scale"] = q * t.sign(), unit
        m, v = m[at], v[at]
    mhat, vhat = m / (1 - BETA1 ** step), v / (1 - BETA2 ** step)
    out["param"] = p - LR * DECAY * p - LR * mhat / (vhat.sqrt() + EPS)
    return out
