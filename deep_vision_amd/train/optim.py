"""Fused optimizers over one flat fp32 parameter buffer.

All parameters of a group live in a single contiguous fp32 buffer (the ``nn.Parameter``s become
views into it) and their ``.grad``s are views into a matching flat gradient buffer. One kernel
launch (csrc/loss_optim.hip) updates the whole model per step, and the data-parallel layer
all-reduces slices of the same flat gradient buffer in place (no bucket copies).

Update rules match torch.optim.SGD / Adam / AdamW / RMSprop exactly (same state names, same
``state_dict`` format), as used by the reference configs (R/ResNet/pytorch/train.py:26-215:
SGD momentum .9 + wd, RMSprop for MobileNet; Adam for LeNet/YOLO/Hourglass/GANs).
On CPU the same classes run the identical math with torch ops.
"""
from __future__ import annotations

import math
from bisect import bisect_left

import torch

from .._ext import lib, ptr, stream_handle
from ..ops.common import on_device


class _FlatOptimizer(torch.optim.Optimizer):
    STATE_NAMES: tuple = ()

    def __init__(self, params, defaults):
        super().__init__(params, defaults)
        self._flat = []  # per group: dict(param, grad, views, gviews, offsets, states)
        for group in self.param_groups:
            self._flat.append(self._flatten_group(group))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        if hasattr(self, "_flat"):  # behind __init__, which flattens its groups itself
            self._flat.append(self._flatten_group(self.param_groups[-1]))

    # ---------------- flat storage ----------------
    @staticmethod
    def _shared_span(ps, sizes):
        """(shared, lo, hi) when every parameter of ``ps`` is a view into ONE existing flat
        buffer pair (parallel.flat.flatten_parameters / another optimizer) and together they tile
        the contiguous range [lo, hi) of it exactly; otherwise None."""
        shared = getattr(ps[0], "_dv_flat", None)
        if shared is None or any(getattr(p, "_dv_flat", None) is not shared for p in ps):
            return None
        spans = sorted((p._dv_off, n) for p, n in zip(ps, sizes))
        lo = spans[0][0]
        end = lo
        for off, n in spans:
            if off != end:
                return None
            end += n
        for p, n in zip(ps, sizes):  # each parameter must still BE its slice of the buffer
            if p.data_ptr() != shared[0][p._dv_off:p._dv_off + n].data_ptr():
                return None
        return shared, lo, end

    def _flatten_group(self, group, old=None):
        ps = group["params"]
        if not ps:
            return None
        dev = ps[0].device
        for p in ps:
            if p.dtype != torch.float32:
                raise TypeError("fused optimizers keep fp32 master parameters")
            if p.device != dev:
                raise ValueError("all parameters of a group must live on one device")
        # reuse an existing flat buffer (parallel.flat.flatten_parameters) when the group's
        # parameters are views that tile a contiguous range of it
        sizes = [p.numel() for p in ps]
        total = sum(sizes)
        span = self._shared_span(ps, sizes)
        views, gviews, offs = [], [], []
        if span is not None:
            shared, lo, hi = span
            pflat, gflat = shared[0][lo:hi], shared[1][lo:hi]
            for p, n in zip(ps, sizes):
                off = p._dv_off - lo
                views.append(pflat[off:off + n].view(p.shape))
                gviews.append(gflat[off:off + n].view(p.shape))
                if p.grad is not None and p.grad.data_ptr() != gviews[-1].data_ptr():
                    gviews[-1].copy_(p.grad)
                p.data = views[-1]
                p.grad = gviews[-1]
                offs.append((off, n))
        else:
            shared = None
            pflat = torch.empty(total, dtype=torch.float32, device=dev)
            gflat = torch.zeros(total, dtype=torch.float32, device=dev)
            off = 0
            for p, n in zip(ps, sizes):
                pv = pflat[off:off + n].view(p.shape)
                gv = gflat[off:off + n].view(p.shape)
                pv.copy_(p.data)
                p.data = pv
                if p.grad is not None:
                    gv.copy_(p.grad)
                p.grad = gv
                views.append(pv)
                gviews.append(gv)
                offs.append((off, n))
                off += n
            shared = (pflat, gflat)
            for p in ps:
                p._dv_flat = shared
            for p, (off, _) in zip(ps, offs):
                p._dv_off = off
        f = dict(param=pflat, grad=gflat, views=views, gviews=gviews, offsets=offs, step=0, first=True, shared=shared)
        f["ptrs"] = [v.data_ptr() for v in views]
        self._share_count(f, ps)
        f["states"] = self._new_states(f)
        if old is not None:  # re-bound after the parameters moved: carry the optimizer state over
            f["step"], f["first"] = old["step"], old["first"]
            if old.get("hp") is not None:
                f["hp"] = old["hp"]
            self._carry_states(old, f)
        return f

    # ---------------- the optimizer's state: fp32 buffers laid out as the flat parameters ----------------
    def _new_states(self, f):
        return {name: torch.zeros_like(f["param"]) for name in self.STATE_NAMES}

    def _carry_states(self, old, f):
        for (o_off, n), (n_off, _) in zip(old["offsets"], f["offsets"]):
            for name in self.STATE_NAMES:
                f["states"][name][n_off:n_off + n].copy_(old["states"][name][o_off:o_off + n])

    def _save_state(self, f, i, shape):
        """State-dict entries of the group's ``i``-th parameter."""
        off, n = f["offsets"][i]
        return {name: buf[off:off + n].view(shape).clone() for name, buf in f["states"].items()}

    def _load_state(self, f, i, st):
        off, n = f["offsets"][i]
        for name in self.STATE_NAMES:
            if name in st:
                f["states"][name][off:off + n].copy_(st[name].reshape(-1).to(f["param"].device))

    def _check_binding(self):
        """Each parameter must still be a view of THIS optimizer's flat buffer. When a later
        ``parallel.DataParallel`` (or anything calling flatten_parameters) moved the parameters
        into a new flat buffer, re-bind transparently -- updating the orphaned old buffer would
        leave the model untrained -- and carry the state over."""
        for gi, (group, f) in enumerate(zip(self.param_groups, self._flat)):
            if f is None:
                continue
            # (the buffer this optimizer holds stays allocated: a parameter moved elsewhere has another address)
            if [p.data_ptr() for p in group["params"]] == f["ptrs"]:
                continue
            if f["param"].is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("parameters were re-flattened under a graph capture")
            self._flat[gi] = self._flatten_group(group, old=f)
            self._rebinds = getattr(self, "_rebinds", 0) + 1

    # ---------------- device-side hyperparameters (HIP-graph replay) ----------------
    def use_device_hparams(self, on: bool = True):
        """Kernels read (lr, bias corrections) from a per-group device tensor ``hp`` instead of
        launch arguments, so a step captured in a HIP graph (train.graph.CapturedStep) follows LR
        schedules and Adam's step count: ``graph_tick()`` writes the next step's values before
        each replay.

        The tensor is allocated ONCE per group and never replaced: every captured graph bakes its
        device pointer in, so a second capture (another input signature) must share it -- a
        fresh tensor would leave the first graph reading freed memory."""
        for f in self._flat:
            if f is None:
                continue
            if on:
                if f.get("hp") is None:
                    f["hp"] = f.get("_hp_keep")
                if f["hp"] is None:
                    f["hp"] = torch.zeros(4, dtype=torch.float32, device=f["param"].device)
                f["_hp_keep"] = f["hp"]
            else:
                f["hp"] = None  # eager launches take host arguments; the buffer stays alive in _hp_keep

    def _hparams(self, group, step):
        """(lr, bias-correction-1, bias-correction-2) of step number ``step`` (1-based)."""
        return float(group["lr"]), 1.0, 1.0

    def _write_hp(self, group, f):
        lr, bc1, bc2 = self._hparams(group, f["step"])
        f["hp"].copy_(torch.tensor([lr, bc1, bc2, float(f["step"])], dtype=torch.float32))

    @torch.no_grad()
    def graph_tick(self):
        """Advance the host step counters as one eager step() would, and write the device
        hyperparameters of that step (ordered on the current stream before the replay)."""
        for group, f in zip(self.param_groups, self._flat):
            if f is None:
                continue
            f["step"] += 1
            f["first"] = False
            self._count_updates(f, [(0, f["param"].numel())])
            self._write_hp(group, f)

    @staticmethod
    def _share_count(f, ps):
        """Give each parameter its update counts, (of its own, of the group's whole steps): the kernels write through raw
        pointers, so a backward pass that reads a parameter again cannot tell from its version
        (ops.common.refuse_updated). A parameter that comes from another group (the third entry: their own
        counts) counts whole steps on its own too, for the passes that remember the other group's."""
        old = [getattr(p, "_dv_updates", None) for p in ps]
        group = old[0][1] if old[0] is not None else None
        if group is None or group[1] != len(ps) or any(c is None or c[1] is not group for c in old):
            group = [0, len(ps), [c[0] for c in old if c is not None]]
            for p, c in zip(ps, old):
                p._dv_updates = ([0] if c is None else c[0], group)
        f["count"], f["counts"] = group, [p._dv_updates[0] for p in ps]

    @staticmethod
    def _count_updates(f, segs):
        if len(segs) == 1 and segs[0][1] == f["param"].numel():
            f["count"][0] += 1
            for count in f["count"][2]:
                count[0] += 1
            return
        for count, (at, n) in zip(f["counts"], f["offsets"]):
            if any(off <= at and at + n <= off + k for off, k in segs):
                count[0] += 1

    def _hp_ptr(self, f):
        hp = f.get("hp")
        return 0 if hp is None else ptr(hp)

    # ---------------- device-side non-finite guard (HIP-graph replay) ----------------
    def use_device_guard(self, on: bool = True):
        """Skip-step on non-finite gradients decided ON THE DEVICE (csrc/loss_optim.hip
        nonfinite_check / nonfinite_tally): every step checks the flat gradients, the update
        kernels become no-ops when any is Inf/NaN, and device counters record the skips -- no host
        synchronisation, so it works inside a captured step. The guard
        tensor [flag, skipped, consecutive, last, applied] is allocated once and never replaced
        (graphs bake its pointer in). In a data-parallel step the checked gradients are the
        all-reduced ones, identical on every rank: the ranks skip together without an extra
        collective.

        ``applied`` counts the steps actually taken (it starts at the host step count): Adam's
        bias corrections read it under the guard, so a skipped replay does not advance them -- as
        an eager skipped step, which never calls step(), does not. The host step count
        (graph_tick, state_dict) and LR schedules still count every replay; the applied count is
        ``step - skipped``."""
        self._dguard_on = bool(on)
        if on and getattr(self, "_dguard", None) is None:
            dev = next((f["param"].device for f in self._flat if f is not None), None)
            if dev is not None and dev.type == "cuda":
                done = getattr(self, "_loaded_applied", None)
                if done is None:
                    done = max((f["step"] for f in self._flat if f is not None), default=0)
                self._dguard = torch.tensor([0.0, 0.0, 0.0, 0.0, float(done)], dtype=torch.float32, device=dev)

    def _guard_active(self):
        return getattr(self, "_dguard_on", False) and getattr(self, "_dguard", None) is not None

    def _skip_ptr(self):
        return ptr(self._dguard) if self._guard_active() else 0

    def device_guard_counts(self):
        """(steps skipped so far, current run of consecutive skips, last step skipped) -- one
        device->host read; call at the logging cadence."""
        if getattr(self, "_dguard", None) is None:
            return 0, 0, False
        v = self._dguard.tolist()
        return int(v[1]), int(v[2]), bool(v[3])

    def param_views(self):
        return [v for f in self._flat if f for v in f["views"]]

    def flat_grads(self):
        return [f["grad"] for f in self._flat if f]

    def flat_params(self):
        """Each group's parameters as the one flat fp32 buffer the update runs over, to be read: what is written to it
        passes by autograd's versions and the cached operands (ops/wcache.py)."""
        return [f["param"] for f in self._flat if f]

    def flat_states(self):
        """Each group's live state buffers by name (``FusedAdamW`` documents its 8-bit ones)."""
        return [dict(f["states"]) for f in self._flat if f]

    @torch.no_grad()
    def zero_grad(self, set_to_none: bool = False):
        self._check_binding()
        for group, f in zip(self.param_groups, self._flat):
            if f is None:
                continue
            f["grad"].zero_()
            for p, gv in zip(group["params"], f["gviews"]):
                if p.grad is not gv:
                    p.grad = gv

    def _sync_grads(self, group, f):
        """Ensure every .grad is the flat view; returns active (offset, n) segments."""
        if all([p.grad is gv for p, gv in zip(group["params"], f["gviews"])]):
            return [(0, f["param"].numel())]
        segs = []
        all_active = True
        for p, gv, (off, n) in zip(group["params"], f["gviews"], f["offsets"]):
            g = p.grad
            if g is None:
                all_active = False
                p.grad = gv
                gv.zero_()
                continue
            if g is not gv:
                gv.copy_(g)
                p.grad = gv
            segs.append((off, n))
        if all_active:
            return [(0, f["param"].numel())]
        # merge adjacent segments
        merged = []
        for off, n in sorted(segs):
            if merged and merged[-1][0] + merged[-1][1] == off:
                merged[-1] = (merged[-1][0], merged[-1][1] + n)
            else:
                merged.append((off, n))
        return merged

    @torch.no_grad()
    def step(self, closure=None, grad_scale: float = 1.0):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._check_binding()
        guard = self._guard_active()
        # the active segments of every group, taken once: _sync_grads binds a None .grad to its
        # (zeroed) flat view, so a second call would report every parameter active and the update
        # would apply weight decay / momentum to parameters that got no gradient this step
        segs_all = [self._sync_grads(group, f) if f is not None else None
                    for group, f in zip(self.param_groups, self._flat)]
        if guard:  # flag any non-finite gradient of any group before the first update launch
            for f in self._flat:
                if f is not None:
                    lib().nonfinite_check(ptr(f["grad"]), f["grad"].numel(), ptr(self._dguard), stream_handle())
        for group, f, segs in zip(self.param_groups, self._flat, segs_all):
            if f is None:
                continue
            f["step"] += 1
            # device hyperparameters: an eager step writes its own; inside a graph capture the
            # values come from graph_tick() before each replay (a captured copy would replay stale)
            if f.get("hp") is not None and not torch.cuda.is_current_stream_capturing():
                self._write_hp(group, f)
            for off, n in segs:
                self._update(group, f, off, n, grad_scale)
            self._count_updates(f, segs)
            f["first"] = False
        if guard:
            lib().nonfinite_tally(ptr(self._dguard), stream_handle())  # counters; re-arms the flag
        if any(f is not None and f["param"].is_cuda for f in self._flat):
            from ..ops import wcache

            wcache.after_step(owner=self)  # one batched re-layout of every cached bf16 weight operand
        return loss

    def _update(self, group, f, off, n, gs):  # pragma: no cover - abstract
        raise NotImplementedError

    @staticmethod
    def _slice(t, off, n):
        return t[off:off + n]

    # ---------------- torch-compatible state_dict ----------------
    def state_dict(self):
        sd = super().state_dict()
        state = {}
        idx = 0
        for group, f in zip(self.param_groups, self._flat):
            if f is None:
                continue
            for i, p in enumerate(group["params"]):
                st = self._save_state(f, i, p.shape)
                if self.STATE_NAMES and not f["first"]:
                    st["step"] = torch.tensor(float(f["step"]))
                    state[idx] = st
                idx += 1
        sd["state"] = state
        # the device guard's applied-step count (steps whose update ran; Adam's bias corrections
        # follow it) and skips: a captured run's "step" also counts skipped replays, an eager run's
        # does not, so the applied count is saved explicitly
        applied = skipped = None
        if getattr(self, "_dguard", None) is not None:
            v = self._dguard.tolist()
            skipped, applied = int(v[1]), int(v[4])
        for g, f in zip(sd["param_groups"], self._flat):
            g["_dv_step"] = f["step"] if f else 0
            if applied is not None:
                g["_dv_applied"], g["_dv_skipped"] = applied, skipped
        return sd

    def load_state_dict(self, state_dict):
        groups = state_dict["param_groups"]
        for g, sg in zip(self.param_groups, groups):
            for k, v in sg.items():
                if k not in ("params", "_dv_step", "_dv_applied", "_dv_skipped"):
                    g[k] = v
        idx = 0
        for sg, group, f in zip(groups, self.param_groups, self._flat):
            if f is None:
                continue
            f["step"] = int(sg.get("_dv_step", 0))
            any_state = False
            for i in range(len(group["params"])):
                st = state_dict["state"].get(idx, state_dict["state"].get(str(idx)))
                if st:
                    any_state = True
                    self._load_state(f, i, st)
                    if "step" in st and f["step"] == 0:
                        f["step"] = int(float(st["step"]))
                idx += 1
            f["first"] = not any_state
        # the device guard's applied-step count: saved by a guarded run, else every saved step applied
        saved = [sg["_dv_applied"] for sg in groups if "_dv_applied" in sg]
        self._loaded_applied = (int(saved[0]) if saved else
                                max((f["step"] for f in self._flat if f is not None), default=0))
        if getattr(self, "_dguard", None) is not None:
            self._dguard[4] = float(self._loaded_applied)


class FusedSGD(_FlatOptimizer):
    STATE_NAMES = ("momentum_buffer",)

    def __init__(self, params, lr=0.1, momentum=0.0, dampening=0.0, weight_decay=0.0, nesterov=False):
        super().__init__(params, dict(lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay,
                                      nesterov=nesterov))

    def _update(self, g, f, off, n, gs):
        p = f["param"][off:off + n]
        gr = f["grad"][off:off + n]
        buf = f["states"]["momentum_buffer"][off:off + n]
        if p.is_cuda:
            lib().sgd(ptr(p), ptr(gr), ptr(buf), n, float(g["lr"]), float(g["momentum"]), float(g["dampening"]),
                      float(g["weight_decay"]), int(g["nesterov"]), int(f["first"]), float(gs), stream_handle(),
                      hp=self._hp_ptr(f), skip=self._skip_ptr())
            return
        d = gr * gs + g["weight_decay"] * p
        if g["momentum"] != 0:
            if f["first"]:
                buf.copy_(d)
            else:
                buf.mul_(g["momentum"]).add_(d, alpha=1 - g["dampening"])
            d = d + g["momentum"] * buf if g["nesterov"] else buf
        p.add_(d, alpha=-g["lr"])


class FusedAdam(_FlatOptimizer):
    STATE_NAMES = ("exp_avg", "exp_avg_sq")

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled=False):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, decoupled=decoupled))

    def _hparams(self, group, step):
        b1, b2 = group["betas"]
        return float(group["lr"]), 1 - b1 ** step, 1 - b2 ** step

    def _update(self, g, f, off, n, gs):
        b1, b2 = g["betas"]
        _, bc1, bc2 = self._hparams(g, f["step"])
        p = f["param"][off:off + n]
        gr = f["grad"][off:off + n]
        m = f["states"]["exp_avg"][off:off + n]
        v = f["states"]["exp_avg_sq"][off:off + n]
        if p.is_cuda:
            lib().adam(ptr(p), ptr(gr), ptr(m), ptr(v), n, float(g["lr"]), float(b1), float(b2), float(g["eps"]),
                       float(g["weight_decay"]), int(g["decoupled"]), float(bc1), float(bc2), float(gs), stream_handle(),
                       hp=self._hp_ptr(f), skip=self._skip_ptr())
            return
        grad = gr * gs
        if g["decoupled"]:
            p.mul_(1 - g["lr"] * g["weight_decay"])
        else:
            grad = grad + g["weight_decay"] * p
        m.mul_(b1).add_(grad, alpha=1 - b1)
        v.mul_(b2).addcmul_(grad, grad, value=1 - b2)
        denom = (v / bc2).sqrt_().add_(g["eps"])
        p.addcdiv_(m, denom, value=-g["lr"] / bc1)


def _mix(h):
    """csrc/adamw.hip mix(): 32 mixed bits of a whole number below 2^32, held in int64."""
    h = h ^ (h >> 16)
    h = (h * 0x6C8E9CF5) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x5D2A4B35) & 0xFFFFFFFF
    return h ^ (h >> 16)


class FusedAdamW(_FlatOptimizer):
    """AdamW (decoupled weight decay, torch.optim.AdamW's update) over the flat buffer, one launch a
    group (csrc/adamw.hip). ``state_bits=32`` keeps fp32 moments ``exp_avg`` / ``exp_avg_sq``.

    ``state_bits=8`` keeps a quarter of that: ``exp_avg`` and ``exp_avg_root`` (the square root of the
    second moment) as ``torch.float8_e4m3fn`` codes, each block of 256 values of a tensor times an
    fp32 scale (``*_scale``). A tensor's codes start at a block of their own and are padded with
    zeros to whole blocks, in the order of the group's parameters. Codes are rounded
    stochastically from a hash of (``seed``, step, place): a run repeats bit for bit. That keeps the mean of
    ``exp_avg`` and of the root; the second moment itself, the root's square, settles up to 6 % above its
    mean (b2 = .999; the roots 1.4 %). Both kinds of state load from either
    kind of checkpoint."""

    STATE_NAMES = ("exp_avg", "exp_avg_sq")
    BLOCK, CHUNK = 256, 4096  # csrc/kernels.h DV_ADAMW_BLOCK, DV_ADAMW_CHUNK

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"FusedAdamW: state_bits must be 8 or 32, got {state_bits!r}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"FusedAdamW: betas must lie in [0, 1), got {betas!r}")
        if eps < 0 or lr < 0 or weight_decay < 0:
            raise ValueError(f"FusedAdamW: lr, eps and weight_decay must not be negative, got {lr!r}, {eps!r}, {weight_decay!r}")
        self.state_bits, self.seed = state_bits, int(seed) & 0xFFFFFFFF
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def _hparams(self, group, step):
        b1, b2 = group["betas"]
        return float(group["lr"]), 1 - b1 ** step, 1 - b2 ** step

    # ---------------- 8-bit state ----------------
    def _new_states(self, f):
        if self.state_bits == 32:
            return super()._new_states(f)
        dev, block, chunks, f["blocks"] = f["param"].device, 0, [], []
        for off, n in f["offsets"]:
            e = -(-n // self.BLOCK)
            f["blocks"].append((block, e))
            chunks += [(off + k, block + k // self.BLOCK, min(self.CHUNK, n - k)) for k in range(0, n, self.CHUNK)]
            block += e
        chunks.sort()  # by place in the flat buffer: a run of whole tensors there is a run of chunks
        f["chunk_starts"] = [c[0] for c in chunks]
        f["chunks"] = torch.tensor(chunks, dtype=torch.int64).reshape(-1, 3).to(dev)
        out = {}
        for name in ("exp_avg", "exp_avg_root"):
            out[name] = torch.zeros(block * self.BLOCK, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
            out[name + "_scale"] = torch.zeros(block, dtype=torch.float32, device=dev)
        return out

    def _slices(self, f, i):
        """The group's ``i``-th parameter's part of each 8-bit state buffer."""
        b, e = f["blocks"][i]
        return {name: buf[b:b + e] if name.endswith("_scale") else buf[b * self.BLOCK:(b + e) * self.BLOCK]
                for name, buf in f["states"].items()}

    def _carry_states(self, old, f):
        if self.state_bits == 32:
            return super()._carry_states(old, f)
        for name, buf in f["states"].items():
            buf.view(torch.uint8).copy_(old["states"][name].view(torch.uint8))

    def _save_state(self, f, i, shape):
        if self.state_bits == 32:
            return super()._save_state(f, i, shape)
        return {name: t.clone() for name, t in self._slices(f, i).items()}

    def load_state_dict(self, state_dict):
        self._check_packed(state_dict["state"])
        super().load_state_dict(state_dict)

    def _check_packed(self, state):
        """Refuse 8-bit states of tensors of other sizes, before any is loaded (one look at the device for all)."""
        sizes, ends = [n for f in self._flat if f is not None for _, n in f["offsets"]], {}
        for idx, n in enumerate(sizes):
            st = state.get(idx, state.get(str(idx))) or {}
            if "exp_avg_root" not in st:
                continue
            blocks = -(-n // self.BLOCK)
            for k in ("exp_avg", "exp_avg_root", "exp_avg_scale", "exp_avg_root_scale"):
                want = blocks if k.endswith("_scale") else blocks * self.BLOCK
                if st[k].numel() != want:
                    raise ValueError(f"FusedAdamW: {k} of a saved 8-bit state has {st[k].numel()} entries, expected {want}")
                if want > n and not k.endswith("_scale"):
                    ends.setdefault(st[k].device, []).append(st[k].reshape(-1)[n:].view(torch.uint8))
        if any((torch.cat(t) & 0x7F).any() for t in ends.values()):
            raise ValueError("FusedAdamW: a saved 8-bit state goes on behind its tensor's end: it is of a larger one")

    def _load_state(self, f, i, st):
        n = f["offsets"][i][1]
        packed = "exp_avg_root" in st
        if self.state_bits == 32 and packed:
            wide = {k: (st[k].float().view(-1, self.BLOCK) * st[k + "_scale"].float()[:, None]).view(-1)[:n]
                    for k in ("exp_avg", "exp_avg_root")}
            st = {"exp_avg": wide["exp_avg"], "exp_avg_sq": wide["exp_avg_root"] ** 2}
        if self.state_bits == 32:
            return super()._load_state(f, i, st)
        mine = self._slices(f, i)
        for name in ("exp_avg", "exp_avg_root"):
            if packed:
                mine[name].view(torch.uint8).copy_(st[name].contiguous().view(torch.uint8))
                mine[name + "_scale"].copy_(st[name + "_scale"])
            elif "exp_avg" in st and "exp_avg_sq" in st:  # 32-bit moments: rounded to nearest, once
                t = st["exp_avg"] if name == "exp_avg" else st["exp_avg_sq"].sqrt()
                wide = torch.zeros(mine[name].numel(), dtype=torch.float32, device=mine[name].device)
                wide[:n].copy_(t.reshape(-1))
                self._store8(mine, name, wide.view(-1, self.BLOCK), 0x80000)

    def _store8(self, states, name, t, noise):
        """Blocks ``t`` [blocks][256] as codes and scales, the kernel's arithmetic (csrc/adamw.hip)."""
        if not t.numel():
            return
        size = t.abs()
        top = torch.where(size < math.inf, size, 0.0).amax(1, keepdim=True)  # of what is finite
        up = torch.where(top >= 2.0 ** -100, torch.full_like(top, 448.0) / top, torch.zeros_like(top))
        s = size * up
        code = (((s * 2.0 ** -120).view(torch.int32).long() + noise) >> 20).clamp_(max=126)
        code = torch.where(s < 1e30, code, 127)
        if name == "exp_avg":
            code = code + 128 * (t < 0)
        else:
            code = torch.maximum(code, (t > 0).long())
        states[name].view(torch.uint8).copy_(code.to(torch.uint8).view(-1))
        states[name + "_scale"].copy_((top * torch.full_like(top, 1 / 448.0))[:, 0])

    # ---------------- update ----------------
    def _update(self, g, f, off, n, gs):
        if not n:
            return
        b1, b2 = g["betas"]
        _, bc1, bc2 = self._hparams(g, f["step"])
        s = f["states"]
        if f["param"].is_cuda:
            args = (float(g["lr"]), float(b1), float(b2), float(g["eps"]), float(g["weight_decay"]), bc1, bc2, float(gs))
            at, gat = ptr(f["param"]), ptr(f["grad"])
            with on_device(f["param"]):
                if self.state_bits == 32:
                    lib().adamw32(at + 4 * off, gat + 4 * off, ptr(s["exp_avg"]) + 4 * off, ptr(s["exp_avg_sq"]) + 4 * off, n,
                                  *args, self._hp_ptr(f), self._skip_ptr(), stream_handle())
                    return
                lo, hi = bisect_left(f["chunk_starts"], off), bisect_left(f["chunk_starts"], off + n)
                lib().adamw8(at, gat, ptr(s["exp_avg"]), ptr(s["exp_avg_scale"]), ptr(s["exp_avg_root"]),
                             ptr(s["exp_avg_root_scale"]), ptr(f["chunks"]) + 24 * lo, hi - lo, *args,
                             f["step"] & 0xFFFFFFFF, self.seed, self._hp_ptr(f), self._skip_ptr(), stream_handle())
            return
        p, gr = f["param"][off:off + n], f["grad"][off:off + n]
        if self.state_bits == 32:
            self._update_cpu(g, p, gr * gs, s["exp_avg"][off:off + n], s["exp_avg_sq"][off:off + n], bc1, bc2)
            return
        for i, (o, k) in enumerate(f["offsets"]):
            if k and off <= o < off + n:
                self._update8_cpu(g, f, i, gs, bc1, bc2)

    @staticmethod
    def _update_cpu(g, p, grad, m, v, bc1, bc2):
        b1, b2 = g["betas"]
        m.copy_(m * b1 + grad * (1 - b1))
        v.copy_(v * b2 + (grad * grad) * (1 - b2))
        p.copy_(p * (1 - g["lr"] * g["weight_decay"]) - g["lr"] / bc1 * (m / (v.sqrt() / math.sqrt(bc2) + g["eps"])))

    def _update8_cpu(self, g, f, i, gs, bc1, bc2):
        (o, n), (block, e), mine = f["offsets"][i], f["blocks"][i], self._slices(f, i)
        dev = f["param"].device
        grad = torch.zeros(e * self.BLOCK, device=dev)
        grad[:n] = f["grad"][o:o + n] * gs
        m, r = ((mine[k].float().view(e, self.BLOCK) * mine[k + "_scale"][:, None]).view(-1)
                for k in ("exp_avg", "exp_avg_root"))
        v, p = r * r, torch.zeros_like(grad)
        p[:n] = f["param"][o:o + n]
        self._update_cpu(g, p, grad, m, v, bc1, bc2)
        f["param"][o:o + n] = p[:n]
        key = _mix((self.seed + f["step"] * 0x9E3779B1) & 0xFFFFFFFF)
        place = torch.arange(block * self.BLOCK, (block + e) * self.BLOCK, device=dev)
        noise = _mix(((place & 0xFFFFFFFF) * 0x2545F491 + (place >> 32) * 0x7A6B3C5D + key) & 0xFFFFFFFF).view(e, self.BLOCK)
        self._store8(mine, "exp_avg", m.view(e, self.BLOCK), noise & 0xFFFFF)
        # the host's vector square root may be an ulp off: through 64 bits it is the kernel's
        self._store8(mine, "exp_avg_root", v.double().sqrt().float().view(e, self.BLOCK), noise >> 12)


class FusedRMSprop(_FlatOptimizer):
    STATE_NAMES = ("square_avg", "momentum_buffer", "grad_avg")

    def __init__(self, params, lr=1e-2, alpha=0.99, eps=1e-8, weight_decay=0.0, momentum=0.0, centered=False):
        super().__init__(params, dict(lr=lr, alpha=alpha, eps=eps, weight_decay=weight_decay, momentum=momentum,
                                      centered=centered))

    def _update(self, g, f, off, n, gs):
        p = f["param"][off:off + n]
        gr = f["grad"][off:off + n]
        sq = f["states"]["square_avg"][off:off + n]
        mom = f["states"]["momentum_buffer"][off:off + n]
        ga = f["states"]["grad_avg"][off:off + n]
        if p.is_cuda:
            lib().rmsprop(ptr(p), ptr(gr), ptr(sq), ptr(mom), ptr(ga), n, float(g["lr"]), float(g["alpha"]),
                          float(g["eps"]), float(g["weight_decay"]), float(g["momentum"]), int(g["centered"]), float(gs),
                          stream_handle(), hp=self._hp_ptr(f), skip=self._skip_ptr())
            return
        grad = gr * gs + g["weight_decay"] * p
        sq.mul_(g["alpha"]).addcmul_(grad, grad, value=1 - g["alpha"])
        if g["centered"]:
            ga.mul_(g["alpha"]).add_(grad, alpha=1 - g["alpha"])
            avg = (sq - ga * ga).sqrt_().add_(g["eps"])
        else:
            avg = sq.sqrt().add_(g["eps"])
        if g["momentum"] > 0:
            mom.mul_(g["momentum"]).addcdiv_(grad, avg)
            p.add_(mom, alpha=-g["lr"])
        else:
            p.addcdiv_(grad, avg, value=-g["lr"])


OPTIMIZERS = {"SGD": FusedSGD, "Adam": FusedAdam, "AdamW": FusedAdamW, "RMSprop": FusedRMSprop}
