"""Cache of the bf16 MFMA operand layouts of every conv / linear weight.

The kernels consume weights as bf16 ``[G][Og][R][S][Cpad]`` (forward) and ``[G][Ig][R][S][Opad]``
(dgrad). Re-laying them out per layer per call costs one launch each (107 per ResNet-50 step).
Here each (parameter, layout) gets a persistent buffer:

* a hit needs the same global *weights epoch*, the same parameter ``_version`` (user in-place
  edits bump it) and the same storage pointer;
* the fused optimizers call ``after_step()`` once per step: the epoch advances and ONE batched
  kernel (csrc/elementwise.hip ``wprep_batched_kernel``) refreshes every registered buffer on the
  current stream, right after the parameter update -- so the next forward / backward only hit.
* a captured training step refreshes its own parameters' buffers in every replay (``step_capture``);
* a buffer that one stream laid out is waited for by the first use on another, until a step has refreshed it.
"""
from __future__ import annotations

import struct
import weakref

import torch

from .._ext import lib, ptr, stream_handle

_entries = {}  # key -> [param weakref, buf, epoch, version, data_ptr, geometry, streams in order behind the layout or None]
_epoch = 0
_tables = {}  # device -> (n_entries_snapshot, descs, chunks, nchunks)
ENABLED = True
_captures = []  # step_capture contexts that are open
_replayed = {}  # those whose graphs ran since the cache was last used


class step_capture:
    """Context of the capture of a whole training step over ``params`` (train.graph.CapturedStep), entered before the
    capture begins. The captured ``after_step()`` refreshes their operands in every replay, from a table that is
    made here: made during the capture it would be copied from host memory that is gone when a replay reads
    it, and the one of eager steps holds other models' operands and is replaced when they change. The object
    keeps everything that the replays touch alive, and belongs to the owner of the graph."""

    def __init__(self, params):
        self.params = {id(p): p for p in params}
        self.table = None

    def __enter__(self):
        _settle()
        keys = [k for k, e in list(_entries.items()) if id(e[0]()) in self.params and e[1].is_cuda and _batched(e[0]())]
        devices = {_entries[k][1].device for k in keys}
        if len(devices) > 1:
            raise ValueError("a captured step's parameters must live on one device")
        self.laid = {k: (_entries[k][1], _entries[k][0]().data_ptr()) for k in keys}
        if devices:
            self.table = _make_table(keys, devices.pop())
        self.version = self._version()
        _captures.append(self)
        return self

    def _version(self):
        return sum([p._version for p in self.params.values()])

    def __exit__(self, *exc):
        _captures.remove(self)

    def refresh(self):
        """Launch, or record, what lays out every operand anew."""
        if self.table is not None:
            lib().wprep_batched(ptr(self.table[0]), ptr(self.table[1]), self.table[2], stream_handle())

    def catch_up(self):
        """Before a replay: parameters that torch operations have changed since (a loaded checkpoint) are laid out anew,
        as the graph's own forward pass only reads the operands."""
        version = self._version()
        if version != self.version:
            self.version = version
            self.refresh()

    def replayed(self):
        """The graph has been launched: the operands it refreshes are those of the new parameters."""
        _replayed[id(self)] = self


def _settle():
    """Bring the entries in line with the replays since the last use: those that every replayed graph refreshes are
    valid, others of its parameters were laid out before the last steps. (A version or an address that has
    changed is not taken over: such an entry is laid out anew.)"""
    global _replayed
    if not _replayed:
        return
    graphs, _replayed = list(_replayed.values()), {}
    for k, e in list(_entries.items()):
        p = e[0]()
        with_it = [c for c in graphs if p is not None and id(p) in c.params]
        if with_it:
            same = all(k in c.laid and c.laid[k][0] is e[1] and c.laid[k][1] == e[4] for c in with_it)
            e[2], e[6] = (_epoch, None) if same else (None, e[6])


def outdated_in_replays():
    """Whether the current stream captures something else than a training step. Its replays meet parameters that
    were changed in between, and this cache has no part in them: a hit records nothing into the graph."""
    return torch.cuda.is_current_stream_capturing() and not _captures


def _capturing():
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


def _key(param, G, pad, mode, Sp=0):
    return (id(param), G, pad, mode, Sp)


def get(param, G, pad, mode, compute, Sp=0):
    """bf16 operand of ``param`` in layout (G, pad, mode[, Sp]); ``compute(out)`` fills a buffer.
    mode 2 = the forward layout with the filter width padded to ``Sp`` (tap-packed stem)."""
    if not ENABLED:
        return compute(None)
    if _replayed:  # (the call itself costs as much as a hit)
        _settle()
    k = _key(param, G, pad, mode, Sp)
    e = _entries.get(k)
    if e is not None and e[0]() is param:
        if e[2] == _epoch and e[3] == param._version and e[4] == param.data_ptr():
            if e[6] is not None:
                _behind(e[6])
            return e[1]
        if _capturing():
            return compute(None)  # the graph's own: nothing is in it before a replay
        buf = compute(e[1])
    else:
        buf = compute(None)
        if _capturing():
            return buf
        _tables.pop(buf.device, None)
    _entries[k] = [weakref.ref(param), buf, _epoch, param._version, param.data_ptr(), (G, pad, mode, Sp),
                   [stream_handle()]]
    return buf


def _behind(streams):
    """Streams that only read a parameter need no order among themselves, but the first of them (``streams[0]``) has
    written its operand: the current one waits for it, once. (A capture begins synchronised.)"""
    now = stream_handle()
    if now in streams or _capturing():
        return
    first = torch.cuda.default_stream() if streams[0] == 0 else torch.cuda.ExternalStream(streams[0])
    torch.cuda.current_stream().wait_stream(first)
    streams.append(now)


def _build_table(device):
    live, params = [], []  # the parameters stay alive while their addresses are written down
    for k, e in list(_entries.items()):
        p = e[0]()
        if p is None:
            del _entries[k]
            continue
        if e[1].device != device or not _batched(p):
            continue
        if e[4] != p.data_ptr():  # moved since its last use: laid out from there by the launch that follows
            e[2], e[4] = None, p.data_ptr()
        live.append(k)
        params.append(p)
    t = _make_table(live, device)
    return None if t is None else (len(_entries), *t, live)


def _batched(p):
    return p.dtype == torch.float32 and p.is_contiguous()


def _make_table(keys, device):
    """(descriptors, chunks, number of chunks) of one launch over the entries ``keys``; None if there are none."""
    descs, chunks = [], []
    chunk = int(lib().WPREP_CHUNK)
    for k in keys:
        e = _entries[k]
        p = e[0]()
        G, O, Ig, R, S, pad, mode, Sp = _geometry(e)
        Og = O // G
        total = G * (Ig if mode == 1 else Og) * R * (Sp if mode == 2 else S) * pad
        di = len(descs)
        descs.append(struct.pack("<qqqiiiiiiii", p.data_ptr(), e[1].data_ptr(), total, G, Og, Ig, R, S, pad, mode, Sp))
        if mode == 1:  # 64x64 transpose tiles per group (wprep_batched_kernel)
            K = Ig * R * S
            ntiles = G * ((K + 63) // 64) * ((pad + 63) // 64)
        else:
            ntiles = (total + chunk - 1) // chunk
        chunks += [(di, c) for c in range(ntiles)]
    if not descs:
        return None
    assert len(descs[0]) == int(lib().WPREP_DESC_BYTES)
    dbuf = torch.frombuffer(bytearray(b"".join(descs)), dtype=torch.uint8).to(device)
    cbuf = torch.tensor(chunks, dtype=torch.int32).reshape(-1, 2).to(device)
    return dbuf, cbuf, len(chunks)


def _geometry(e):
    G, pad, mode, Sp = e[5]
    p = e[0]()
    O, Ig, R, S = p.shape if p.dim() == 4 else (p.shape[0], p.shape[1], 1, 1)
    return G, O, Ig, R, S, pad, mode, Sp


def _table_params(t):
    """The table's parameters as strong references (held across the launch: a garbage-collected
    model could otherwise free one between the check and the bookkeeping), or None when the
    table is stale (an entry added / dropped, a parameter dead or re-allocated)."""
    if t[0] != len(_entries):
        return None
    params = []
    for k in t[4]:
        e = _entries.get(k)
        p = e[0]() if e is not None else None
        if p is None or p.data_ptr() != e[4]:
            return None
        params.append(p)
    return params


def after_step(device=None, owner=None):
    """Advance the weights epoch and refresh every cached operand of ``device`` in one launch. In a capture, where
    the host does not see the steps, refresh those of the captured step or of the optimizer ``owner``."""
    global _epoch
    if _entries and _capturing():
        if _captures:
            _captures[-1].refresh()
        if owner is not None:
            _refresh_one_by_one(owner, _captures[-1].params if _captures else ())
        return
    _settle()
    _epoch += 1
    if not ENABLED or not _entries:
        return
    device = device or torch.device("cuda", torch.cuda.current_device())
    t = _tables.get(device)
    params = _table_params(t) if t is not None else None
    while params is None:
        t = _build_table(device)  # (drops dead entries; bakes in the current data pointers)
        if t is None:
            _tables.pop(device, None)
            return
        _tables[device] = t
        params = _table_params(t)  # None only if a parameter died while the table was built
    lib().wprep_batched(ptr(t[1]), ptr(t[2]), t[3], stream_handle())
    for k, p in zip(t[4], params):
        e = _entries[k]
        # (whoever reads the parameters next is ordered behind this step, which has written them too)
        e[2], e[3], e[4], e[6] = _epoch, p._version, p.data_ptr(), None


def _refresh_one_by_one(owner, done=()):
    """A step captured by hand: a launch an operand, whose arguments the graph holds itself. The optimizer keeps
    the operands, as it keeps the parameters."""
    mine = {id(p) for g in owner.param_groups for p in g["params"]}
    for e in list(_entries.values()):
        p = e[0]()
        if p is None or id(p) not in mine or id(p) in done or not _batched(p):
            continue
        G, O, Ig, R, S, pad, mode, Sp = _geometry(e)
        lib().wprep(ptr(p), ptr(e[1]), G, O // G, Ig, R, S, pad, mode, Sp, stream_handle())
        owner.__dict__.setdefault("_captured_operands", []).append(e[1])


def clear():
    _entries.clear()
    _tables.clear()
    _replayed.clear()
