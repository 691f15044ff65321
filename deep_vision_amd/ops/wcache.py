"""Cache of the bf16 MFMA operand layouts of every conv / linear weight.

The kernels consume weights as bf16 ``[G][Og][R][S][Cpad]`` (forward) and ``[G][Ig][R][S][Opad]``
(dgrad). Re-laying them out per layer per call costs one launch each (107 per ResNet-50 step).
Here each (parameter, layout) gets a persistent buffer:

* a hit needs the same global *weights epoch*, the same parameter ``_version`` (user in-place
  edits bump it) and the same storage pointer;
* the fused optimizers call ``after_step()`` once per step: the epoch advances and ONE batched
  kernel (csrc/elementwise.hip ``wprep_batched_kernel``) refreshes every registered buffer on the
  current stream, right after the parameter update -- so the next forward / backward only hit.
"""
from __future__ import annotations

import struct
import weakref

import torch

from .._ext import lib, ptr, stream_handle

_entries = {}  # key -> [param weakref, buf, epoch, version, data_ptr, geometry, (event, streams behind it) or None]
_epoch = 0
_tables = {}  # device -> (n_entries_snapshot, descs, chunks, nchunks)
ENABLED = True
_step_captures = 0


class step_capture:
    """Context of the capture of a whole training step (train.graph.CapturedStep): the captured ``after_step()``
    refreshes the cached operands in every replay."""

    def __enter__(self):
        global _step_captures
        _step_captures += 1

    def __exit__(self, *exc):
        global _step_captures
        _step_captures -= 1


def outdated_in_replays():
    """Whether the current stream captures something else than a training step. Its replays meet parameters that
    were changed in between, and this cache has no part in them: a hit records nothing into the graph."""
    return torch.cuda.is_current_stream_capturing() and not _step_captures


def _key(param, G, pad, mode, Sp=0):
    return (id(param), G, pad, mode, Sp)


def get(param, G, pad, mode, compute, Sp=0):
    """bf16 operand of ``param`` in layout (G, pad, mode[, Sp]); ``compute(out)`` fills a buffer.
    mode 2 = the forward layout with the filter width padded to ``Sp`` (tap-packed stem)."""
    if not ENABLED:
        return compute(None)
    k = _key(param, G, pad, mode, Sp)
    e = _entries.get(k)
    if e is not None and e[0]() is param:
        if e[2] == _epoch and e[3] == param._version and e[4] == param.data_ptr():
            if e[6] is not None:
                _behind(e[6])
            return e[1]
        buf = compute(e[1])
    else:
        buf = compute(None)
        _tables.pop(buf.device, None)
    _entries[k] = [weakref.ref(param), buf, _epoch, param._version, param.data_ptr(), (G, pad, mode, Sp), _laid_out(buf)]
    return buf


def _laid_out(buf):
    """The event behind the launch that fills ``buf``. Streams that only read a parameter need no order among
    themselves, but the first of them has written its operand."""
    if not buf.is_cuda or torch.cuda.is_current_stream_capturing():
        return None
    event = torch.cuda.Event()
    event.record()
    return event, {stream_handle()}


def _behind(ready):
    event, streams = ready
    if stream_handle() not in streams and not torch.cuda.is_current_stream_capturing():  # (captures begin synchronised)
        torch.cuda.current_stream().wait_event(event)
        streams.add(stream_handle())


def _build_table(device):
    descs, chunks = [], []
    chunk = int(lib().WPREP_CHUNK)
    live = []
    for k, e in list(_entries.items()):
        p = e[0]()
        if p is None:
            del _entries[k]
            continue
        if e[1].device != device or p.dtype != torch.float32 or not p.is_contiguous():
            continue
        if e[4] != p.data_ptr():  # moved since its last use: laid out from there by the launch that follows
            e[2], e[4] = None, p.data_ptr()
        G, pad, mode, Sp = e[5]
        shp = p.shape if p.dim() == 4 else (p.shape[0], p.shape[1], 1, 1)
        O, Ig, R, S = shp
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
        live.append(k)
    if not descs:
        return None
    assert len(descs[0]) == int(lib().WPREP_DESC_BYTES)
    dbuf = torch.frombuffer(bytearray(b"".join(descs)), dtype=torch.uint8).to(device)
    cbuf = torch.tensor(chunks, dtype=torch.int32).reshape(-1, 2).to(device)
    return (len(_entries), dbuf, cbuf, len(chunks), live)


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


def after_step(device=None):
    """Advance the weights epoch and refresh every cached operand of ``device`` in one launch."""
    global _epoch
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


def clear():
    _entries.clear()
    _tables.clear()
