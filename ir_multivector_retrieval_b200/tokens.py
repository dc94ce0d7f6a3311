"""Token operators on device tensors: a table read by token id with scaling
and its gradient by sorted tokens, and rows sorted by group (an expert, a
centroid, a token id) and back, with weights applied, and their gradients.

``plan`` sorts the ids once; the table's gradient (``lookup_grad``) and the
grouping (``group``, ``ungroup``) read it. A group is any id below ``rows``:
the expert a router chose, the centroid ``tac.cluster_flat`` assigned.

All tensors are torch tensors on one GPU: rows f32, bf16 or f16, ids int32,
int64 or uint32, scales and weights f32. Inputs whose rows are not consecutive
inside, or 2^32 and more elements apart, are copied first; such outputs are
refused. Ids outside [0, rows), negative ones among them, name no row. The
calls enqueue on the stream given to ``ctx.set_stream``, else on torch's
current stream, and return without waiting; after one ordinary call on the GPU
they may be captured into a CUDA graph. There is no CPU fallback.

No autograd graph is made: results are detached, also where an input requires
a gradient, and the gradients are calls of their own. A tensor given as
``out`` counts as changed in place, so a graph that saved what it held before
is refused by ``backward``. Inputs and outputs of a call must not overlap.
"""
from __future__ import annotations

import atexit
import ctypes as C
import functools
import threading
from dataclasses import dataclass

import torch
from torch.autograd.graph import increment_version as _written

from . import _lib
from ._lib import CODES, MvrError

MAX_IDS = 2**31 - 1

_F32, _I32 = torch.float32, torch.int32
_ROW_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # mvr_dtype
_ID_BYTES = {torch.int32: 4, torch.uint32: 4, torch.int64: 8}


def _refuse(msg: str, name: str = "InvalidArgument"):
    raise MvrError(CODES[name], msg)


def _dtype(t, what: str) -> int:
    d = _ROW_TYPES.get(getattr(t, "dtype", None))
    if d is None:
        _refuse(f"{what} must be a float32, bfloat16 or float16 tensor, not {getattr(t, 'dtype', type(t))}")
    return d


def _id_bytes(ids) -> int:
    n = _ID_BYTES.get(getattr(ids, "dtype", None))
    if n is None:
        _refuse(f"ids must be an int32, int64 or uint32 tensor, not {getattr(ids, 'dtype', type(ids))}")
    return n


def _ends(shape) -> set:
    """Where the dimensions of a shape end, counted in elements from its last
    dimension to the first: what splitting and merging dimensions keeps."""
    ends, k = set(), 1
    for d in reversed(shape):
        k *= d
        ends.add(k)
    ends.discard(1)
    return ends


def _in_order(shape, of) -> bool:
    """Whether values of shape `shape` stand for those of shape `of` one by one
    in memory order: the same dimensions, some of them split or merged (flat
    among them). A transposed shape has as many values, each beside the wrong
    one. Both shapes have the same number of values."""
    a, b = _ends(shape), _ends(of)
    return 0 in a or a <= b or b <= a


def _rows(t, what: str, n: int | None = None, dim: int | None = None, of=None):
    """`t` as a 2-D view, its row length and its row stride. Copied where its
    rows are not consecutive inside or 2^32 and more elements apart, which the
    library refuses: such rows are few. `of`: the shape of what its rows belong
    to."""
    if t.dim() != 2:
        if t.dim() < 2:
            _refuse(f"{what} must have rows: at least two dimensions", "DimMismatch")
        if t.shape[-1] == 0:
            _refuse(f"{what} has rows of length 0", "DimMismatch")
        lead = t.shape[:-1]
        t = t.reshape(-1, t.shape[-1])
        if of is not None and lead != of and t.shape[0] == n and not _in_order(lead, of):
            _refuse(f"{what} has rows in shape {tuple(lead)}, not {tuple(of)}", "LengthMismatch")
    m, d = t.shape
    if dim is not None and d != dim:
        _refuse(f"{what} has rows of {d}, not {dim}", "DimMismatch")
    if n is not None and m != n:
        _refuse(f"{what} has {m} rows, not {n}", "LengthMismatch")
    if d == 0:
        _refuse(f"{what} has rows of length 0", "DimMismatch")
    stride, one = t.stride()
    if one != 1 and d > 1 or stride >> 32 and m > 1:
        t = t.contiguous()
        stride = d
    return t, d, stride if m > 1 else d


def _out_rows(t, what: str, n: int, dim: int, dtype, of=None):
    """Address and row stride of an output given by the caller: written in
    place, so never copied. `of`: the shape of what its rows belong to."""
    if t.dtype != dtype:
        _refuse(f"{what} must be {dtype}, not {t.dtype}")
    if t.dim() < 2 or t.shape[-1] != dim:
        _refuse(f"{what} must have rows of {dim}", "DimMismatch")
    if t.numel() != n * dim:
        _refuse(f"{what} must have {n} rows of {dim}", "OutBufferWrongSize")
    if t.dim() > 2:
        if of is not None and t.shape[:-1] != of and not _in_order(t.shape[:-1], of):
            _refuse(f"{what} must have {dim} elements for each id of {tuple(of)}", "OutBufferWrongSize")
        try:
            t = t.view(n, dim)
        except RuntimeError:
            _refuse(f"{what} must be viewable as {n} rows")
    stride, one = t.stride()
    if dim > 1 and one != 1 or n > 1 and stride < dim:
        _refuse(f"{what} must have consecutive, separate rows")
    return t.data_ptr(), stride if n > 1 else dim


def _f32(t, n: int, of, what: str):
    """`t` with one value for each of the n ids of shape `of`."""
    if t.dtype != _F32:
        _refuse(f"{what} must be float32, not {t.dtype}")
    if t.shape != of:
        if t.numel() != n:
            _refuse(f"{what} has {t.numel()} values, not {n}", "LengthMismatch")
        if not _in_order(t.shape, of):
            _refuse(f"{what} has shape {tuple(t.shape)}, not {tuple(of)}", "LengthMismatch")
    return t if t.is_contiguous() else t.contiguous()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _stream_of(device: int) -> int:
    """Handle of torch's current stream; 1 names the legacy default stream,
    whose own handle, 0, would select a context's own stream."""
    return _raw_stream(device) or 1


class _Follower:
    """A context of its own for each GPU, for calls that name none: its stream
    is the one torch used at the last call, so that it is only set anew when
    that changes."""

    def __init__(self, device: int):
        self.ctx = _lib.Context(device)
        self.at = None


_followers: dict = {}
_followers_lock = threading.Lock()


@atexit.register
def _let_go():
    # a context waits for its stream when it ends, and a stream of the
    # program's may be gone by then
    for f in _followers.values():
        f.ctx.lib.mvr_ctx_set_stream(f.ctx.handle, None)


def _follower(device: int) -> _Follower:
    f = _followers.get(device)
    if f is None:
        with _followers_lock:
            f = _followers.get(device)
            if f is None:
                f = _followers[device] = _Follower(device)
    return f


def _run(ctx, device: int, name: str, *args):
    """The library's `name` on the right context and stream, its status
    checked. Contexts are not for two calls at once, hence the locks."""
    if ctx is None:
        f = _followers.get(device) or _follower(device)
        ctx = f.ctx
        with ctx.lock:
            here = _raw_stream(device) or 1
            if f.at != here:
                ctx.lib.mvr_ctx_set_stream(ctx.handle, here)
                f.at = here
            status = getattr(ctx.lib, name)(ctx.handle, *args)
            if status:
                ctx.check(status)
        return
    if ctx.device != device:
        _refuse(f"tensors on device {device}, context on device {ctx.device}")
    with ctx.lock:
        own = ctx.stream == 0
        if own:
            ctx.lib.mvr_ctx_set_stream(ctx.handle, _stream_of(device))
        try:
            status = getattr(ctx.lib, name)(ctx.handle, *args)
            if status:
                ctx.check(status)
        finally:
            if own:
                ctx.lib.mvr_ctx_set_stream(ctx.handle, None)


def _device_of(*tensors) -> int:
    """The GPU that all the tensors lie on."""
    device = -1
    for t in tensors:
        if t is None:
            continue
        d = t.get_device() if isinstance(t, torch.Tensor) else -1
        if d < 0:
            _refuse("all tensors must be CUDA tensors (there is no CPU fallback)")
        if d != device:
            if device >= 0:
                _refuse(f"tensors on devices {device} and {d}")
            device = d
    return device


def _on_its_stream(call):
    """With a stream given to ``ctx.set_stream`` that is not torch's current
    one, results and copies come from that stream's memory pool, and the
    inputs stay alive for it."""

    @functools.wraps(call)
    def wrapped(*args, ctx=None, **kw):
        if ctx is None or ctx.stream == 0 or ctx.stream == _stream_of(ctx.device):
            return call(*args, ctx=ctx, **kw)
        s = torch.cuda.ExternalStream(ctx.stream, device=ctx.device)
        for t in (*args, *kw.values()):
            for u in (t.offsets, t.order, t.keys, t.slot) if isinstance(t, Plan) else (t,):
                if isinstance(u, torch.Tensor) and u.is_cuda:
                    u.record_stream(s)
        with torch.cuda.stream(s):
            return call(*args, ctx=ctx, **kw)

    return wrapped


@dataclass
class Plan:
    """The ids of n tokens (``columns`` each) in stable sorted order, as int32
    tensors. ``order[p]`` is the flat index of the id at sorted place p,
    ``keys[p]`` its value, ``offsets`` (rows + 1) the first place of each
    value; ``slot`` has the ids' shape and holds each one's place, -1 where it
    names no row. ``offsets[rows]`` is the number of ids that name a row;
    from there on ``order`` lists those that name none and ``keys`` is ``rows``."""

    rows: int
    offsets: object
    order: object
    keys: object
    slot: object

    @property
    def n_ids(self) -> int:
        return self.slot.numel()

    @property
    def columns(self) -> int:
        return self.slot.shape[-1] if self.slot.dim() > 1 else 1

    @property
    def n(self) -> int:
        s = self.slot.shape
        return self.slot.numel() // s[-1] if len(s) > 1 and s[-1] else s[0] if len(s) == 1 else 0

    def _check(self):
        offsets, order, keys, slot = self.offsets, self.order, self.keys, self.slot
        if not (offsets.dtype == order.dtype == keys.dtype == slot.dtype == _I32 and offsets.is_contiguous()
                and order.is_contiguous() and keys.is_contiguous() and slot.is_contiguous()):
            _refuse("a plan's tensors must be contiguous int32 tensors")
        n = slot.numel()
        if offsets.numel() != self.rows + 1 or order.numel() != n or keys.numel() != n:
            _refuse("plan: sizes differ", "LengthMismatch")
        return n


@functools.lru_cache(maxsize=256)
def _plan_bytes(n: int, rows: int) -> int:
    need = C.c_uint64(0)
    st = _lib.load().mvr_token_plan_bytes(n, rows, C.byref(need))
    if st:
        raise MvrError(st, "token_plan_bytes")
    return need.value


@functools.lru_cache(maxsize=256)
def _grad_bytes(n: int, dim: int) -> int:
    need = C.c_uint64(0)
    st = _lib.load().mvr_lookup_grad_bytes(n, dim, C.byref(need))
    if st:
        raise MvrError(st, "lookup_grad_bytes")
    return need.value


def _workspace(like, need: int):
    return like.new_empty(need, dtype=torch.uint8) if need else None


def _ptr(t):
    return None if t is None else t.data_ptr()


@_on_its_stream
def plan(ids, rows: int, *, ctx=None) -> Plan:
    """Sort the ids ([n] or [n, columns]) by value, stable."""
    rows = int(rows)
    if not 0 < rows < MAX_IDS:
        _refuse(f"rows must be in [1, 2^31 - 2], not {rows}")
    idb = _id_bytes(ids)
    dims = ids.dim()
    if dims not in (1, 2):
        _refuse("ids must have one or two dimensions")
    if dims == 2 and ids.shape[1] == 0:
        _refuse("ids have no columns")
    n = ids.numel()
    if n > MAX_IDS:
        _refuse("more than 2^31 - 1 ids")
    device = _device_of(ids)
    ids = ids.contiguous()
    offsets, order, keys, slot = ids.new_empty(rows + 1 + 3 * n, dtype=_I32).split((rows + 1, n, n, n))
    if dims == 2:
        slot = slot.view(ids.shape)
    need = _plan_bytes(n, rows)
    ws = _workspace(ids, need)
    _run(ctx, device, "mvr_token_plan_device", ids.data_ptr(), idb, n, rows, offsets.data_ptr(), order.data_ptr(),
         keys.data_ptr(), slot.data_ptr(), _ptr(ws), need)
    return Plan(rows, offsets, order, keys, slot)


@_on_its_stream
def lookup(table, ids, *, scale=None, alpha: float = 1.0, out=None, ctx=None):
    """``out[i] = (alpha * scale[i]) * table[ids[i]]``: the ids' shape plus the
    table's row length, in the table's type; zero rows where an id names none.
    ``scale`` (the ids' shape, f32) and ``out`` are optional. What has the ids'
    shape here and below may have its dimensions split or merged, flat for
    instance; another shape of as many values is refused."""
    dt = _dtype(table, "table")
    idb = _id_bytes(ids)
    n = ids.numel()
    if table.dim() != 2:
        _refuse("table must have two dimensions", "DimMismatch")
    device = _device_of(table, ids, scale, out)
    rows = table.shape[0]
    table, dim, ts = _rows(table, "table")
    flat = ids.contiguous()
    if scale is not None:
        scale = _f32(scale, n, ids.shape, "scale")
    given = out
    if out is None:
        out = table.new_empty((*ids.shape, dim))
        po, so = out.data_ptr(), dim
    else:
        po, so = _out_rows(out, "out", n, dim, table.dtype, ids.shape)
    _run(ctx, device, "mvr_lookup_device", table.data_ptr(), dt, rows, dim, ts, flat.data_ptr(), idb, n, _ptr(scale),
         alpha, po, so)
    if given is not None:
        _written(given)
    return out


@_on_its_stream
def lookup_grad(grad, plan: Plan, *, scale=None, alpha: float = 1.0, table=None, out=None, accumulate: bool = False,
                ctx=None):
    """Gradients of ``lookup`` from that of its output (the ids' shape plus the
    row length) and the plan of its ids: the table's, ``dtable[v] = sum alpha *
    scale[i] * grad[i]`` over the ids of v (rows without an id: zeros), and,
    where ``table`` is given, also the scale's, ``alpha * <grad[i],
    table[ids[i]]>`` as the second of a pair. ``out`` (grad's type or f32)
    receives the first; with ``accumulate`` the sums are added to it and rows
    without an id are not touched."""
    dt = _dtype(grad, "grad")
    n = plan._check()
    rows = plan.rows
    if accumulate and out is None:
        _refuse("accumulate needs out")
    device = _device_of(grad, plan.offsets, plan.order, plan.keys, plan.slot, scale, table, out)
    grad, dim, gs = _rows(grad, "grad", n, None, plan.slot.shape)
    if scale is not None:
        scale = _f32(scale, n, plan.slot.shape, "scale")
    tp, ts, dscale = None, dim, None
    if table is not None:
        if table.dtype != grad.dtype:
            _refuse(f"table is {table.dtype}, grad {grad.dtype}")
        table, _, ts = _rows(table, "table", rows, dim)
        tp = table.data_ptr()
        dscale = grad.new_empty(plan.slot.shape, dtype=_F32)
    given = out
    if out is None:
        out = grad.new_empty((rows, dim))
        po, so, odt = out.data_ptr(), dim, dt
    else:
        odt = _dtype(out, "out")
        if odt not in (dt, 0):
            _refuse("out must have grad's type or float32")
        po, so = _out_rows(out, "out", rows, dim, out.dtype)
    need = _grad_bytes(n, dim)
    ws = _workspace(grad, need)
    _run(ctx, device, "mvr_lookup_grad_device", grad.data_ptr(), dt, gs, n, rows, dim, plan.offsets.data_ptr(),
         plan.order.data_ptr(), plan.keys.data_ptr(), _ptr(scale), alpha, tp, ts, po, odt, so, int(accumulate),
         _ptr(dscale), _ptr(ws), need)
    if given is not None:
        _written(given)
    return out if dscale is None else (out, dscale)


def _token_call(name: str, src, what: str, from_n: int, plan: Plan, weights, to_n: int, out, ctx):
    """group and ungroup: rows of `src` to rows of `out`."""
    dt = _dtype(src, what)
    n_ids = plan._check()
    slot = plan.slot
    device = _device_of(src, slot, weights, out)
    src, dim, ss = _rows(src, what, from_n)
    if weights is not None:
        weights = _f32(weights, n_ids, slot.shape, "weights")
    given = out
    if out is None:
        out = src.new_empty((to_n, dim))
        po, so = out.data_ptr(), dim
    else:
        po, so = _out_rows(out, "out", to_n, dim, src.dtype)
    _run(ctx, device, name, src.data_ptr(), dt, ss, plan.n, plan.columns, dim, slot.data_ptr(), _ptr(weights), po, so)
    if given is not None:
        _written(given)
    return out


def _token_grad(name: str, src, from_n: int, plan: Plan, weights, other, other_what: str, other_n: int, to_n: int,
                out, ctx):
    """Their gradients: also the weights' where the forward rows are given."""
    dt = _dtype(src, "dout")
    n_ids = plan._check()
    slot = plan.slot
    device = _device_of(src, slot, weights, other, out)
    src, dim, ss = _rows(src, "dout", from_n)
    if weights is not None:
        weights = _f32(weights, n_ids, slot.shape, "weights")
    dw, op, os_ = None, None, dim
    if other is not None:
        if other.dtype != src.dtype:
            _refuse(f"{other_what} is {other.dtype}, dout {src.dtype}")
        other, _, os_ = _rows(other, other_what, other_n, dim)
        op = other.data_ptr()
        dw = src.new_empty(slot.shape, dtype=_F32)
    given = out
    if out is None:
        out = src.new_empty((to_n, dim))
        po, so = out.data_ptr(), dim
    else:
        po, so = _out_rows(out, "out", to_n, dim, src.dtype)
    _run(ctx, device, name, src.data_ptr(), dt, ss, plan.n, plan.columns, dim, slot.data_ptr(), _ptr(weights), op, os_,
         po, so, _ptr(dw))
    if given is not None:
        _written(given)
    return out if dw is None else (out, dw)


@_on_its_stream
def group(x, plan: Plan, *, weights=None, out=None, ctx=None):
    """The rows of x (one a token) in sorted order: ``out[slot[i, c]] =
    weights[i, c] * x[i]``, n * columns rows. Rows behind the last sorted one
    keep what ``out`` held (without ``out`` they are undefined)."""
    return _token_call("mvr_group_rows_device", x, "x", plan.n, plan, weights, plan.n_ids, out, ctx)


@_on_its_stream
def group_grad(dout, plan: Plan, *, weights=None, x=None, out=None, ctx=None):
    """Gradients of ``group`` from that of its output: ``dx[i] = sum_c
    weights[i, c] * dout[slot[i, c]]`` and, where ``x`` is given, also that of
    the weights, ``<x[i], dout[slot[i, c]]>``, as the second of a pair."""
    return _token_grad("mvr_group_rows_grad_device", dout, plan.n_ids, plan, weights, x, "x", plan.n, plan.n, out, ctx)


@_on_its_stream
def ungroup(xs, plan: Plan, *, weights=None, out=None, ctx=None):
    """Sorted rows back to their tokens: ``out[i] = sum_c weights[i, c] *
    xs[slot[i, c]]``; zeros for a token none of whose ids names a row."""
    return _token_call("mvr_ungroup_rows_device", xs, "xs", plan.n_ids, plan, weights, plan.n, out, ctx)


@_on_its_stream
def ungroup_grad(dout, plan: Plan, *, weights=None, xs=None, out=None, ctx=None):
    """Gradients of ``ungroup`` from that of its output: ``dxs[slot[i, c]] =
    weights[i, c] * dout[i]`` (rows behind the last sorted one keep what
    ``out`` held) and, where ``xs`` is given, also that of the weights,
    ``<dout[i], xs[slot[i, c]]>``, as the second of a pair."""
    return _token_grad("mvr_ungroup_rows_grad_device", dout, plan.n, plan, weights, xs, "xs", plan.n_ids, plan.n_ids,
                       out, ctx)


__all__ = ["Plan", "plan", "lookup", "lookup_grad", "group", "group_grad", "ungroup", "ungroup_grad"]
