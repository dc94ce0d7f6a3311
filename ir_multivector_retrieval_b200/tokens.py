"""Token operators on device tensors: a table read by token id with scaling
and its gradient by sorted tokens, and rows sorted by group (an expert, a
centroid, a token id) and back, with weights applied, and their gradients.

``plan`` sorts the ids once; the table's gradient (``lookup_grad``) and the
grouping (``group``, ``ungroup``) read it. A group is any id below ``rows``:
the expert a router chose, the centroid ``tac.cluster_flat`` assigned.

All tensors are torch tensors on one GPU: rows f32, bf16 or f16, ids int32,
int64 or uint32, scales and weights f32. Ids outside [0, rows), negative ones
among them, name no row. The calls enqueue on the stream given to
``ctx.set_stream``, else on torch's current stream, and return without
waiting; they may be captured into a CUDA graph. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

from . import _lib
from ._lib import CODES, MvrError

MAX_IDS = 2**31 - 1


def _refuse(msg: str, name: str = "InvalidArgument"):
    raise MvrError(CODES[name], msg)


def _torch():
    import torch

    return torch


_types: dict = {}


def _dtype(t, what: str) -> int:
    if not _types:
        torch = _torch()
        _types.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    d = _types.get(t.dtype)
    if d is None:
        _refuse(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    return d


def _is_device(t) -> bool:
    return hasattr(t, "is_cuda") and t.is_cuda


def _id_bytes(ids) -> int:
    torch = _torch()
    if ids.dtype in (torch.int32, torch.uint32):
        return 4
    if ids.dtype == torch.int64:
        return 8
    _refuse(f"ids must be int32, int64 or uint32, not {ids.dtype}")


def _rows(t, what: str, n: int | None = None, dim: int | None = None):
    """`t` as a 2-D view (copied where its rows are not consecutive) and its
    row stride."""
    if t.dim() < 2:
        _refuse(f"{what} must have rows: at least two dimensions", "DimMismatch")
    if t.dim() > 2:
        t = t.reshape(-1, t.shape[-1])
    if dim is not None and t.shape[1] != dim:
        _refuse(f"{what} has rows of {t.shape[1]}, not {dim}", "DimMismatch")
    if n is not None and t.shape[0] != n:
        _refuse(f"{what} has {t.shape[0]} rows, not {n}", "LengthMismatch")
    if t.shape[1] == 0:
        _refuse(f"{what} has rows of length 0", "DimMismatch")
    if t.stride(1) != 1 and t.shape[1] > 1 or t.stride(0) < 0:
        t = t.contiguous()
    return t, t.stride(0)


def _out_rows(t, what: str, n: int, dim: int, dtype):
    """An output given by the caller: written in place, so never copied."""
    if t.dtype != dtype:
        _refuse(f"{what} must be {dtype}, not {t.dtype}")
    if t.dim() < 2 or t.shape[-1] != dim:
        _refuse(f"{what} must have rows of {dim}", "DimMismatch")
    if t.numel() != n * dim:
        _refuse(f"{what} must have {n} rows of {dim}", "OutBufferWrongSize")
    if t.dim() > 2:
        try:
            t = t.view(n, dim)
        except RuntimeError:
            _refuse(f"{what} must be viewable as {n} rows")
    if dim > 1 and t.stride(1) != 1 or n > 1 and t.stride(0) < dim:
        _refuse(f"{what} must have consecutive, separate rows")
    return t, t.stride(0) if n > 1 else max(t.stride(0), dim)


def _f32(t, n: int, what: str):
    if t is None:
        return None
    if t.dtype != _torch().float32:
        _refuse(f"{what} must be float32, not {t.dtype}")
    if t.numel() != n:
        _refuse(f"{what} has {t.numel()} values, not {n}", "LengthMismatch")
    return t if t.is_contiguous() else t.contiguous()


class _Call:
    """One call's context and stream: tensors checked to lie on the context's
    GPU, the context switched to the stream for the calls made inside."""

    __slots__ = ("ctx", "handle", "lib", "own", "scope", "tensors")

    def __init__(self, ctx, tensors):
        dev = None
        for t in tensors:
            if t is None:
                continue
            if not _is_device(t):
                _refuse("all tensors must be CUDA tensors (there is no CPU fallback)")
            if dev is None:
                dev = t.device
            elif t.device != dev:
                _refuse(f"tensors on {dev} and {t.device}")
        if ctx is None:
            ctx = _lib.default_context(dev.index)
        elif ctx.device != dev.index:
            _refuse(f"tensors on {dev}, context on device {ctx.device}")
        self.ctx, self.handle, self.lib = ctx, ctx.handle, ctx.lib
        self.tensors = tensors
        self.own = self.scope = None

    def __enter__(self):
        ctx = self.ctx
        torch = _torch()
        ctx.lock.acquire()
        try:
            here = torch.cuda.current_stream(ctx.device).cuda_stream
            if ctx.stream == 0:
                # handle 0 would select the context's own stream: 1 names the legacy default stream
                self.own = here or 1
                self.lib.mvr_ctx_set_stream(self.handle, self.own)
            elif ctx.stream != here and not (ctx.stream == 1 and here == 0):
                # results come from the memory pool of the stream that writes
                # them, and inputs stay alive for it
                s = torch.cuda.ExternalStream(ctx.stream, device=ctx.device)
                for t in self.tensors:
                    if t is not None:
                        t.record_stream(s)
                self.scope = torch.cuda.stream(s)
                self.scope.__enter__()
        except BaseException:
            ctx.lock.release()
            raise
        return self

    def __exit__(self, *exc):
        try:
            if self.scope is not None:
                self.scope.__exit__(*exc)
            if self.own is not None:
                self.lib.mvr_ctx_set_stream(self.handle, None)
        finally:
            self.ctx.lock.release()
        return False


def _ptr(t):
    return None if t is None else t.data_ptr()


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
        torch = _torch()
        for name in ("offsets", "order", "keys", "slot"):
            t = getattr(self, name)
            if t.dtype != torch.int32 or not t.is_contiguous():
                _refuse(f"plan.{name} must be a contiguous int32 tensor")
        if self.offsets.numel() != self.rows + 1 or not self.order.numel() == self.keys.numel() == self.slot.numel():
            _refuse("plan: sizes differ", "LengthMismatch")
        return self


def plan(ids, rows: int, *, ctx=None) -> Plan:
    """Sort the ids ([n] or [n, columns]) by value, stable."""
    torch = _torch()
    rows = int(rows)
    if not 0 < rows < MAX_IDS:
        _refuse(f"rows must be in [1, 2^31 - 2], not {rows}")
    if not hasattr(ids, "dim") or ids.dim() not in (1, 2):
        _refuse("ids must be a tensor of one or two dimensions")
    if ids.dim() == 2 and ids.shape[1] == 0:
        _refuse("ids have no columns")
    idb = _id_bytes(ids)
    n = ids.numel()
    if n > MAX_IDS:
        _refuse("more than 2^31 - 1 ids")
    with _Call(ctx, (ids,)) as c:
        ids = ids.contiguous()
        dev = ids.device
        need = C.c_uint64(0)
        c.ctx.check(c.lib.mvr_token_plan_bytes(n, rows, C.byref(need)), "token_plan_bytes")
        offsets = torch.empty(rows + 1, dtype=torch.int32, device=dev)
        order = torch.empty(n, dtype=torch.int32, device=dev)
        keys = torch.empty(n, dtype=torch.int32, device=dev)
        slot = torch.empty(ids.shape, dtype=torch.int32, device=dev)
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        c.ctx.check(c.lib.mvr_token_plan_device(c.handle, ids.data_ptr(), idb, n, rows, offsets.data_ptr(),
                                                order.data_ptr(), keys.data_ptr(), slot.data_ptr(), ws.data_ptr(),
                                                need.value), "token_plan")
    return Plan(rows, offsets, order, keys, slot)


def lookup(table, ids, *, scale=None, alpha: float = 1.0, out=None, ctx=None):
    """``out[i] = (alpha * scale[i]) * table[ids[i]]``: the ids' shape plus the
    table's row length, in the table's type; zero rows where an id names none.
    ``scale`` (the ids' shape, f32) and ``out`` are optional."""
    torch = _torch()
    dt = _dtype(table, "table")
    idb = _id_bytes(ids)
    n = ids.numel()
    if table.dim() != 2:
        _refuse("table must have two dimensions", "DimMismatch")
    with _Call(ctx, (table, ids, scale, out)) as c:
        table, ts = _rows(table, "table")
        rows, dim = table.shape
        ids = ids.contiguous()
        scale = _f32(scale, n, "scale")
        if out is None:
            res = torch.empty((*ids.shape, dim), dtype=table.dtype, device=table.device)
            ptr_out, so = res.data_ptr(), dim
        else:
            res = out
            o, so = _out_rows(out, "out", n, dim, table.dtype)
            ptr_out = o.data_ptr()
        c.ctx.check(c.lib.mvr_lookup_device(c.handle, table.data_ptr(), dt, rows, dim, ts, ids.data_ptr(), idb, n,
                                            _ptr(scale), alpha, ptr_out, so), "lookup")
    return res


def lookup_grad(grad, plan: Plan, *, scale=None, alpha: float = 1.0, table=None, out=None, accumulate: bool = False,
                ctx=None):
    """Gradients of ``lookup`` from that of its output (the ids' shape plus the
    row length) and the plan of its ids: the table's, ``dtable[v] = sum alpha *
    scale[i] * grad[i]`` over the ids of v (rows without an id: zeros), and,
    where ``table`` is given, also the scale's, ``alpha * <grad[i],
    table[ids[i]]>`` as the second of a pair. ``out`` (grad's type or f32)
    receives the first; with ``accumulate`` the sums are added to it and rows
    without an id are not touched."""
    torch = _torch()
    dt = _dtype(grad, "grad")
    plan._check()
    n = plan.n_ids
    if accumulate and out is None:
        _refuse("accumulate needs out")
    with _Call(ctx, (grad, plan.offsets, plan.order, plan.keys, plan.slot, scale, table, out)) as c:
        grad, gs = _rows(grad, "grad", n)
        dim = grad.shape[1]
        scale = _f32(scale, n, "scale")
        dev = grad.device
        tp, ts, dscale = None, dim, None
        if table is not None:
            if table.dtype != grad.dtype:
                _refuse(f"table is {table.dtype}, grad {grad.dtype}")
            table, ts = _rows(table, "table", plan.rows, dim)
            tp = table.data_ptr()
            dscale = torch.empty(plan.slot.shape, dtype=torch.float32, device=dev)
        if out is None:
            res = torch.empty((plan.rows, dim), dtype=grad.dtype, device=dev)
            po, so, odt = res.data_ptr(), dim, dt
        else:
            res = out
            odt = _dtype(out, "out")
            if odt not in (dt, 0):
                _refuse("out must have grad's type or float32")
            o, so = _out_rows(out, "out", plan.rows, dim, out.dtype)
            po = o.data_ptr()
        need = C.c_uint64(0)
        c.ctx.check(c.lib.mvr_lookup_grad_bytes(n, dim, C.byref(need)), "lookup_grad_bytes")
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        c.ctx.check(c.lib.mvr_lookup_grad_device(
            c.handle, grad.data_ptr(), dt, gs, n, plan.rows, dim, plan.offsets.data_ptr(), plan.order.data_ptr(),
            plan.keys.data_ptr(), plan.slot.data_ptr(), _ptr(scale), alpha, tp, ts, po, odt, so, int(accumulate),
            _ptr(dscale), ws.data_ptr(), need.value), "lookup_grad")
    return res if table is None else (res, dscale)


def _weights(weights, plan: Plan):
    return _f32(weights, plan.n_ids, "weights")


def group(x, plan: Plan, *, weights=None, out=None, ctx=None):
    """The rows of x (one a token) in sorted order: ``out[slot[i, c]] =
    weights[i, c] * x[i]``, n * columns rows. Rows behind the last sorted one
    keep what ``out`` held (without ``out`` they are undefined)."""
    torch = _torch()
    dt = _dtype(x, "x")
    plan._check()
    with _Call(ctx, (x, plan.slot, weights, out)) as c:
        x, xst = _rows(x, "x", plan.n)
        dim = x.shape[1]
        weights = _weights(weights, plan)
        if out is None:
            out = torch.empty((plan.n_ids, dim), dtype=x.dtype, device=x.device)
        o, so = _out_rows(out, "out", plan.n_ids, dim, x.dtype)
        c.ctx.check(c.lib.mvr_group_rows_device(c.handle, x.data_ptr(), dt, xst, plan.n, plan.columns, dim,
                                                plan.slot.data_ptr(), _ptr(weights), o.data_ptr(), so), "group")
    return out


def group_grad(dout, plan: Plan, *, weights=None, x=None, out=None, ctx=None):
    """Gradients of ``group`` from that of its output: ``dx[i] = sum_c
    weights[i, c] * dout[slot[i, c]]`` and, where ``x`` is given, also that of
    the weights, ``<x[i], dout[slot[i, c]]>``, as the second of a pair."""
    torch = _torch()
    dt = _dtype(dout, "dout")
    plan._check()
    with _Call(ctx, (dout, plan.slot, weights, x, out)) as c:
        dout, ds = _rows(dout, "dout", plan.n_ids)
        dim = dout.shape[1]
        weights = _weights(weights, plan)
        dw, xp, xst = None, None, dim
        if x is not None:
            if x.dtype != dout.dtype:
                _refuse(f"x is {x.dtype}, dout {dout.dtype}")
            x, xst = _rows(x, "x", plan.n, dim)
            xp = x.data_ptr()
            dw = torch.empty(plan.slot.shape, dtype=torch.float32, device=dout.device)
        if out is None:
            out = torch.empty((plan.n, dim), dtype=dout.dtype, device=dout.device)
        o, so = _out_rows(out, "out", plan.n, dim, dout.dtype)
        c.ctx.check(c.lib.mvr_group_rows_grad_device(c.handle, dout.data_ptr(), dt, ds, plan.n, plan.columns, dim,
                                                     plan.slot.data_ptr(), _ptr(weights), xp, xst, o.data_ptr(), so,
                                                     _ptr(dw)), "group_grad")
    return out if x is None else (out, dw)


def ungroup(xs, plan: Plan, *, weights=None, out=None, ctx=None):
    """Sorted rows back to their tokens: ``out[i] = sum_c weights[i, c] *
    xs[slot[i, c]]``; zeros for a token none of whose ids names a row."""
    torch = _torch()
    dt = _dtype(xs, "xs")
    plan._check()
    with _Call(ctx, (xs, plan.slot, weights, out)) as c:
        xs, st = _rows(xs, "xs", plan.n_ids)
        dim = xs.shape[1]
        weights = _weights(weights, plan)
        if out is None:
            out = torch.empty((plan.n, dim), dtype=xs.dtype, device=xs.device)
        o, so = _out_rows(out, "out", plan.n, dim, xs.dtype)
        c.ctx.check(c.lib.mvr_ungroup_rows_device(c.handle, xs.data_ptr(), dt, st, plan.n, plan.columns, dim,
                                                  plan.slot.data_ptr(), _ptr(weights), o.data_ptr(), so), "ungroup")
    return out


def ungroup_grad(dout, plan: Plan, *, weights=None, xs=None, out=None, ctx=None):
    """Gradients of ``ungroup`` from that of its output: ``dxs[slot[i, c]] =
    weights[i, c] * dout[i]`` (rows behind the last sorted one keep what
    ``out`` held) and, where ``xs`` is given, also that of the weights,
    ``<dout[i], xs[slot[i, c]]>``, as the second of a pair."""
    torch = _torch()
    dt = _dtype(dout, "dout")
    plan._check()
    with _Call(ctx, (dout, plan.slot, weights, xs, out)) as c:
        dout, ds = _rows(dout, "dout", plan.n)
        dim = dout.shape[1]
        weights = _weights(weights, plan)
        dw, xp, xst = None, None, dim
        if xs is not None:
            if xs.dtype != dout.dtype:
                _refuse(f"xs is {xs.dtype}, dout {dout.dtype}")
            xs, xst = _rows(xs, "xs", plan.n_ids, dim)
            xp = xs.data_ptr()
            dw = torch.empty(plan.slot.shape, dtype=torch.float32, device=dout.device)
        if out is None:
            out = torch.empty((plan.n_ids, dim), dtype=dout.dtype, device=dout.device)
        o, so = _out_rows(out, "out", plan.n_ids, dim, dout.dtype)
        c.ctx.check(c.lib.mvr_ungroup_rows_grad_device(c.handle, dout.data_ptr(), dt, ds, plan.n, plan.columns, dim,
                                                       plan.slot.data_ptr(), _ptr(weights), xp, xst, o.data_ptr(), so,
                                                       _ptr(dw)), "ungroup_grad")
    return out if xs is None else (out, dw)


__all__ = ["Plan", "plan", "lookup", "lookup_grad", "group", "group_grad", "ungroup", "ungroup_grad"]
