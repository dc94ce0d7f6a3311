"""What is measured of the token operators: the embedding lookup with scaling
and its gradient by sorted tokens, and tokens sorted by group (expert,
centroid) and back, with weights applied, and their gradients.

``run`` computes a case in elementary torch operations, or, with ``own`` set,
through ``ir_multivector_retrieval_b200.tokens``. A case names the pass
(``op``), the tokens ``n``, the row length ``dim``, the table rows or groups
``rows``, the choices a token has (``columns``), the element type, the type of
the ids, whether rows are scaled / weighted, how the ids are spread and the
share of ids that name no row (padding, dropped choices).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ID_TYPES = {"int32": torch.int32, "int64": torch.int64}
OPS = ("lookup", "lookup_grad", "group", "group_grad", "ungroup", "ungroup_grad")
ALPHA = 8.0  # the constant scale of a lookup: sqrt(dim) at the 64-float token vectors


def _case(name, op, n, dim, rows, columns=1, dtype="f32", ids="int32", weighted=True, spread="zipf", pad=0.0):
    c = dict(op=op, n=n, dim=dim, rows=rows, columns=columns, dtype=dtype, ids=ids, weighted=weighted, spread=spread,
             pad=pad)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # the tokens of one query read their rows of the anchor table: latency
        _case("lookup query 32x64 f32", "lookup", 32, 64, 19_221, weighted=False, spread="uniform"),
        # a padded batch of sequences reads a vocabulary table, a weight a token
        _case("lookup batch 8191x1024 bf16", "lookup", 8_191, 1_024, 50_000, dtype="bf16", ids="int64", pad=0.15),
        # every token vector of a corpus from its centroid, scaled by its norm
        _case("lookup corpus 1521797x64 f32", "lookup", 1_521_797, 64, 32_768),
        # the gradient of a few short queries
        _case("lookup_grad 513x128 f16", "lookup_grad", 513, 128, 1_000, dtype="f16", pad=0.1),
        # one training step of a vocabulary table: most of its rows get none
        _case("lookup_grad 16384x1024 bf16", "lookup_grad", 16_384, 1_024, 50_000, dtype="bf16", ids="int64"),
        # centroids and norms learned over a whole corpus: very long and empty rows
        _case("lookup_grad 1521797x64 f32", "lookup_grad", 1_521_797, 64, 32_768),
        # one token in decoding, sent to 8 of 128 experts
        _case("group 1x4096 bf16 8/128", "group", 1, 4_096, 128, columns=8, dtype="bf16", weighted=False),
        # a corpus in the order of its two nearest centroids
        _case("group 1521797x64 f32 2/32768", "group", 1_521_797, 64, 32_768, columns=2, weighted=False),
        # an odd prefill batch back from its experts, some choices dropped
        _case("ungroup 4093x2048 f16 8/64", "ungroup", 4_093, 2_048, 64, columns=8, dtype="f16", pad=0.03),
        # a few decoding tokens back from their experts
        _case("ungroup 7x4096 bf16 4/32", "ungroup", 7, 4_096, 32, columns=4, dtype="bf16"),
        # a training step: through the routing and through the weighted sum
        _case("group_grad 8192x1024 bf16 4/64", "group_grad", 8_192, 1_024, 64, columns=4, dtype="bf16"),
        _case("ungroup_grad 8192x2048 bf16 8/128", "ungroup_grad", 8_192, 2_048, 128, columns=8, dtype="bf16",
              pad=0.02),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(OPS)
    look = op.startswith("lookup")
    dtype = rng.choice(("f32", "bf16", "f16"))
    dim = rng.choice((64, 128, 256, 1_024)) if rng.random() < 0.5 else _log(rng, 4, 4_096)
    rows = _log(rng, 2, 65_536)
    columns = 1 if look else rng.choice((1, 2, 4, 6, 8))
    # pairs x dim stays below the corpus cases' 1,521,797 x 64
    n = _log(rng, 1, max(2, min(1_500_000, 90_000_000 // (dim * columns))))
    while look and rows * dim > 50_000_000:
        rows = (rows + 1) // 2
    weighted = rng.random() < 0.7 if op in ("lookup", "lookup_grad", "group") else True
    return _case(None, op, n, dim, rows, columns, dtype, rng.choice(("int32", "int64")), weighted,
                 rng.choice(("zipf", "uniform")), rng.choice((0.0, 0.0, 0.05, 0.3)))


def _normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _make_ids(case, g):
    n, c, rows = case["n"], case["columns"], case["rows"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    if case["spread"] == "zipf":
        w = 1.0 / torch.arange(1, rows + 1, device="cuda", dtype=torch.float64) ** 1.1
        first = torch.searchsorted(torch.cumsum(w / w.sum(), 0), u, right=True).clamp_(max=rows - 1)
        # the popular rows lie anywhere in the table
        first = torch.randperm(rows, generator=g, device="cuda")[first]
    else:
        first = (u * rows).long().clamp_(max=rows - 1)
    step = torch.randint(1, max(2, rows // c), (n,), generator=g, device="cuda")
    ids = (first[:, None] + step[:, None] * torch.arange(c, device="cuda")) % rows
    if case["pad"]:
        ids[torch.rand(n, c, generator=g, device="cuda") < case["pad"]] = -1
    return ids.to(ID_TYPES[case["ids"]])


def _sorted_plan(ids, rows):
    """The arrays of a plan: valid pairs in stable order of their ids."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < rows), flat, rows)
    keys, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(keys, torch.arange(rows + 1, device=keys.device))
    slot = torch.empty_like(order)
    slot[order] = torch.arange(order.numel(), device=order.device)
    slot = torch.where(key < rows, slot, -1)
    return dict(offsets=offsets.int(), order=order.int(), keys=keys.int(), slot=slot.int().view(ids.shape))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    n, dim, rows, c, t = case["n"], case["dim"], case["rows"], case["columns"], TYPES[case["dtype"]]
    s = dict(case=case, ids=_make_ids(case, g))
    op = case["op"]
    if op.startswith("lookup"):
        s["ids"] = s["ids"].view(-1)
        s["table"] = _normal(g, rows, dim, dtype=t, std=1 / math.sqrt(dim))
        s["scale"] = torch.rand(n, generator=g, device="cuda") + 0.25 if case["weighted"] else None
        if op == "lookup_grad":
            s["grad"] = _normal(g, n, dim, dtype=t)
        return s
    s["weights"] = torch.rand(n, c, generator=g, device="cuda") if case["weighted"] else None
    if op == "group":
        s["x"] = _normal(g, n, dim, dtype=t)
        s["xs"] = torch.zeros(n * c, dim, dtype=t, device="cuda")  # the program's buffer for the sorted rows
        return s
    s["plan"] = _sorted_plan(s["ids"], rows)
    if op == "group_grad":
        s["x"] = _normal(g, n, dim, dtype=t)
        s["dxs"] = _normal(g, n * c, dim, dtype=t)
    elif op == "ungroup":
        s["xs"] = _normal(g, n * c, dim, dtype=t)
    else:
        s["dy"] = _normal(g, n, dim, dtype=t)
        s["xs"] = _normal(g, n * c, dim, dtype=t)
        s["dxs"] = torch.zeros(n * c, dim, dtype=t, device="cuda")
    return s


def _run_own(s):
    from ir_multivector_retrieval_b200 import tokens

    case = s["case"]
    op, rows = case["op"], case["rows"]
    if op == "lookup":
        return tokens.lookup(s["table"], s["ids"], scale=s["scale"], alpha=ALPHA)
    if op == "lookup_grad":
        p = tokens.plan(s["ids"], rows)
        if s["scale"] is None:
            return tokens.lookup_grad(s["grad"], p, alpha=ALPHA)
        return tokens.lookup_grad(s["grad"], p, scale=s["scale"], alpha=ALPHA, table=s["table"])
    if op == "group":
        p = tokens.plan(s["ids"], rows)
        return tokens.group(s["x"], p, weights=s["weights"], out=s["xs"]), p.offsets, p.slot
    p = tokens.Plan(rows=rows, **s["plan"])
    if op == "group_grad":
        return tokens.group_grad(s["dxs"], p, weights=s["weights"], x=s["x"])
    if op == "ungroup":
        return tokens.ungroup(s["xs"], p, weights=s["weights"])
    return tokens.ungroup_grad(s["dy"], p, weights=s["weights"], xs=s["xs"], out=s["dxs"])


def _rows_of(xs, slot):
    """xs[slot] in 32 bits, zero rows where there is none."""
    r = xs.float()[slot.long().clamp(min=0)]
    return r.masked_fill_((slot < 0)[..., None], 0.0)


def _spread_rows(rows, slot, p, dtype):
    """The rows [n, c, dim] at their sorted places, zero rows behind the last."""
    out = torch.zeros(p + 1, rows.shape[-1], dtype=torch.float32, device=rows.device)
    at = slot.reshape(-1).long()
    out[torch.where(at < 0, p, at)] = rows.reshape(-1, rows.shape[-1])
    return out[:p].to(dtype)


def run(state):
    if own:
        return _run_own(state)
    s, case = state, state["case"]
    op, rows, t = case["op"], case["rows"], TYPES[case["dtype"]]
    if op.startswith("lookup"):
        ids = s["ids"].long()
        valid = (ids >= 0) & (ids < rows)
        at = torch.where(valid, ids, 0)
        scale = torch.full((case["n"],), ALPHA, device="cuda") if s["scale"] is None else ALPHA * s["scale"]
        if op == "lookup":
            r = s["table"].float()[at] * scale[:, None]
            return r.masked_fill_(~valid[:, None], 0.0).to(t)
        # up to a seventh of all tokens share one row: the sums are long
        g = s["grad"].double().mul_((scale * valid).double()[:, None])
        dt = torch.zeros(rows, case["dim"], dtype=torch.float64, device="cuda").index_add_(0, at, g)
        if s["scale"] is None:
            return dt.to(t)
        del g
        ds = (s["grad"].float() * s["table"].float()[at]).sum(1) * ALPHA
        return dt.to(t), ds.masked_fill_(~valid, 0.0)
    if op == "group":
        p = _sorted_plan(s["ids"], rows)
        x = s["x"].float()[:, None, :]
        x = x.expand(-1, case["columns"], -1) if s["weights"] is None else x * s["weights"][..., None]
        return _spread_rows(x, p["slot"], s["ids"].numel(), t), p["offsets"], p["slot"]
    slot, w = s["plan"]["slot"], s["weights"]
    if op == "ungroup":
        return (_rows_of(s["xs"], slot) * w[..., None]).sum(1).to(t)
    if op == "group_grad":
        r = _rows_of(s["dxs"], slot)
        return (r * w[..., None]).sum(1).to(t), (r * s["x"].float()[:, None, :]).sum(2)
    dy = s["dy"].float()[:, None, :]
    dw = (_rows_of(s["xs"], slot) * dy).sum(2)
    return _spread_rows(dy * w[..., None], slot, slot.numel(), t), dw


def work(case):
    n, dim, rows, c = case["n"], case["dim"], case["rows"], case["columns"]
    e = 4 if case["dtype"] == "f32" else 2
    idb = 8 if case["ids"] == "int64" else 4
    op, pairs = case["op"], n * c
    valid = int(pairs * (1 - case["pad"]))
    table = min(valid, rows) * dim * e
    w4 = 4 * pairs if case["weighted"] else 0
    if op == "lookup":
        return {"bytes": n * idb + w4 + table + n * dim * e, "flops": valid * dim}
    if op == "lookup_grad":
        more = table + 8 * n if case["weighted"] else 0
        return {"bytes": n * idb + valid * dim * e + rows * dim * e + more,
                "flops": valid * dim * (4 if case["weighted"] else 2)}
    if op == "group":
        return {"bytes": pairs * idb + w4 + n * dim * e + valid * dim * e + 4 * pairs + 4 * (rows + 1),
                "flops": valid * dim}
    if op == "ungroup":
        return {"bytes": 4 * pairs + w4 + valid * dim * e + n * dim * e, "flops": 2 * valid * dim}
    if op == "group_grad":
        return {"bytes": 4 * pairs + w4 + valid * dim * e + 2 * n * dim * e + 4 * pairs, "flops": 4 * valid * dim}
    return {"bytes": 4 * pairs + w4 + n * dim * e + 2 * valid * dim * e + 4 * pairs, "flops": 3 * valid * dim}


def exact(case, seed):
    """The outputs from the definitions, in 64 bits, on the host."""
    s = prepare(case, seed)

    def host(name):
        v = s.get(name)
        return None if v is None else v.double().cpu().numpy()

    n, dim, rows, c, op = case["n"], case["dim"], case["rows"], case["columns"], case["op"]
    ids = s["ids"].long().cpu().numpy().reshape(-1)
    named = np.flatnonzero((ids >= 0) & (ids < rows))  # the pairs that take part
    if op.startswith("lookup"):
        table, scale = host("table"), host("scale")
        factor = np.full(n, ALPHA) if scale is None else ALPHA * scale
        if op == "lookup":
            out = np.zeros((n, dim))
            out[named] = factor[named, None] * table[ids[named]]
            return out
        grad, dt = host("grad"), np.zeros((rows, dim))
        by = named[np.argsort(ids[named], kind="stable")]
        if by.size:
            starts = np.flatnonzero(np.r_[True, ids[by][1:] != ids[by][:-1]])
            dt[ids[by][starts]] = np.add.reduceat(grad[by] * factor[by, None], starts, axis=0)
        if scale is None:
            return dt
        ds = np.zeros(n)
        ds[named] = ALPHA * np.einsum("ij,ij->i", grad[named], table[ids[named]])
        return dt, ds
    place = np.full(n * c, -1)
    place[named[np.argsort(ids[named], kind="stable")]] = np.arange(named.size)
    at, token = place[named], named // c
    w = np.ones(n * c) if s["weights"] is None else host("weights").reshape(-1)
    if op in ("group", "ungroup_grad"):
        out = np.zeros((n * c, dim))
        src = host("x" if op == "group" else "dy")
        out[at] = w[named, None] * src[token]
        if op == "group":
            return out, None, None
        dw = np.zeros(n * c)
        dw[named] = np.einsum("ij,ij->i", host("xs")[at], src[token])
        return out, dw.reshape(n, c)
    src, y = host("xs" if op == "ungroup" else "dxs"), np.zeros((n, dim))
    if named.size:
        starts = np.flatnonzero(np.r_[True, token[1:] != token[:-1]])
        y[token[starts]] = np.add.reduceat(w[named, None] * src[at], starts, axis=0)
    if op == "ungroup":
        return y
    dw = np.zeros(n * c)
    dw[named] = np.einsum("ij,ij->i", host("x")[token], src[at])
    return y, dw.reshape(n, c)

