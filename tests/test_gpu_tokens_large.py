"""Token operators at the sizes from which large batches take other launch
shapes (several accesses a thread, more places a group of lanes, wider tiles,
more passes), against the same definitions and tolerances as
test_gpu_tokens.py, whose batches stay below them.

On 148 SMs: a lookup and a group take several accesses a thread from 606,208
accesses of 32 bytes on (1,212,416 narrower ones); the table's gradient gives a
group of lanes 64, 32, 16 or 8 places, the most that leaves 1,184 blocks, and
up to 16 in one block where that takes all of them; a plan's offsets are filled
by four places a thread from 1,212,416 ids on."""
import pytest
import torch

from ir_multivector_retrieval_b200 import tokens
from ir_multivector_retrieval_b200._lib import MvrError
from test_gpu_tokens import BF16, F16, F32, TINY, U, U32, gen, lookup_grad_check, lookup_ref, make_ids, normal, plan_of, within

pytestmark = pytest.mark.gpu


# ---- plan --------------------------------------------------------------------------

@pytest.mark.parametrize("n,rows", [(606_208, 300_000), (606_209, 300_000), (1_300_003, 300_000), (2_000_003, 1000),
                                    (65_536, 40), (65_537, 3_000_000), (20_000, 3_000_000), (100_003, 3_000_000),
                                    (700_001, 3_000_000), (8000, 20_000_000), (8192, 100_000_000),
                                    (8193, 100_000_000)])
@pytest.mark.parametrize("spread,pad", [("uniform", 0.0), ("head", 0.3)])
def test_plan(n, rows, spread, pad):
    ids = make_ids(gen(n + rows), (n,), rows, torch.int64 if n % 2 else torch.int32, spread, pad)
    p = tokens.plan(ids, rows)
    offsets, order, keys, slot, valid = plan_of(ids, rows)
    assert torch.equal(p.offsets.long(), offsets)
    assert torch.equal(p.order.long(), order)
    assert torch.equal(p.keys.long(), keys)
    assert torch.equal(p.slot.long(), slot)


@pytest.mark.parametrize("n", [8000, 20_000, 70_001])
def test_plan_of_keys_of_31_bits(n):
    rows = 2**30 + 7
    ids = make_ids(gen(n), (n,), rows, torch.int64, pad=0.1)
    ids[:3] = torch.tensor([rows - 1, 2**30, 2**30 - 1], device="cuda")
    p = tokens.plan(ids, rows)
    key = torch.where((ids >= 0) & (ids < rows), ids, rows)
    keys, order = torch.sort(key, stable=True)
    assert torch.equal(p.keys.long(), keys) and torch.equal(p.order.long(), order)
    place = torch.empty_like(order)
    place[order] = torch.arange(n, device="cuda")
    assert torch.equal(p.slot.long(), torch.where(key < rows, place, -1))
    step = 2**27
    for v in range(0, rows + 1, step):
        want = torch.searchsorted(keys, torch.arange(v, min(v + step, rows + 1), device="cuda"))
        assert torch.equal(p.offsets[v:v + step].long(), want)


# ---- lookup ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,n,rows,dim", [(F32, 700_001, 32_768, 8), (F32, 250_003, 5000, 24), (F32, 250_001, 5000, 20),
                                              (F32, 410_003, 300, 6), (F32, 450_001, 300, 3), (BF16, 700_001, 900, 16),
                                              (BF16, 1_300_003, 900, 8), (F16, 250_001, 40, 10), (F16, 20_001, 40, 1000),
                                              (BF16, 410_003, 40, 3)])
@pytest.mark.parametrize("scaled", [False, True])
def test_lookup(dtype, n, rows, dim, scaled):
    g = gen(n + dim)
    table = normal(g, rows, dim, dtype=dtype)
    ids = make_ids(g, (n,), rows, torch.int64 if rows % 3 else torch.int32, pad=0.1)
    scale = torch.rand(n, generator=g, device="cuda") + 0.1 if scaled else None
    buf = torch.full((n + 1, dim), 9.0, dtype=dtype, device="cuda")
    out = tokens.lookup(table, ids, scale=scale, alpha=1.5 if scaled else 1.0, out=buf[:n])
    want = lookup_ref(table, ids, scale, 1.5 if scaled else 1.0)
    if scaled:
        within(out, want, (U[dtype] + 3 * U32) * want.abs() + TINY[dtype])
    else:
        assert torch.equal(out.double(), want)
    assert bool((buf[n] == 9).all())


# ---- the table's gradient ------------------------------------------------------------

GRADS = [(F32, 130, 9, 64), (F32, 200, 50, 64), (F32, 255, 3, 64), (F32, 256, 3, 64), (BF16, 400, 3, 64),
         (F32, 400_003, 32_768, 64), (F32, 700_001, 32_768, 64), (F32, 1_300_003, 32_768, 64), (F32, 700_001, 500, 33),
         (F32, 2_500_003, 40_000, 8), (F32, 310_003, 5000, 256), (BF16, 700_001, 900_000, 64), (BF16, 1_300_003, 70, 64),
         (BF16, 2_500_003, 32_768, 64), (F16, 1_300_003, 2000, 128), (F16, 320_003, 2000, 512)]


@pytest.mark.parametrize("dtype,n,rows,dim", GRADS)
@pytest.mark.parametrize("spread,scaled", [("uniform", False), ("head", True), ("one", True)])
def test_lookup_grad(dtype, n, rows, dim, spread, scaled):
    g = gen(n + dim)
    grad = normal(g, n, dim, dtype=dtype)
    ids = make_ids(g, (n,), rows, spread=spread, pad=0.05 if scaled else 0.0)
    scale = torch.rand(n, generator=g, device="cuda") + 0.1 if scaled else None
    p = tokens.plan(ids, rows)
    table = normal(g, rows, dim, dtype=dtype)
    dt, ds = tokens.lookup_grad(grad, p, scale=scale, alpha=0.75, table=table)
    lookup_grad_check(grad, ids, rows, scale, 0.75, dt)
    assert torch.equal(tokens.lookup_grad(grad, p, scale=scale, alpha=0.75), dt)
    base = normal(g, rows, dim)
    acc = tokens.lookup_grad(grad, p, scale=scale, alpha=0.75, out=base.clone(), accumulate=True)
    lookup_grad_check(grad, ids, rows, scale, 0.75, acc, base)
    empty = p.offsets[1:] == p.offsets[:-1]
    assert torch.equal(acc[empty], base[empty]) and bool((dt[empty] == 0).all())
    del acc, base, dt
    for a in range(0, n, 250_000):  # the products in 64 bits are several GB
        b = min(n, a + 250_000)
        prod = 0.75 * grad[a:b].double() * lookup_ref(table, ids[a:b], None, 1.0)
        within(ds[a:b], prod.sum(1), 1.001 * (dim + 2) * U32 * prod.abs().sum(1))


# ---- rows into sorted order and back ---------------------------------------------------

ROWS = [(F32, 350_003, 2, 16), (F32, 350_003, 3, 16), (F32, 350_003, 9, 16), (F32, 700_001, 1, 8), (F32, 160_003, 4, 64),
        (F32, 250_001, 2, 20), (F16, 250_001, 5, 10), (BF16, 410_003, 2, 3), (BF16, 130_003, 12, 80), (F16, 410_003, 3, 24)]


@pytest.mark.parametrize("dtype,n,columns,dim", ROWS)
@pytest.mark.parametrize("weighted", [False, True])
def test_group_and_back(dtype, n, columns, dim, weighted):
    g = gen(n + columns)
    ids = make_ids(g, (n, columns), 300, pad=0.05)
    p = tokens.plan(ids, 300)
    valid = int(p.offsets[-1])
    slot = p.slot.long()
    ok, at = slot >= 0, slot.clamp(min=0)
    x, rows = normal(g, n, dim, dtype=dtype), normal(g, n * columns, dim, dtype=dtype)
    w = torch.rand(n, columns, generator=g, device="cuda") if weighted else None
    w64 = torch.ones(n, columns, dtype=torch.float64, device="cuda") if w is None else w.double()
    want = (x.double()[:, None, :] * w64[..., None])[ok]
    tol = (U[dtype] + U32) * want.abs() + TINY[dtype]
    buf = torch.full((n * columns, dim), 9.0, dtype=dtype, device="cuda")
    within(tokens.group(x, p, weights=w, out=buf)[slot[ok]], want, tol)
    assert bool((buf[valid:] == 9).all())
    dxs, dw = tokens.ungroup_grad(x, p, weights=w, xs=rows, out=torch.full_like(buf, 9.0))
    within(dxs[slot[ok]], want, tol)
    assert bool((dxs[valid:] == 9).all())
    # without the weights' gradient: the launch of group
    assert torch.equal(tokens.ungroup_grad(x, p, weights=w, out=torch.full_like(buf, 9.0)), dxs)
    del want, tol, buf, dxs
    picked = rows.double()[at].masked_fill_(~ok[..., None], 0.0)
    prod = picked * x.double()[:, None, :]
    of, off = prod.sum(2), 1.001 * (dim + 2) * U32 * prod.abs().sum(2)
    within(dw, of, off)
    del prod
    terms = picked.mul_(w64[..., None])
    want, tol = terms.sum(1), 1.001 * (columns + 2) * U32 * terms.abs().sum(1)
    tol = tol + U[dtype] * (want.abs() + tol) + TINY[dtype]
    within(tokens.ungroup(rows, p, weights=w), want, tol)
    within(tokens.group_grad(rows, p, weights=w), want, tol)
    dx, dw = tokens.group_grad(rows, p, weights=w, x=x)
    within(dx, want, tol)
    within(dw, of, off)


def test_inputs_2_to_the_32_apart():
    stride, dim = 2**32 + 8, 24
    buf = torch.zeros(2 * stride + dim, dtype=BF16, device="cuda")
    far = buf.as_strided((3, dim), (stride, 1))
    near = normal(gen(7), 3, dim, dtype=BF16)
    far.copy_(near)
    ids = torch.tensor([2, 0, 1], device="cuda")
    p = tokens.plan(ids, 3)
    assert torch.equal(tokens.lookup(far, ids), near[ids])
    dt, ds = tokens.lookup_grad(far, p, table=far)
    wt, ws = tokens.lookup_grad(near, p, table=near)
    assert torch.equal(dt, wt) and torch.equal(ds, ws)
    assert torch.equal(tokens.group(far, p), tokens.group(near, p))
    assert torch.equal(tokens.ungroup(far, p), tokens.ungroup(near, p))
    for fn, kw in ((tokens.group_grad, "x"), (tokens.ungroup_grad, "xs")):
        for a, b in zip(fn(far, p, **{kw: far}), fn(near, p, **{kw: near})):
            assert torch.equal(a, b)
    with pytest.raises(MvrError) as e:  # an output is written in place
        tokens.lookup(near, ids, out=far)
    assert e.value.name == "InvalidArgument" and torch.equal(far, near)


# ---- shapes ----------------------------------------------------------------------------

def test_shapes_split_merged_and_transposed():
    g = gen(9)
    b, c, k, rows, dim = 6, 5, 4, 30, 48
    ids = make_ids(g, (b * c, k), rows, pad=0.1)
    p = tokens.plan(ids, rows)
    x, w = normal(g, b * c, dim), torch.rand(b * c, k, generator=g, device="cuda")
    want = tokens.ungroup(tokens.group(x, p, out=torch.zeros(b * c * k, dim, device="cuda")), p, weights=w)
    xs = tokens.group(x.view(b, c, dim), p, out=torch.zeros(b * c * k, dim, device="cuda"))
    for same in (w.view(b, c, k), w.view(-1), w.t().contiguous().t(), w.view(b * c, 1, k)):
        assert torch.equal(tokens.ungroup(xs, p, weights=same), want)
    for other in (w.t(), w.view(b, c, k).transpose(0, 2), w.view(k, b * c)):
        with pytest.raises(MvrError) as e:
            tokens.ungroup(xs, p, weights=other)
        assert e.value.name == "LengthMismatch"
    table, grad = normal(g, rows, dim), normal(g, b * c, k, dim)
    want = tokens.lookup(table, ids, scale=w)
    out = torch.zeros(b, c, k, dim, device="cuda")
    assert torch.equal(tokens.lookup(table, ids, scale=w.view(b, c, k), out=out).view_as(want), want)
    dt, ds = tokens.lookup_grad(grad.view(b, c, k, dim), p, scale=w.view(-1), table=table)
    wt, ws = tokens.lookup_grad(grad, p, scale=w, table=table)
    assert torch.equal(dt, wt) and torch.equal(ds, ws)
    for call in (lambda: tokens.lookup(table, ids, scale=w.t()),
                 lambda: tokens.lookup_grad(grad.transpose(0, 1), p), lambda: tokens.lookup_grad(grad, p, scale=w.t())):
        with pytest.raises(MvrError) as e:
            call()
        assert e.value.name == "LengthMismatch"


def test_an_output_counts_as_changed():
    g = gen(10)
    table, ids = normal(g, 9, 16), make_ids(g, (7,), 9)
    out = torch.zeros(7, 16, device="cuda")
    leaf = torch.ones(7, 16, device="cuda", requires_grad=True)
    loss = (leaf * out).sum()
    tokens.lookup(table, ids, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
