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
