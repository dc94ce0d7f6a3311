"""Token operators on the GPU against their definitions in 64 bits.

Tolerances count roundings: U[t] is half a step of the element type relative
to the value; a sum of m products in f32, whatever its order, is off by at
most (m + 2) half steps of f32 relative to the sum of the products' sizes;
below the normal range of f16 half a step is 2^-25."""
import ctypes as C

import pytest
import torch

from ir_multivector_retrieval_b200 import Context, tokens
from ir_multivector_retrieval_b200._lib import CODES, MvrError

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
U = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {F32: 2.0**-149, BF16: 2.0**-133, F16: 2.0**-25}
U32 = 2.0**-24


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def make_ids(g, shape, rows, dtype=torch.int32, spread="uniform", pad=0.0):
    u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
    if spread == "one":  # all ids the same
        ids = torch.full(shape, rows - 1, device="cuda", dtype=torch.int64)
    elif spread == "head":  # most ids on a few values, some anywhere
        ids = (u**8 * rows).long()
    else:
        ids = (u * rows).long()
    ids.clamp_(max=rows - 1)
    if pad:
        drop = torch.rand(shape, generator=g, device="cuda") < pad
        # negative and too large ids name no row alike
        ids = torch.where(drop, torch.where(u < 0.5, -1, rows), ids)
    return ids.to(dtype)


def plan_of(ids, rows):
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < rows), flat, rows)
    keys, order = torch.sort(key, stable=True)
    valid = int((key < rows).sum())
    slot = torch.empty_like(order)
    slot[order] = torch.arange(order.numel(), device="cuda")
    slot[key >= rows] = -1
    offsets = torch.searchsorted(keys, torch.arange(rows + 1, device="cuda"))
    return offsets, order, keys, slot.view(ids.shape), valid


def within(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {(got.double() - want).abs().max().item():.3g}"


# ---- plan --------------------------------------------------------------------

@pytest.mark.parametrize("n,rows", [(1, 1), (1, 100_000), (2, 3), (31, 2), (32, 256), (33, 255), (257, 257),
                                    (1000, 1), (1024, 1023), (2047, 40_000), (2048, 65_535), (4096, 128),
                                    (4097, 65_536), (10_000, 70_000), (65_537, 8), (300_001, 262_144),
                                    (1_000_003, 1000), (16, 20_000_000)])
@pytest.mark.parametrize("spread,pad", [("uniform", 0.0), ("head", 0.3)])
def test_plan_is_the_stable_sort(n, rows, spread, pad):
    ids = make_ids(gen(n + rows), (n,), rows, torch.int64 if n % 2 else torch.int32, spread, pad)
    p = tokens.plan(ids, rows)
    offsets, order, keys, slot, valid = plan_of(ids, rows)
    assert torch.equal(p.offsets.long(), offsets)
    assert torch.equal(p.order[:valid].long(), order[:valid])
    assert torch.equal(p.keys.long(), keys)
    assert torch.equal(p.slot.long(), slot)


@pytest.mark.parametrize("n", [1, 5000, 50_000])
def test_plan_of_ids_that_name_nothing(n):
    ids = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    ids[::2] = 2**40 + 3  # its low half would name row 3
    p = tokens.plan(ids, 9)
    assert int(p.offsets.abs().sum()) == 0 and bool((p.slot == -1).all()) and bool((p.keys == 9).all())


def test_plan_of_no_ids():
    p = tokens.plan(torch.empty(0, dtype=torch.int32, device="cuda"), 1000)
    assert p.offsets.shape == (1001,) and int(p.offsets.abs().sum()) == 0 and p.slot.numel() == 0


def test_plan_of_columns_and_id_types():
    ids = make_ids(gen(3), (333, 5), 40, torch.int64, pad=0.1)
    want = tokens.plan(ids, 40)
    assert want.slot.shape == (333, 5) and (want.n, want.columns) == (333, 5)
    valid = int(want.offsets[-1])
    for other in (ids.int(), ids.to(torch.uint32), ids.t().contiguous().t()):
        p = tokens.plan(other, 40)
        assert torch.equal(p.slot, want.slot) and torch.equal(p.offsets, want.offsets)
        assert torch.equal(p.order[:valid], want.order[:valid]) and torch.equal(p.keys, want.keys)


# ---- lookup --------------------------------------------------------------------

def lookup_ref(table, ids, scale, alpha):
    rows = table.shape[0]
    i = ids.long()
    ok = (i >= 0) & (i < rows)
    f = torch.full(i.shape, alpha, dtype=torch.float64, device="cuda")
    f = f if scale is None else f * scale.double()
    return torch.where(ok[..., None], table.double()[torch.where(ok, i, 0)] * f[..., None], 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (1, 7, 4096), (3, 5, 3), (32, 100, 64), (33, 1000, 100),
                                        (257, 3, 20), (1000, 513, 128), (777, 50, 257), (130, 40, 1030),
                                        (5000, 90, 6), (20_001, 300, 8), (64, 3, 8200)])
@pytest.mark.parametrize("scaled", [False, True])
def test_lookup(dtype, n, rows, dim, scaled):
    g = gen(n + dim)
    table = normal(g, rows, dim, dtype=dtype)
    ids = make_ids(g, (n,), rows, torch.int64 if dim % 2 else torch.int32, pad=0.2 if n > 3 else 0.0)
    scale = torch.rand(n, generator=g, device="cuda") + 0.1 if scaled else None
    out = tokens.lookup(table, ids, scale=scale, alpha=1.7 if scaled else 1.0)
    assert out.shape == (n, dim) and out.dtype == dtype
    want = lookup_ref(table, ids, scale, float(torch.tensor(1.7)) if scaled else 1.0)
    if scaled:
        within(out, want, (U[dtype] + 3 * U32) * want.abs() + TINY[dtype])
    else:
        assert torch.equal(out.double(), want)  # a copy


def test_lookup_shapes_strides_and_alignments():
    g = gen(5)
    wide = normal(g, 50, 200, dtype=BF16)
    ids = make_ids(g, (6, 7), 50, torch.int64)
    want = tokens.lookup(wide, ids)
    assert want.shape == (6, 7, 200)
    for a, b in ((0, 64), (1, 65), (2, 66), (3, 11), (4, 60), (8, 136), (199, 200)):
        view = wide[:, a:b]
        assert torch.equal(tokens.lookup(view, ids), want[..., a:b])
        # into the columns of a wider buffer; what lies beside them stays
        buf = torch.full((42, 230), 9.0, dtype=BF16, device="cuda")
        out = buf[:, 5:5 + b - a]
        assert tokens.lookup(view, ids, out=out) is out
        assert torch.equal(out, want[..., a:b].reshape(42, -1))
        assert bool((buf[:, :5] == 9).all()) and bool((buf[:, 5 + b - a:] == 9).all())
    assert torch.equal(tokens.lookup(wide.t().contiguous().t(), ids), want)
    assert torch.equal(tokens.lookup(wide[::2], ids // 2), wide[::2][ids // 2])
    assert torch.equal(tokens.lookup(wide[:1].expand(50, 200), ids), wide[0].expand(6, 7, 200))
    assert tokens.lookup(wide, torch.empty(0, 3, dtype=torch.int32, device="cuda")).shape == (0, 3, 200)


def test_lookup_keeps_infinities_and_ignores_other_rows():
    table = torch.tensor([[1.0, float("inf")], [float("nan"), -0.0], [float("nan"), float("inf")]], device="cuda")
    out = tokens.lookup(table, torch.tensor([0, -1, 3, 1], device="cuda"))
    assert out[0].tolist() == [1.0, float("inf")] and out[1:3].abs().sum() == 0
    assert torch.isnan(out[3, 0]) and torch.signbit(out[3, 1])


# ---- lookup gradients ----------------------------------------------------------

def lookup_grad_check(grad, ids, rows, scale, alpha, dt, base=None):
    """dt against the definition; `base` what it was added to."""
    n, dim = grad.shape
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < rows)
    f = torch.full((n,), alpha, dtype=torch.float64, device="cuda")
    f = f if scale is None else f * scale.reshape(-1).double()
    terms = grad.double()[ok] * f[ok, None]
    want = torch.zeros(rows, dim, dtype=torch.float64, device="cuda").index_add_(0, flat[ok], terms)
    size = torch.zeros_like(want).index_add_(0, flat[ok], terms.abs())
    m = torch.bincount(flat[ok], minlength=rows).double()[:, None]
    tol = (m + 2) * U32 * size
    if base is not None:
        want = want + base.double()
        tol = tol + U32 * want.abs()
    within(dt, want, 1.001 * tol + U[dt.dtype] * (want.abs() + tol) + TINY[dt.dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,dim,spread", [
    (1, 1, 1, "uniform"), (1, 5, 300, "uniform"), (5, 4, 3, "uniform"), (32, 19, 64, "uniform"),
    (63, 2, 64, "head"), (64, 2, 64, "one"), (65, 1, 64, "one"), (513, 100, 100, "uniform"),
    (1000, 10_000, 128, "uniform"), (2048, 7, 20, "head"), (4000, 3, 64, "one"), (4096, 4, 128, "one"),
    (9001, 5, 257, "head"), (30_000, 1000, 64, "head"), (100_003, 2, 8, "one"), (777, 30, 1030, "head"),
    (50_000, 49, 6, "uniform"), (300, 3, 4100, "head"), (2000, 40, 512, "head"), (3000, 40, 1024, "head"),
    (20_000, 60_000, 16, "uniform"), (120_000, 300, 33, "head")])
@pytest.mark.parametrize("scaled", [False, True])
def test_lookup_grad(dtype, n, rows, dim, spread, scaled):
    g = gen(n + dim)
    grad = normal(g, n, dim, dtype=dtype)
    ids = make_ids(g, (n,), rows, spread=spread, pad=0.1 if scaled and n > 5 else 0.0)
    scale = torch.rand(n, generator=g, device="cuda") + 0.1 if scaled else None
    alpha = 0.75
    p = tokens.plan(ids, rows)
    table = normal(g, rows, dim, dtype=dtype)
    dt, ds = tokens.lookup_grad(grad, p, scale=scale, alpha=alpha, table=table)
    lookup_grad_check(grad, ids, rows, scale, alpha, dt)
    prod = alpha * grad.double() * lookup_ref(table, ids, None, 1.0)
    within(ds, prod.sum(1), 1.001 * (dim + 2) * U32 * prod.abs().sum(1))
    assert torch.equal(tokens.lookup_grad(grad, p, scale=scale, alpha=alpha), dt)
    # added to a table in 32 bits: rows without a token keep what they held
    base = normal(g, rows, dim)
    acc = base.clone()
    assert tokens.lookup_grad(grad, p, scale=scale, alpha=alpha, out=acc, accumulate=True) is acc
    lookup_grad_check(grad, ids, rows, scale, alpha, acc, base)
    empty = p.offsets[1:] == p.offsets[:-1]
    assert torch.equal(acc[empty], base[empty])
    assert bool((dt[empty] == 0).all())


@pytest.mark.parametrize("n,rows,dim", [(70_000, 40, 128), (300_000, 5000, 64), (262_145, 100_000, 32), (9000, 70_000, 512)])
def test_lookup_grad_of_many_tokens_with_64_bit_ids(n, rows, dim):
    g = gen(n)
    ids = make_ids(g, (n,), rows, torch.int64, "head", pad=0.02)
    p = tokens.plan(ids, rows)
    offsets, order, keys, slot, valid = plan_of(ids, rows)
    assert torch.equal(p.offsets.long(), offsets) and torch.equal(p.slot.long(), slot)
    assert torch.equal(p.order.long(), order) and torch.equal(p.keys.long(), keys)  # those that name no row last
    grad, table = normal(g, n, dim, dtype=BF16), normal(g, rows, dim, dtype=BF16)
    dt, ds = tokens.lookup_grad(grad, p, alpha=0.5, table=table, out=torch.empty(rows, dim, device="cuda"))
    lookup_grad_check(grad, ids, rows, None, 0.5, dt)
    prod = 0.5 * grad.double() * lookup_ref(table, ids, None, 1.0)
    within(ds, prod.sum(1), 1.001 * (dim + 2) * U32 * prod.abs().sum(1))


def test_lookup_grad_of_nothing():
    g = gen(1)
    for ids in (torch.empty(0, dtype=torch.int32, device="cuda"), torch.full((70,), -1, device="cuda")):
        p = tokens.plan(ids, 33)
        grad = torch.full((ids.numel(), 12), float("nan"), device="cuda")
        dt, ds = tokens.lookup_grad(grad, p, table=normal(g, 33, 12))
        assert bool((dt == 0).all()) and bool((ds == 0).all())
        base = normal(g, 33, 12)
        assert torch.equal(tokens.lookup_grad(grad, p, out=base.clone(), accumulate=True), base)


def test_lookup_grad_of_padding_reads_no_gradient():
    g = gen(2)
    ids = make_ids(g, (400,), 20)
    ids[100:200] = -100
    grad = normal(g, 400, 64)
    clean = grad.clone()
    clean[100:200] = 0
    grad[100:200] = float("nan")
    scale = torch.rand(400, generator=g, device="cuda")
    p = tokens.plan(ids, 20)
    table = normal(g, 20, 64)
    dt, ds = tokens.lookup_grad(grad, p, scale=scale.masked_fill(ids < 0, float("inf")), table=table)
    wt, ws = tokens.lookup_grad(clean, p, scale=scale, table=table)
    assert torch.equal(dt, wt) and torch.equal(ds, ws) and bool((ds[100:200] == 0).all())


@pytest.mark.parametrize("dim", [16, 64, 700])
def test_padding_has_no_gradient_whatever_the_constant(dim):
    g = gen(dim)
    ids = make_ids(g, (60,), 7)
    ids[::3] = -1
    p = tokens.plan(ids, 7)
    dt, ds = tokens.lookup_grad(normal(g, 60, dim), p, alpha=float("inf"), table=normal(g, 7, dim))
    assert bool((ds[::3] == 0).all()) and not torch.isfinite(ds[ids >= 0]).any()
    out = tokens.lookup(normal(g, 7, dim), ids, alpha=float("inf"))
    assert bool((out[::3] == 0).all())


def test_one_row_has_any_stride():
    x = torch.arange(8.0, device="cuda")
    row = x.as_strided((1, 8), (2**40, 1))
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = tokens.plan(zero, 1)
    out = torch.zeros(8, device="cuda").as_strided((1, 8), (2**40, 1))
    for r in (tokens.lookup(row, zero, out=out), tokens.lookup_grad(row, p), tokens.group(row, p), tokens.ungroup(row, p)):
        assert torch.equal(r.view(-1), x)


def test_lookup_grad_strides_and_alignments():
    g = gen(4)
    ids = make_ids(g, (3, 300), 40, spread="head")
    p = tokens.plan(ids, 40)
    wide = normal(g, 3, 300, 200, dtype=F16)
    wt = normal(g, 40, 200, dtype=F16)
    for a, b in ((0, 64), (1, 65), (2, 66), (3, 11), (8, 136), (0, 200)):
        dt, ds = tokens.lookup_grad(wide[..., a:b], p, table=wt[:, a:b])
        assert ds.shape == ids.shape
        lookup_grad_check(wide[..., a:b].reshape(900, -1), ids, 40, None, 1.0, dt)
        buf = torch.full((40, 230), 9.0, dtype=F16, device="cuda")
        tokens.lookup_grad(wide[..., a:b], p, out=buf[:, 7:7 + b - a])
        # another alignment may add in another order: held to the definition
        lookup_grad_check(wide[..., a:b].reshape(900, -1), ids, 40, None, 1.0, buf[:, 7:7 + b - a])
        assert bool((buf[:, :7] == 9).all()) and bool((buf[:, 7 + b - a:] == 9).all())
        wide_out = torch.full((40, 230), 9.0, device="cuda")  # in 32 bits, at odd places
        tokens.lookup_grad(wide[..., a:b], p, out=wide_out[:, 3:3 + b - a])
        lookup_grad_check(wide[..., a:b].reshape(900, -1), ids, 40, None, 1.0, wide_out[:, 3:3 + b - a])
        assert bool((wide_out[:, :3] == 9).all()) and bool((wide_out[:, 3 + b - a:] == 9).all())
        base = normal(g, 40, b - a, dtype=F16)  # added to, in 16 bits
        acc = base.clone()
        tokens.lookup_grad(wide[..., a:b], p, out=acc, accumulate=True)
        lookup_grad_check(wide[..., a:b].reshape(900, -1), ids, 40, None, 1.0, acc, base)
    one = normal(g, 1, 64)
    dt = tokens.lookup_grad(one.expand(900, 64), p)  # a broadcast gradient
    lookup_grad_check(one.expand(900, 64), ids, 40, None, 1.0, dt)


def test_lookup_gradients_against_differences():
    # the lookup is linear in the table and in the scale: a difference of the
    # forward pass along a direction is the gradient's product with it
    g = gen(8)
    n, rows, dim = 700, 50, 64
    table, d_table = normal(g, rows, dim), normal(g, rows, dim)
    ids = make_ids(g, (n,), rows, pad=0.1, spread="head")
    scale, d_scale = torch.rand(n, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
    cot = normal(g, n, dim)
    dt, ds = tokens.lookup_grad(cot, tokens.plan(ids, rows), scale=scale, alpha=2.0, table=table)

    def loss(t, s):
        return (tokens.lookup(t, ids, scale=s, alpha=2.0).double() * cot.double())

    for moved, grad, step in (((table + d_table, scale), dt, d_table), ((table, scale + d_scale), ds, d_scale)):
        hi, lo = loss(*moved), loss(table, scale)
        # each output, and the moved input, is within 4 half steps; the gradient's sums within 2 + n terms'
        tol = 8 * U32 * (hi.abs().sum() + lo.abs().sum()) * 2 + (n + 2) * U32 * (grad.double() * step.double()).abs().sum() * 8
        assert abs((hi.sum() - lo.sum() - (grad.double() * step.double()).sum()).item()) <= tol.item()


# ---- rows into sorted order and back ---------------------------------------------

SHAPES = [(1, 1, 1, 1), (1, 8, 4096, 128), (2, 3, 5, 4), (7, 4, 1024, 32), (64, 2, 64, 9), (333, 1, 100, 17),
          (500, 6, 257, 64), (1025, 3, 20, 2000), (200, 16, 128, 40), (3000, 2, 64, 700), (50, 5, 2056, 6),
          (40, 8, 8200, 12), (6000, 8, 6, 5), (9, 33, 64, 50)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,columns,dim,rows", SHAPES)
@pytest.mark.parametrize("weighted", [False, True])
def test_group_and_its_gradient(dtype, n, columns, dim, rows, weighted):
    g = gen(n + dim)
    ids = make_ids(g, (n, columns), rows, pad=0.15)
    p = tokens.plan(ids, rows)
    valid = int(p.offsets[-1])
    x = normal(g, n, dim, dtype=dtype)
    w = torch.rand(n, columns, generator=g, device="cuda") if weighted else None
    w64 = torch.ones(n, columns, dtype=torch.float64, device="cuda") if w is None else w.double()
    out = torch.full((n * columns, dim), 7.0, dtype=dtype, device="cuda")
    assert tokens.group(x, p, weights=w, out=out) is out
    slot = p.slot.long()
    ok = slot >= 0
    pairs = x.double()[:, None, :] * w64[..., None]
    want = pairs[ok]
    got = out[slot[ok]]
    within(got, want, (U[dtype] + U32) * want.abs() + TINY[dtype])
    assert bool((out[valid:] == 7).all())

    dout = normal(g, n * columns, dim, dtype=dtype)
    dout[valid:] = float("nan")  # not read
    dx, dw = tokens.group_grad(dout, p, weights=w, x=x)
    rows64 = dout.double()[slot.clamp(min=0)].masked_fill(~ok[..., None], 0.0)
    terms = rows64 * w64[..., None]
    want, size = terms.sum(1), terms.abs().sum(1)
    tol = 1.001 * (columns + 2) * U32 * size
    within(dx, want, tol + U[dtype] * (want.abs() + tol) + TINY[dtype])
    prod = rows64 * x.double()[:, None, :]
    within(dw, prod.sum(2), 1.001 * (dim + 2) * U32 * prod.abs().sum(2))
    assert torch.equal(tokens.group_grad(dout, p, weights=w), dx)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,columns,dim,rows", SHAPES)
@pytest.mark.parametrize("weighted", [False, True])
def test_ungroup_and_its_gradient(dtype, n, columns, dim, rows, weighted):
    g = gen(n + dim + 1)
    ids = make_ids(g, (n, columns), rows, torch.int64, "head", pad=0.15)
    p = tokens.plan(ids, rows)
    valid = int(p.offsets[-1])
    slot = p.slot.long()
    ok = slot >= 0
    xs = normal(g, n * columns, dim, dtype=dtype)
    xs[valid:] = float("nan")  # not read
    w = torch.rand(n, columns, generator=g, device="cuda").masked_fill(~ok, float("nan")) if weighted else None
    w64 = torch.ones(n, columns, dtype=torch.float64, device="cuda") if w is None else w.double()
    rows64 = xs.double()[slot.clamp(min=0)].masked_fill(~ok[..., None], 0.0)
    terms = (rows64 * w64[..., None]).masked_fill(~ok[..., None], 0.0)
    want, size = terms.sum(1), terms.abs().sum(1)
    tol = 1.001 * (columns + 2) * U32 * size
    out = tokens.ungroup(xs, p, weights=w)
    within(out, want, tol + U[dtype] * (want.abs() + tol) + TINY[dtype])
    none = ~ok.any(1)
    assert bool((out[none] == 0).all())

    dy = normal(g, n, dim, dtype=dtype)
    dxs = torch.full((n * columns, dim), 7.0, dtype=dtype, device="cuda")
    got, dw = tokens.ungroup_grad(dy, p, weights=w, xs=xs, out=dxs)
    assert got is dxs and bool((dxs[valid:] == 7).all())
    want = (dy.double()[:, None, :] * w64[..., None])[ok]
    within(dxs[slot[ok]], want, (U[dtype] + U32) * want.abs() + TINY[dtype])
    prod = rows64 * dy.double()[:, None, :]
    within(dw, prod.sum(2), 1.001 * (dim + 2) * U32 * prod.abs().sum(2))
    assert bool((dw[~ok] == 0).all())
    assert torch.equal(tokens.ungroup_grad(dy, p, weights=w, out=dxs.clone()), dxs)


def test_group_strides_and_alignments():
    g = gen(11)
    ids = make_ids(g, (90, 3), 13, pad=0.1)
    p = tokens.plan(ids, 13)
    valid = int(p.offsets[-1])
    wide = normal(g, 90, 200, dtype=BF16)
    wxs = normal(g, 270, 200, dtype=BF16)
    w = torch.rand(3, 90, generator=g, device="cuda").t()  # not contiguous
    for a, b in ((0, 64), (1, 65), (2, 66), (3, 11), (4, 60), (8, 136), (0, 200)):
        buf = torch.full((270, 230), 9.0, dtype=BF16, device="cuda")
        out = tokens.group(wide[:, a:b], p, weights=w, out=buf[:, 5:5 + b - a])
        ref = tokens.group(wide[:, a:b].contiguous(), p, weights=w.contiguous())
        assert torch.equal(out[:valid], ref[:valid])
        assert bool((buf[:, :5] == 9).all()) and bool((buf[:, 5 + b - a:] == 9).all())
        assert bool((buf[valid:] == 9).all())
        back = tokens.ungroup(wxs[:, a:b], p, weights=w)
        assert torch.equal(back, tokens.ungroup(wxs[:, a:b].contiguous(), p, weights=w))
        for fn, d, other in ((tokens.group_grad, wxs, wide), (tokens.ungroup_grad, wide, wxs)):
            kw = "x" if fn is tokens.group_grad else "xs"
            r, dw = fn(d[:, a:b], p, weights=w, **{kw: other[:, a:b]})
            want = (d.double()[:, a:b], other.double()[:, a:b])
            tok, srt = (want[1], want[0]) if fn is tokens.group_grad else want
            ok = p.slot >= 0
            prod = (srt[p.slot.long().clamp(min=0)] * tok[:, None, :]).masked_fill(~ok[..., None], 0.0)
            within(dw, prod.sum(2), 1.001 * (b - a + 2) * U32 * prod.abs().sum(2))
    one = normal(g, 1, 64)
    assert torch.equal(tokens.group(one.expand(90, 64), p)[:valid], one.expand(valid, 64))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,columns,dim", [(40_000, 2, 64), (40_000, 1, 64), (30_000, 4, 16), (20_000, 8, 32), (70_001, 2, 8),
                                           (3000, 3, 1024), (9000, 12, 64)])
def test_group_of_many_tokens(dtype, n, columns, dim):
    # enough for every launch shape that large batches take
    g = gen(n + columns)
    ids = make_ids(g, (n, columns), 300, pad=0.05)
    p = tokens.plan(ids, 300)
    slot = p.slot.long()
    ok, at = slot >= 0, slot.clamp(min=0)
    x, rows = normal(g, n, dim, dtype=dtype), normal(g, n * columns, dim, dtype=dtype)
    w = torch.rand(n, columns, generator=g, device="cuda")
    want = (x.double()[:, None, :] * w.double()[..., None])[ok]
    within(tokens.group(x, p, weights=w)[slot[ok]], want, (U[dtype] + U32) * want.abs() + TINY[dtype])
    dxs, dw = tokens.ungroup_grad(x, p, weights=w, xs=rows)
    within(dxs[slot[ok]], want, (U[dtype] + U32) * want.abs() + TINY[dtype])
    picked = rows.double()[at].masked_fill(~ok[..., None], 0.0)
    prod = picked * x.double()[:, None, :]
    within(dw, prod.sum(2), 1.001 * (dim + 2) * U32 * prod.abs().sum(2))
    terms = picked * w.double()[..., None]
    want, tol = terms.sum(1), 1.001 * (columns + 2) * U32 * terms.abs().sum(1)
    within(tokens.ungroup(rows, p, weights=w), want, tol + U[dtype] * (want.abs() + tol) + TINY[dtype])
    dx, dw2 = tokens.group_grad(rows, p, weights=w, x=x)
    within(dx, want, tol + U[dtype] * (want.abs() + tol) + TINY[dtype])
    within(dw2, prod.sum(2), 1.001 * (dim + 2) * U32 * prod.abs().sum(2))


def test_group_of_nothing():
    p = tokens.plan(torch.empty(0, 4, dtype=torch.int32, device="cuda"), 5)
    x = torch.empty(0, 16, device="cuda")
    assert tokens.group(x, p).shape == (0, 16) and tokens.ungroup(x, p).shape == (0, 16)
    p = tokens.plan(torch.full((6, 2), -1, device="cuda"), 5)
    out = torch.full((12, 8), 3.0, device="cuda")
    tokens.group(torch.ones(6, 8, device="cuda"), p, out=out)
    assert bool((out == 3).all())
    y = tokens.ungroup(torch.full((12, 8), float("nan"), device="cuda"), p, weights=torch.full((6, 2), float("inf"), device="cuda"))
    assert bool((y == 0).all())


@pytest.mark.parametrize("n,columns,dim", [(40, 2, 64), (40, 4, 256), (40, 8, 64), (40, 12, 64), (3, 3, 5000), (3000, 4, 1024)])
def test_dropped_choices_meet_no_infinity(n, columns, dim):
    g = gen(n)
    ids = make_ids(g, (n, columns), 9, pad=0.4)
    p = tokens.plan(ids, 9)
    drop = p.slot < 0
    x = torch.full((n, dim), float("inf"), device="cuda")
    rows = normal(g, n * columns, dim).abs() + 1
    _, dw = tokens.group_grad(rows, p, x=x)
    assert bool((dw[drop] == 0).all()) and bool((dw[~drop] == float("inf")).all())
    dxs, dw = tokens.ungroup_grad(x, p, xs=rows)
    assert bool((dw[drop] == 0).all()) and bool((dw[~drop] == float("inf")).all())


def test_the_same_row_twice():
    # one token may choose one group several times: a place for each
    ids = torch.tensor([[2, 2, 2], [0, 2, 0]], device="cuda")
    p = tokens.plan(ids, 3)
    assert p.offsets.tolist() == [0, 2, 2, 6] and p.slot.tolist() == [[2, 3, 4], [0, 5, 1]]
    x = torch.tensor([[1.0], [10.0]], device="cuda")
    assert tokens.group(x, p).view(-1).tolist() == [10, 10, 1, 1, 1, 10]
    assert tokens.ungroup(tokens.group(x, p), p).view(-1).tolist() == [3, 30]


# ---- together ----------------------------------------------------------------------

def test_a_layer_of_experts_and_its_table():
    """Rows read by token id, routed to groups with a matrix each, summed back
    by their weights, and all gradients, against autograd in 64 bits."""
    g = gen(20)
    n, columns, dim, vocab, groups = 300, 2, 64, 90, 5
    table, mats = normal(g, vocab, dim), normal(g, groups, dim, dim) / 8
    ids = make_ids(g, (n,), vocab, pad=0.05, spread="head")
    choice = make_ids(g, (n, columns), groups, pad=0.1)
    scale, w = torch.rand(n, generator=g, device="cuda"), torch.rand(n, columns, generator=g, device="cuda")
    dy = normal(g, n, dim)

    ip, cp = tokens.plan(ids, vocab), tokens.plan(choice, groups)
    x = tokens.lookup(table, ids, scale=scale, alpha=2.0)
    xs = tokens.group(x, cp, out=torch.zeros(n * columns, dim, device="cuda"))
    ends = cp.offsets.tolist()
    hs = torch.zeros_like(xs)
    for e in range(groups):
        hs[ends[e]:ends[e + 1]] = (xs[ends[e]:ends[e + 1]].double() @ mats[e].double()).float()
    y = tokens.ungroup(hs, cp, weights=w)
    dhs, dw = tokens.ungroup_grad(dy, cp, weights=w, xs=hs)
    dxs = torch.zeros_like(xs)
    for e in range(groups):
        dxs[ends[e]:ends[e + 1]] = (dhs[ends[e]:ends[e + 1]].double() @ mats[e].double().t()).float()
    dx = tokens.group_grad(dxs, cp)
    dt, ds = tokens.lookup_grad(dx, ip, scale=scale, alpha=2.0, table=table)

    t64, s64, w64 = (v.double().requires_grad_() for v in (table, scale, w))
    ok = (ids >= 0) & (ids < vocab)
    x64 = torch.where(ok[:, None], t64[torch.where(ok, ids, 0).long()] * (2.0 * s64)[:, None], 0.0)
    used = (choice >= 0) & (choice < groups)
    h64 = torch.einsum("nd,ncde->nce", x64, mats.double()[torch.where(used, choice, 0).long()])
    y64 = (torch.where(used[..., None], h64, 0.0) * w64[..., None]).sum(1)
    y64.backward(dy.double())
    # the forward pass rounds x (3), xs, hs (1 each) and two weighted terms (4): below 16 half steps of the
    # largest partial sums; the backward pass adds dim or the longest row's sums
    longest = int((ip.offsets[1:] - ip.offsets[:-1]).max())
    for got, want, m in ((y, y64, 16), (dw, w64.grad, 16 + dim), (dt, t64.grad, 32 + longest), (ds, s64.grad, 32 + dim)):
        scale_of = want.detach().abs().max() * 8  # products of 64 unit terms cancel to an eighth of their size
        within(got, want.detach(), m * U32 * scale_of * 8)


def test_the_same_inputs_give_the_same_bits():
    g = gen(30)
    ids = make_ids(g, (200_000,), 500, spread="head")
    grad, table = normal(g, 200_000, 64), normal(g, 500, 64)
    p = tokens.plan(ids, 500)
    first = tokens.lookup_grad(grad, p, table=table)
    for _ in range(4):
        again = tokens.lookup_grad(grad, tokens.plan(ids, 500), table=table)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def _pass(s):
    p = tokens.plan(s["ids"], 64)
    x = tokens.lookup(s["table"], s["ids"], scale=s["scale"])
    xs = tokens.group(x.view(-1, x.shape[-1]), tokens.plan(s["choice"], 16))
    dt = tokens.lookup_grad(x, p, scale=s["scale"], table=s["table"])
    cp = tokens.plan(s["choice"], 16)
    y = tokens.ungroup(xs, cp, weights=s["w"])
    return (x, y, *dt, *tokens.ungroup_grad(y, cp, weights=s["w"], xs=xs))


def _state(seed, n=1500):
    g = gen(seed)
    return dict(ids=make_ids(g, (n,), 64, spread="head"), table=normal(g, 64, 128), choice=make_ids(g, (n, 2), 16),
                scale=torch.rand(n, generator=g, device="cuda"), w=torch.rand(n, 2, generator=g, device="cuda"))


@pytest.mark.parametrize("n", [1500, 70_001])
def test_captured_graphs_replay_on_new_inputs(n):
    states = [_state(40, n), _state(41, n)]
    for s in states:
        _pass(s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_pass(s))
        graphs.append(gr)
    for k, (s, seed) in enumerate(zip(states, (50, 51))):
        for name, v in _state(seed, n).items():
            s[name].copy_(v)
    # both graphs in flight at once, each on a stream of its own
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for s, out in zip(states, outs):
        for a, b in zip(out, _pass(s)):
            assert torch.equal(a, b)


def test_streams():
    s = _state(60, n=60_000)
    want = [v.clone() for v in _pass(s)]
    torch.cuda.synchronize()
    side, late = torch.cuda.Stream(), torch.zeros(8192, 8192, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # torch's current stream: ordered behind what runs there
        for _ in range(3):
            late = late @ late
        s["scale"].mul_(0).add_(s["scale"].new_ones(())).mul_(0.5)
        half = _pass(s)
        x = tokens.lookup(s["table"], s["ids"], scale=torch.full_like(s["scale"], 0.5))
    torch.cuda.synchronize()
    assert torch.equal(half[0], x)
    # a context with a stream of its own choice
    s2 = _state(60, n=60_000)
    torch.cuda.synchronize()
    with Context(0) as ctx:
        st = torch.cuda.Stream()
        ctx.set_stream(st.cuda_stream)
        out = tokens.lookup(s2["table"], s2["ids"], scale=s2["scale"], ctx=ctx)
        p = tokens.plan(s2["ids"], 64, ctx=ctx)
        dt = tokens.lookup_grad(out, p, scale=s2["scale"], table=s2["table"], ctx=ctx)
        st.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(dt[0], want[2]) and torch.equal(dt[1], want[3])


def test_two_threads_on_one_context():
    import threading

    states = [_state(70 + k, n=3000) for k in range(4)]
    want = [[v.clone() for v in _pass(s)] for s in states]
    torch.cuda.synchronize()
    got, failed = {}, []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[k] = _pass(states[k])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # reported below
            failed.append(e)

    th = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in th]
    [t.join() for t in th]
    assert not failed, failed
    for k in range(4):
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k]))


def test_places_beyond_32_bits():
    # rows a quarter of 2^32 elements apart: the last place is beyond 32 bits
    stride, dim = 2**30 + 64, 64
    buf = torch.zeros(4 * stride + dim, dtype=BF16, device="cuda")
    rows = buf.as_strided((5, dim), (stride, 1))
    g = gen(80)
    x = normal(g, 5, dim, dtype=BF16)
    ids = torch.tensor([[4], [0], [2], [1], [3]], device="cuda")
    p = tokens.plan(ids, 5)
    tokens.group(x, p, out=rows)
    assert torch.equal(rows[p.slot.view(-1).long()], x)
    assert torch.equal(tokens.ungroup(rows, p), x)
    assert torch.equal(tokens.lookup(rows, ids.view(-1)), rows[ids.view(-1)])
    assert torch.equal(tokens.lookup_grad(rows, tokens.plan(ids.view(-1), 5))[ids.view(-1)], rows)
    buf.zero_()
    tokens.lookup(x, ids.view(-1), out=rows)
    assert torch.equal(rows, x[ids.view(-1)])
    buf.zero_()
    tokens.lookup_grad(x, tokens.plan(ids.view(-1), 5), out=rows)
    assert torch.equal(rows[ids.view(-1)], x)


# ---- refusals ----------------------------------------------------------------------

def _name(fn, *a, **k):
    with pytest.raises(MvrError) as e:
        fn(*a, **k)
    return e.value.name


def test_refusals():
    x = torch.zeros(6, 8, device="cuda")
    ids = torch.zeros(6, dtype=torch.int32, device="cuda")
    p = tokens.plan(ids, 4)
    p2 = tokens.plan(torch.zeros(3, 2, dtype=torch.int64, device="cuda"), 4)
    t = torch.zeros(4, 8, device="cuda")
    assert _name(tokens.lookup, t.cpu(), ids) == "InvalidArgument"
    assert _name(tokens.lookup, t[0], ids) == "DimMismatch"
    assert _name(tokens.lookup, t[:, :0], ids) == "DimMismatch"
    assert _name(tokens.lookup, t[:0], ids) == "InvalidArgument"
    assert _name(tokens.lookup, t, ids, scale=torch.zeros(5, device="cuda")) == "LengthMismatch"
    assert _name(tokens.lookup, t, ids, scale=torch.zeros(6, device="cuda", dtype=F16)) == "InvalidArgument"
    assert _name(tokens.lookup, t, ids, out=torch.zeros(5, 8, device="cuda")) == "OutBufferWrongSize"
    assert _name(tokens.lookup, t, ids, out=torch.zeros(6, 7, device="cuda")) == "DimMismatch"
    assert _name(tokens.lookup, t, ids, out=torch.zeros(6, 8, device="cuda", dtype=BF16)) == "InvalidArgument"
    assert _name(tokens.lookup, t, ids, out=torch.zeros(8, 6, device="cuda").t()) == "InvalidArgument"
    assert _name(tokens.lookup, t, ids, out=t[:1].expand(6, 8)) == "InvalidArgument"
    assert _name(tokens.lookup_grad, x[:5], p) == "LengthMismatch"
    assert _name(tokens.lookup_grad, x, p, table=torch.zeros(5, 8, device="cuda")) == "LengthMismatch"
    assert _name(tokens.lookup_grad, x, p, table=t.half()) == "InvalidArgument"
    assert _name(tokens.lookup_grad, x, p, out=t.half()) == "InvalidArgument"
    assert _name(tokens.lookup_grad, x.half(), p, out=t.bfloat16()) == "InvalidArgument"
    assert _name(tokens.group, x, p2) == "LengthMismatch"
    assert _name(tokens.ungroup, x[:3], p2) == "LengthMismatch"
    assert _name(tokens.group, x[:3], p2, weights=torch.zeros(5, device="cuda")) == "LengthMismatch"
    assert _name(tokens.group_grad, x, p2, x=x[:3].half()) == "InvalidArgument"
    assert _name(tokens.ungroup_grad, x[:3], p2, xs=x[:, :4]) == "DimMismatch"
    # a call that was refused leaves the context usable
    assert tokens.lookup(t, ids).shape == (6, 8)


def test_c_entry_refusals(ctx):
    lib, h = ctx.lib, ctx.handle
    x = torch.zeros(64, 64, device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")
    a, j = x.data_ptr(), i.data_ptr()
    torch.cuda.synchronize()  # the context's own stream does not wait for torch's
    bad, dim = CODES["InvalidArgument"], CODES["DimMismatch"]

    def lookup(table=a, dtype=0, rows=4, d=8, ts=8, ids=j, idb=4, n=2, scale=None, out=a + 4096, os=8):
        return lib.mvr_lookup_device(h, table, dtype, rows, d, ts, ids, idb, n, scale, 1.0, out, os)

    assert lookup() == 0
    for kw in (dict(table=None), dict(dtype=3), dict(dtype=-1), dict(rows=0), dict(rows=2**31 - 1), dict(ids=None),
               dict(idb=2), dict(ids=j + 2), dict(idb=8, ids=j + 4), dict(out=None), dict(os=7), dict(os=2**32),
               dict(ts=2**32), dict(d=2**20 + 1, os=2**21), dict(n=2**40), dict(table=a + 2),
               dict(out=a + 4098), dict(scale=a + 1)):
        assert lookup(**kw) == bad, kw
    assert lookup(d=0) == dim and lookup(n=0, ids=None, out=None) == 0

    need = C.c_uint64(0)
    assert lib.mvr_token_plan_bytes(64, 4, C.byref(need)) == 0
    ws = torch.zeros(need.value + 64, dtype=torch.uint8, device="cuda")
    o = [torch.zeros(64, dtype=torch.int32, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()

    def plan(ids=j, idb=4, n=64, rows=4, off=o[0].data_ptr(), order=o[1].data_ptr(), keys=o[2].data_ptr(),
             slot=o[3].data_ptr(), w=ws.data_ptr(), nb=need.value):
        return lib.mvr_token_plan_device(h, ids, idb, n, rows, off, order, keys, slot, w, nb)

    assert plan() == 0
    for kw in (dict(ids=None), dict(idb=1), dict(rows=0), dict(n=2**31), dict(off=None), dict(order=None),
               dict(keys=None), dict(slot=None), dict(order=o[1].data_ptr() + 1)):
        assert plan(**kw) == bad, kw
    if need.value:
        assert plan(w=None) == bad and plan(nb=need.value - 1) == bad and plan(w=ws.data_ptr() + 4) == bad

    def group(src=a, dtype=0, ss=8, n=4, columns=2, d=8, slot=o[3].data_ptr(), w=None, out=a + 4096, os=8):
        return lib.mvr_group_rows_device(h, src, dtype, ss, n, columns, d, slot, w, out, os)

    assert group() == 0
    for kw in (dict(src=None), dict(dtype=7), dict(n=2**31), dict(columns=0), dict(slot=None), dict(w=a + 1),
               dict(out=None), dict(os=7), dict(src=a + 1), dict(n=2**30, columns=4)):
        assert group(**kw) == bad, kw
    assert group(d=0) == dim
    assert lib.mvr_ungroup_rows_grad_device(h, a, 0, 8, 4, 2, 8, o[3].data_ptr(), None, None, 8, a + 4096, 8,
                                            a + 8192) == bad  # the weights' gradient without xs
    assert lib.mvr_group_rows_grad_device(h, a, 0, 8, 4, 2, 8, o[3].data_ptr(), None, None, 8, a + 4096, 8,
                                          a + 8192) == bad
    ctx.sync()
