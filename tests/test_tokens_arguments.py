"""What the token operators make of their arguments, without a GPU: host
tensors stand for device tensors and the library's calls are only noted."""
import pytest
import torch

from ir_multivector_retrieval_b200 import tokens
from ir_multivector_retrieval_b200._lib import MvrError


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(tokens, "_device_of", lambda *t: 0)
    monkeypatch.setattr(tokens, "_run", lambda ctx, device, name, *args: made.append(name))
    return made


def _plan(*shape, rows=8):
    n = torch.Size(shape).numel()
    i32 = torch.int32
    return tokens.Plan(rows, torch.zeros(rows + 1, dtype=i32), torch.arange(n, dtype=i32), torch.zeros(n, dtype=i32),
                       torch.arange(n, dtype=i32).view(shape))


def _refused(calls, fn, *a, **k):
    with pytest.raises(MvrError) as e:
        fn(*a, **k)
    assert not calls  # nothing was launched
    return e.value.name


# ---- shapes: as many values in another order are not the ids' --------------------

OTHER = [((6, 4), (4, 6)), ((6, 4), (2, 12)), ((2, 6), (6, 2)), ((3, 1, 5), (5, 3)), ((2, 3, 4), (4, 3, 2)),
         ((2, 3, 4), (2, 4, 3)), ((2, 3, 4), (3, 2, 4))]
SAME = [((6, 4), (6, 4)), ((6, 4), (24,)), ((24,), (6, 4)), ((6, 4), (2, 3, 4)), ((6, 4), (6, 1, 4)), ((6,), (6, 1)),
        ((6,), (1, 6)), ((6, 1), (1, 6)), ((1,), ()), ((), (1, 1)), ((2, 3, 4), (6, 4)), ((0, 4), (4, 0)), ((5, 0), (0,))]


@pytest.mark.parametrize("ids,got", OTHER)
def test_values_in_another_order_are_refused(calls, ids, got):
    t, n = torch.zeros(8, 16), torch.Size(ids).numel()
    i = torch.zeros(ids, dtype=torch.int32)
    assert _refused(calls, tokens.lookup, t, i, scale=torch.zeros(got)) == "LengthMismatch"
    assert _refused(calls, tokens.lookup, t, i, out=torch.zeros(*got, 16)) == "OutBufferWrongSize"
    p = _plan(*ids)
    grad = torch.zeros(n, 16)
    assert _refused(calls, tokens.lookup_grad, grad, p, scale=torch.zeros(got)) == "LengthMismatch"
    assert _refused(calls, tokens.lookup_grad, torch.zeros(*got, 16), p) == "LengthMismatch"
    w, x, xs = torch.zeros(got), torch.zeros(p.n, 16), torch.zeros(n, 16)
    for fn, a in ((tokens.group, x), (tokens.ungroup, xs), (tokens.group_grad, xs), (tokens.ungroup_grad, x)):
        assert _refused(calls, fn, a, p, weights=w) == "LengthMismatch"


def test_transposed_weights_are_refused(calls):
    p = _plan(6, 4)
    w = torch.zeros(6, 4)
    tokens.group(torch.zeros(6, 16), p, weights=w)
    calls.clear()
    assert _refused(calls, tokens.group, torch.zeros(6, 16), p, weights=w.t()) == "LengthMismatch"
    # one value a token is not one a choice
    assert _refused(calls, tokens.group, torch.zeros(6, 16), p, weights=torch.zeros(6)) == "LengthMismatch"


@pytest.mark.parametrize("ids,got", SAME)
def test_values_in_the_ids_order_are_taken(calls, ids, got):
    t, n = torch.zeros(8, 16), torch.Size(ids).numel()
    i = torch.zeros(ids, dtype=torch.int32)
    out = torch.zeros(*got, 16) if got else torch.zeros(1, 16)
    assert tokens.lookup(t, i, scale=torch.zeros(got), out=out) is out
    if ids:
        p = _plan(*ids)
        grad = torch.zeros(*got, 16) if got else torch.zeros(1, 16)
        tokens.lookup_grad(grad, p, scale=torch.zeros(got), table=t)
        if len(ids) > 1 and n:
            tokens.group(torch.zeros(p.n, 16), p, weights=torch.zeros(got))
            tokens.ungroup_grad(torch.zeros(p.n, 16), p, weights=torch.zeros(got), xs=torch.zeros(n, 16))
    assert calls


# ---- outputs given by the caller ---------------------------------------------------

def _writes(rows, dim):
    """Every call that takes an output, with the shape of that output."""
    i, p = torch.zeros(6, dtype=torch.int32), _plan(6, 2)
    q, t = _plan(6), torch.zeros(rows, dim)
    x, xs = torch.zeros(6, dim), torch.zeros(12, dim)
    return [(lambda o: tokens.lookup(t, i, out=o), 6), (lambda o: tokens.lookup_grad(x, q, out=o), rows),
            (lambda o: tokens.lookup_grad(x, q, table=t, out=o, accumulate=True), rows),
            (lambda o: tokens.group(x, p, out=o), 12), (lambda o: tokens.ungroup(xs, p, out=o), 6),
            (lambda o: tokens.group_grad(xs, p, out=o), 6), (lambda o: tokens.group_grad(xs, p, x=x, out=o), 6),
            (lambda o: tokens.ungroup_grad(x, p, out=o), 12), (lambda o: tokens.ungroup_grad(x, p, xs=xs, out=o), 12)]


@pytest.mark.parametrize("k", range(9))
def test_an_output_counts_as_changed(calls, k):
    call, n = _writes(8, 16)[k]
    out = torch.zeros(n, 16)
    leaf = torch.ones(n, 16, requires_grad=True)
    loss = (leaf * out).sum()  # saves what out holds
    call(out)
    assert calls
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    wide = torch.zeros(n, 40)  # a view counts for its base
    before = wide._version
    call(wide[:, 3:19])
    assert wide._version > before
    with torch.inference_mode():
        call(torch.zeros(n, 16))


def test_inputs_do_not_count_as_changed(calls):
    for call, n in _writes(8, 16):
        closed = {k: v for k, v in zip(call.__code__.co_freevars, (c.cell_contents for c in call.__closure__))}
        tensors = [v for v in closed.values() if isinstance(v, torch.Tensor)]
        before = [t._version for t in tensors]
        call(torch.zeros(n, 16))
        assert [t._version for t in tensors] == before


@pytest.mark.parametrize("shape", [(6, 0), (2, 3, 0), (0, 3, 0)])
def test_rows_of_no_length_are_refused(calls, shape):
    p = _plan(shape[0] if len(shape) == 2 else shape[0] * shape[1])
    for fn in (tokens.lookup_grad, tokens.group, tokens.ungroup, tokens.group_grad, tokens.ungroup_grad):
        assert _refused(calls, fn, torch.zeros(shape), p) == "DimMismatch"


# ---- strides -------------------------------------------------------------------------

@pytest.mark.parametrize("stride", [2**32 - 1, 2**32, 2**40])
def test_inputs_far_apart_are_copied(calls, stride):
    # without memory: the library takes strides below 2^32
    far = torch.empty(1, device="meta").as_strided((3, 16), (stride, 1))
    t, dim, got = tokens._rows(far, "x")
    assert t.shape == (3, 16) and dim == 16 and got == (stride if stride < 2**32 else 16) and t.stride(0) == got
    one, _, got = tokens._rows(far[:1], "x")
    assert one.data_ptr() == far.data_ptr() and got == 16  # a single row has no stride to copy for
