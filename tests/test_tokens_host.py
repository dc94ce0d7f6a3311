"""Token operators without a GPU: what the host side refuses and computes."""
import ctypes as C

import pytest
import torch

from ir_multivector_retrieval_b200 import _lib, tokens
from ir_multivector_retrieval_b200._lib import CODES, MvrError


def _plan(n=4, columns=None, rows=8):
    shape = (n,) if columns is None else (n, columns)
    k = n * (columns or 1)
    i32 = torch.int32
    return tokens.Plan(rows, torch.zeros(rows + 1, dtype=i32), torch.arange(k, dtype=i32),
                       torch.zeros(k, dtype=i32), torch.arange(k, dtype=i32).view(shape))


def _name(fn, *a, **k):
    with pytest.raises(MvrError) as e:
        fn(*a, **k)
    return e.value.name


@pytest.mark.parametrize("columns,n,got", [(None, 4, (4, 1)), (3, 4, (4, 3)), (1, 5, (5, 1)), (2, 0, (0, 2)), (None, 0, (0, 1))])
def test_plan_sizes(columns, n, got):
    p = _plan(n, columns)
    assert (p.n, p.columns) == got and p.n_ids == got[0] * got[1]


def test_host_tensors_are_refused():
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    assert _name(tokens.lookup, x, ids) == "InvalidArgument"
    assert _name(tokens.plan, ids, 8) == "InvalidArgument"
    for fn in (tokens.group, tokens.ungroup, tokens.lookup_grad, tokens.group_grad, tokens.ungroup_grad):
        assert _name(fn, x, _plan()) == "InvalidArgument"


@pytest.mark.parametrize("rows", [0, -1, 2**31 - 1, 2**40])
def test_plan_refuses_row_counts(rows):
    assert _name(tokens.plan, torch.zeros(4, dtype=torch.int32), rows) == "InvalidArgument"


@pytest.mark.parametrize("ids", [torch.zeros(2, 2, 2, dtype=torch.int32), torch.zeros(2, 0, dtype=torch.int32),
                                 torch.zeros(4), torch.zeros(4, dtype=torch.int16), torch.tensor(3)])
def test_plan_refuses_ids(ids):
    assert _name(tokens.plan, ids, 8) == "InvalidArgument"


def test_types_are_refused():
    assert _name(tokens.lookup, torch.zeros(4, 8, dtype=torch.float64), torch.zeros(4, dtype=torch.int32)) == \
        "InvalidArgument"
    assert _name(tokens.group, torch.zeros(4, 8, dtype=torch.int32), _plan()) == "InvalidArgument"


def test_bad_plans_are_refused():
    p = _plan()
    p.slot = p.slot.long()
    assert _name(tokens.group, torch.zeros(4, 8), p) == "InvalidArgument"
    p = _plan()
    p.order = p.order[:-1]
    assert _name(tokens.lookup_grad, torch.zeros(4, 8), p) == "LengthMismatch"
    p = _plan()
    p.rows = 9
    assert _name(tokens.lookup_grad, torch.zeros(4, 8), p) == "LengthMismatch"


def test_accumulate_needs_out():
    assert _name(tokens.lookup_grad, torch.zeros(4, 8), _plan(), accumulate=True) == "InvalidArgument"


def test_workspace_sizes():
    lib, b = _lib.load(), C.c_uint64(7)
    bad = CODES["InvalidArgument"]
    assert lib.mvr_token_plan_bytes(0, 5, C.byref(b)) == 0
    small = b.value
    assert lib.mvr_token_plan_bytes(1_000_000, 5, C.byref(b)) == 0 and b.value >= small
    assert lib.mvr_token_plan_bytes(2**31 - 1, 2**31 - 2, C.byref(b)) == 0
    assert lib.mvr_token_plan_bytes(2**31, 5, C.byref(b)) == bad
    assert lib.mvr_token_plan_bytes(5, 0, C.byref(b)) == bad
    assert lib.mvr_token_plan_bytes(5, 2**31 - 1, C.byref(b)) == bad
    assert lib.mvr_token_plan_bytes(5, 5, None) == bad
    assert lib.mvr_lookup_grad_bytes(2**31 - 1, 64, C.byref(b)) == 0
    assert lib.mvr_lookup_grad_bytes(2**31, 64, C.byref(b)) == bad
    assert lib.mvr_lookup_grad_bytes(5, 0, C.byref(b)) == bad
    assert lib.mvr_lookup_grad_bytes(5, 5, None) == bad


def test_a_null_context_is_refused():
    lib, bad = _lib.load(), CODES["InvalidArgument"]
    assert lib.mvr_lookup_device(None, None, 0, 1, 1, 1, None, 4, 0, None, 1.0, None, 1) == bad
    assert lib.mvr_token_plan_device(None, None, 4, 0, 1, None, None, None, None, None, 0) == bad
    assert lib.mvr_group_rows_device(None, None, 0, 1, 0, 1, 1, None, None, None, 1) == bad
    assert lib.mvr_ungroup_rows_device(None, None, 0, 1, 0, 1, 1, None, None, None, 1) == bad
