"""CPU: what the linear layers over row groups check before they call a kernel -- groups that a caller has altered, operands whose derivative would be lost."""
import copy
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils import _pytree

from bnn_chaos_model_amd import _native as N
from bnn_chaos_model_amd import member_linear as M
from bnn_chaos_model_amd import ops


# ---- groups --------------------------------------------------------------------------------------------------------------------------------
def some_groups(rows=6, G=2):
    return ops.RowGroups(torch.arange(rows, dtype=torch.int32), torch.zeros(G + 1, dtype=torch.int32), (rows,))


def check(groups, rows=6, G=2, gather=True):
    return M._check_groups(groups, torch.zeros(rows, 3), G, gather)   # (both on the CPU: "the same device")


def rebuilt(groups, **kw):
    """The ways a named tuple is made from another one: all of them must end in the same checks."""
    values = {**groups._asdict(), **kw}
    yield groups._replace(**kw)
    yield type(groups)(**values)
    yield type(groups)._make(values.values())
    yield copy.copy(groups)._replace(**kw)
    leaves, spec = _pytree.tree_flatten(groups)
    yield _pytree.tree_unflatten(leaves, spec)._replace(**kw)


def test_groups_as_they_are_made_pass():
    assert check(some_groups()) == (6, 1)
    assert check(some_groups()._replace(shape=(3, 2)), rows=3) == (3, 2)
    assert check(some_groups()._replace(shape=(3, 2)), rows=6, gather=False) == (3, 2)


@pytest.mark.parametrize("kw,rows,error", [
    (dict(shape=(60,)), 60, ValueError),                                       # more pairs than order holds
    (dict(shape=(6, 7)), 6, ValueError),
    (dict(shape=(5,)), 5, ValueError),
    (dict(shape=()), 6, ValueError),
    (dict(shape=(6, 1, 1)), 6, ValueError),
    (dict(order=torch.arange(6)), 6, TypeError),                               # 64-bit indices
    (dict(offsets=torch.zeros(3, dtype=torch.int64)), 6, TypeError),
    (dict(order=[0, 1, 2, 3, 4, 5]), 6, TypeError),
    (dict(offsets=None), 6, TypeError),
    (dict(order=torch.arange(12, dtype=torch.int32)[::2]), 6, ValueError),     # strided
    (dict(offsets=torch.zeros(6, dtype=torch.int32)[::2]), 6, ValueError),
    (dict(order=torch.arange(5, dtype=torch.int32)), 6, ValueError),
    (dict(offsets=torch.zeros(2, dtype=torch.int32)), 6, ValueError)])
def test_altered_groups_are_refused(kw, rows, error):
    for groups in rebuilt(some_groups(), **kw):
        with pytest.raises(error):
            check(groups, rows=rows)


def test_a_tensor_of_the_groups_altered_in_place_is_refused():
    groups = some_groups()
    groups.order.resize_(4)
    with pytest.raises(ValueError):
        check(groups)


def test_group_rows_returns_the_checked_type():
    """(No subclass that a check could pass over.)"""
    assert not [c for c in vars(M).values() if isinstance(c, type) and issubclass(c, M.RowGroups) and c is not M.RowGroups]


# ---- forward-mode derivatives ----------------------------------------------------------------------------------------------------------------
def layer_calls():
    """(name of the operand that is replaced, the call with it) of every entry point that takes values a derivative may run through."""
    x, w, b, dy = torch.zeros(6, 3), torch.zeros(2, 4, 3), torch.zeros(2, 4), torch.zeros(6, 4)
    gr = some_groups()
    xq, wq = ops.QuantRows(torch.zeros(6, 3, dtype=torch.int8), torch.ones(6)), ops.QuantRows(torch.zeros(2, 4, 3, dtype=torch.int8), torch.ones(2, 4))
    yield "x", x, lambda t: ops.grouped_linear(t, w, gr, bias=b)
    yield "weight", w, lambda t: ops.grouped_linear(x, t, gr, bias=b)
    yield "bias", b, lambda t: ops.grouped_linear(x, w, gr, bias=t)
    yield "dy", dy, lambda t: ops.grouped_linear_grads(t, x, w, gr)
    yield "x", x, lambda t: ops.grouped_linear_grads(dy, t, w, gr)
    yield "weight", w, lambda t: ops.grouped_linear_grads(dy, x, t, gr)
    yield "y", dy, lambda t: ops.grouped_linear_grads(dy, x, w, gr, y=t)
    yield "x", x, lambda t: ops.quantize_rows(t)
    yield "x", x, lambda t: ops.int8_linear(t, wq, groups=gr)
    yield "bias", b, lambda t: ops.int8_linear(x, wq, groups=gr, bias=t)
    yield "x.scale", xq.scale, lambda t: ops.int8_linear(xq._replace(scale=t), wq, groups=gr)
    yield "weight.scale", wq.scale, lambda t: ops.int8_linear(xq, wq._replace(scale=t), groups=gr)


@pytest.mark.parametrize("i", range(12))
def test_operands_with_a_tangent_are_refused(i):
    """... instead of a result without one, which a caller reads as a derivative of zero."""
    name, t, call = list(layer_calls())[i]
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match=f"^{name} carries a forward-mode tangent"):
            call(forward_ad.make_dual(t, torch.ones_like(t)))
        with torch.no_grad(), pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(TypeError):       # a plain operand next to a dual level: the next check (these are on the CPU)
            call(t)


# ---- the kernels that the tests reach --------------------------------------------------------------------------------------------------------
FEW, SHORT, TILE, DW, DW_LISTED = range(5)   # (bnn_grouped_kind)


def form(fn, q, *args):
    out = (C.c_int32 * 6)()
    assert fn(C.byref(q), *args, out) == 0
    return tuple(out)


def forms(rows, members, copies, K, No, dtype, moved):
    """{(pass, bytes of an operand's element): what it runs} for dense operands as torch allocates them (addresses of whole 512 bytes)."""
    L, es, c = N.lib(), 4 if dtype == 0 else 2, max(copies, 1)
    q = N.BnnGrouped(rows, c, members, K, No, dtype, moved, moved, 0, K, No, No * K, K, 512, 512)
    out = {("forward", es): form(L.bnn_grouped_linear_form, q, 0, 512, 512, 512), ("dx of copies" if c > 1 and moved else "dx", es): form(L.bnn_grouped_linear_form, q, 1, 512, 512, 512),
           ("dw", es): form(L.bnn_grouped_linear_form, q, 2, 512, 512, 512), ("int8", 1): form(L.bnn_int8_linear_form, q, 512, 512, 512)}
    return out


def test_the_sizes_reach_every_kernel():
    from test_member_linear_forms import SIZES
    got = set()
    for (n, G, c, K, No) in SIZES:
        for dtype in (0, 1):
            for moved in (1, 0):
                for (what, es), (kind, rows, outputs, direct, steps, splits) in forms(n, G, c, K, No, dtype, moved).items():
                    if kind == TILE and (No if what.startswith("dx") else K) * es <= 4 * 128:
                        continue    # (at least five stages, so that the loop turns)
                    got.add((what, es, kind, rows, outputs, direct, steps, splits > 1))
    tiles = [(64, 64, 0), (64, 64, 1), (128, 128, 0), (128, 128, 1), (256, 256, 1)]
    want = set()
    for what, es in (("forward", 4), ("forward", 2), ("int8", 1)):
        want |= {(what, es, FEW, r, o, d, 0, False) for r, o in ((16, 16), (16, 32), (32, 32)) for d in (0, 1)}
        want |= {(what, es, SHORT, r, o, 0, s, False) for r, o in ((64, 64), (64, 128), (128, 128)) for s in (1, 2, 3, 4)}
        want |= {(what, es, TILE, r, o, d, 0, False) for r, o, d in tiles}
    want |= {("int8", 1, TILE, 256, 128, 0, 0, False), ("forward", 4, SHORT, 128, 64, 0, 3, False), ("int8", 1, SHORT, 128, 64, 0, 1, False)}
    for what in ("dx", "dx of copies"):
        want |= {(what, es, TILE, r, o, d, 0, False) for es in (4, 2) for r, o, d in tiles}
    for kind in (DW, DW_LISTED):
        want |= {("dw", es, kind, t, t, d, 0, False) for es in (4, 2) for t in (64, 128) for d in (0, 1)} | {("dw", 2, kind, 256, 256, 1, 0, False)}
        want |= {("dw", es, kind, 64, 64, d, 0, True) for es in (4, 2) for d in (0, 1)}
    assert not want - got, sorted(want - got)
    assert not {f for f in got if f not in want and f[2] != SHORT}      # a form that is new must be written down here


def test_form_refuses_what_the_calls_refuse():
    L, out = N.lib(), (C.c_int32 * 6)()
    q = N.BnnGrouped(4, 1, 2, 8, 3, 0, 0, 0, 0, 8, 3, 24, 8, None, 1)
    for p in (-1, 3):
        assert L.bnn_grouped_linear_form(C.byref(q), p, 16, 16, 16, out) == N.ERR_INVALID
    assert L.bnn_grouped_linear_form(C.byref(q), 0, 16, 16, 16, None) == L.bnn_int8_linear_form(C.byref(q), 16, 16, 16, None) == N.ERR_INVALID
    q.copies = 0
    assert L.bnn_grouped_linear_form(C.byref(q), 0, 16, 16, 16, out) == L.bnn_int8_linear_form(C.byref(q), 16, 16, 16, out) == N.ERR_INVALID
    empty = N.BnnGrouped(0, 1, 2, 8, 3, 0, 0, 0, 0, 8, 3, 24, 8, None, 1)
    assert all(L.bnn_grouped_linear_form(C.byref(empty), p, 16, 16, 16, out) == 0 for p in range(3))
