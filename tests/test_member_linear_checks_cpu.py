"""CPU: what the linear layers over row groups check before they call a kernel -- groups that a caller has altered, operands whose derivative would be lost."""
import copy

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils import _pytree

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
