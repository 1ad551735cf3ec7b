"""CPU: what the grouped and 8-bit linear layers refuse, in the Python surface and at the C boundary (every refusal comes before any GPU call)."""
import ctypes as C

import pytest
import torch

from bnn_chaos_model_amd import _native as N
from bnn_chaos_model_amd import ops


def test_cpu_tensors_and_wrong_types_are_refused():
    with pytest.raises(TypeError):
        ops.group_rows(torch.zeros(4, dtype=torch.int32), 2)
    with pytest.raises(TypeError):
        ops.group_rows([0, 1], 2)
    x, w = torch.zeros(4, 8), torch.zeros(2, 3, 8)
    gr = ops.RowGroups(torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), (4,))
    with pytest.raises(TypeError):
        ops.grouped_linear(x, w, gr)
    with pytest.raises(TypeError):
        ops.grouped_linear_grads(x, x, w, gr)
    with pytest.raises(TypeError):
        ops.quantize_rows(x)
    with pytest.raises(TypeError):
        ops.int8_linear(x, ops.QuantRows(w[0].to(torch.int8), torch.zeros(3)))
    with pytest.raises(TypeError):
        ops.int8_linear(ops.QuantRows(x.to(torch.int8), torch.zeros(4)), ops.QuantRows(w[0].to(torch.int8), torch.zeros(3)))


def grouped(**kw):
    q = N.BnnGrouped(4, 1, 2, 8, 3, 0, 0, 0, 0, 8, 3, 24, 8, None, 1)   # (addresses that are never read: the calls below are refused first)
    for k, v in kw.items():
        setattr(q, k, v)
    return q


@pytest.mark.parametrize("change,code", [(dict(rows=-1), N.ERR_INVALID), (dict(copies=0), N.ERR_INVALID), (dict(members=0), N.ERR_INVALID), (dict(inputs=0), N.ERR_INVALID),
                                         (dict(outputs=0), N.ERR_INVALID), (dict(dtype=3), N.ERR_INVALID), (dict(dtype=-1), N.ERR_INVALID),
                                         (dict(rows=1 << 31), N.ERR_RANGE), (dict(rows=1 << 30), N.ERR_RANGE), (dict(rows=(1 << 30) // 3 + 1, copies=3), N.ERR_RANGE), (dict(rows=1 << 30, copies=4), N.ERR_RANGE), (dict(inputs=(1 << 24) + 1), N.ERR_RANGE),
                                         (dict(members=(1 << 24) + 1), N.ERR_RANGE), (dict(gather=1), N.ERR_INVALID), (dict(scatter=1), N.ERR_INVALID),
                                         (dict(offsets=None), N.ERR_INVALID)])
def test_c_boundary_refuses_bad_descriptors(change, code):
    L, q = N.lib(), grouped(**change)
    assert L.bnn_grouped_linear(C.byref(q), 16, 16, None, 16, None) == code
    assert len(L.bnn_last_error()) > 5
    assert L.bnn_grouped_linear_dx(C.byref(q), 16, 16, 16, 16, None) == code
    assert L.bnn_grouped_linear_dw(C.byref(q), 16, 16, 16, None, 16, None) == code
    if change != dict(offsets=None):
        assert L.bnn_int8_linear(C.byref(q), 16, 16, 16, 16, None, 16, None) == code


def test_c_boundary_refuses_missing_pointers_and_sizes():
    L, q = N.lib(), grouped()
    for args in ((None, 16, None, 16), (16, None, None, 16), (16, 16, None, None)):
        assert L.bnn_grouped_linear(C.byref(q), *args, None) == N.ERR_INVALID
    assert L.bnn_grouped_linear(None, 16, 16, None, 16, None) == N.ERR_INVALID
    assert L.bnn_grouped_linear_dx(C.byref(grouped(copies=2, gather=1, order=16)), 16, 16, 16, None, None) == N.ERR_INVALID   # the copies' workspace
    assert L.bnn_grouped_linear_dw(C.byref(q), 16, 16, None, None, None, None) == N.ERR_INVALID
    assert L.bnn_int8_linear(C.byref(grouped(inputs=131073)), 16, 16, 16, 16, None, 16, None) == N.ERR_RANGE
    assert L.bnn_int8_linear(C.byref(grouped(offsets=None)), 16, 16, 16, 16, None, 16, None) == N.ERR_INVALID          # two members, no offsets
    assert L.bnn_int8_linear(C.byref(q), 16, None, 16, 16, None, 16, None) == N.ERR_INVALID
    assert L.bnn_quantize_rows(16, 0, 4, 8, 8, 16, 7, 16, None) == N.ERR_INVALID
    assert L.bnn_quantize_rows(None, 0, 4, 8, 8, 16, 8, 16, None) == N.ERR_INVALID
    assert L.bnn_group_rows_i32(16, 4, 0, 16, 16, None, None) == N.ERR_INVALID
    assert L.bnn_group_rows_i32(16, 4, 4097, 16, 16, None, None) == N.ERR_UNSUPPORTED
    assert L.bnn_group_rows_i32(16, 1 << 31, 4, 16, 16, 16, None) == L.bnn_group_rows_i32(16, 1 << 30, 4, 16, 16, 16, None) == N.ERR_RANGE
    assert L.bnn_group_rows_i32(16, 100000, 4, 16, 16, None, None) == N.ERR_INVALID                                    # the sort's workspace
    assert L.bnn_group_rows_i32(16, 4, 4, 16, None, None, None) == N.ERR_INVALID
    assert L.bnn_relu_grad(16, 8, None, 8, 4, 8, 0, 16, None) == N.ERR_INVALID
    # dx of copies is dense: refused before anything is enqueued
    assert L.bnn_grouped_linear_dx(C.byref(grouped(copies=2, gather=1, order=16, x_row=9)), 16, 16, 16, 16, None) == N.ERR_INVALID
    assert b"dense" in L.bnn_last_error()


def test_empty_batches_need_no_device():
    L, q = N.lib(), grouped(rows=0)
    assert L.bnn_grouped_linear(C.byref(q), None, None, None, None, None) == 0
    assert L.bnn_grouped_linear_dx(C.byref(q), None, None, None, None, None) == 0
    assert L.bnn_int8_linear(C.byref(q), None, None, None, None, None, None, None) == 0
    assert L.bnn_quantize_rows(None, 0, 0, 8, 8, None, 8, None, None) == 0
    assert L.bnn_grouped_linear_dw_workspace_bytes(C.byref(q)) == 0 and L.bnn_grouped_linear_dx_workspace_bytes(C.byref(q)) == 0


def test_workspace_sizes():
    L = N.lib()
    assert L.bnn_group_rows_workspace_bytes(4096, 30) == 0 and L.bnn_group_rows_workspace_bytes(8193, 30) >= 3 * 31 * 4
    assert L.bnn_grouped_linear_dx_workspace_bytes(C.byref(grouped(copies=3, gather=1, order=16))) == 4 * 3 * 8 * 4
    assert L.bnn_grouped_linear_dx_workspace_bytes(C.byref(grouped(copies=3))) == 0
    from bnn_chaos_model_amd.member_linear import int8_rows_workspace
    for rows, copies, gather, k in ((1, 1, 0, 1), (7, 3, 0, 41), (7, 3, 1, 41), (5, 1, 1, 4096)):
        q = grouped(rows=rows, copies=copies, gather=gather, order=16, inputs=k)
        assert L.bnn_int8_linear_rows_workspace_bytes(C.byref(q)) == int8_rows_workspace(rows if gather else rows * copies, k)


def test_float_rows_in_8_bits_refusals():
    L, q = N.lib(), grouped()
    ok = (16, 1, 16, 16, 16, None, 16, None)
    for i, bad in ((0, None), (2, None), (3, None), (4, None), (6, None), (1, 3), (1, -1)):
        args = list(ok)
        args[i] = bad
        assert L.bnn_int8_linear_rows(C.byref(q), *args) == N.ERR_INVALID
    assert L.bnn_int8_linear_rows(C.byref(grouped(inputs=131073)), *ok) == N.ERR_RANGE
    assert L.bnn_int8_linear_rows(C.byref(grouped(gather=1)), *ok) == N.ERR_INVALID
    assert L.bnn_int8_linear_rows(C.byref(grouped(rows=0)), None, 0, None, None, None, None, None, None) == 0


def test_grids_beyond_the_launch_limit_are_refused():
    L = N.lib()
    for dtype in (0, 1):
        q = grouped(rows=1 << 29, inputs=4096, outputs=1 << 24, dtype=dtype)   # (rows of more than 256 bytes: tiles)
        assert L.bnn_grouped_linear(C.byref(q), 16, 16, None, 16, None) == N.ERR_RANGE
        assert L.bnn_int8_linear(C.byref(q), 16, 16, 16, 16, None, 16, None) == N.ERR_RANGE
    assert L.bnn_grouped_linear_dx(C.byref(grouped(rows=1 << 29, inputs=1 << 24)), 16, 16, 16, None, None) == N.ERR_RANGE
    assert L.bnn_grouped_linear_dw(C.byref(grouped(members=1 << 24, inputs=1024, outputs=1024)), 16, 16, 16, None, 16, None) == N.ERR_RANGE
    assert L.bnn_grouped_linear_dw(C.byref(grouped(inputs=1 << 24, outputs=1 << 24)), 16, 16, 16, None, 16, None) == N.ERR_RANGE
