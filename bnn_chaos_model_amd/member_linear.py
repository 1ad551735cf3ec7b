"""Linear layers over row groups: rows sorted by the ensemble member that evaluates them, the layer of every member on its own rows (with
gradients), and the same layer on 8-bit operands.  ops.py offers these names next to the fused forward; this file holds their checks and calls.

The reference evaluates one random member per chunk of rows (figures/spock/regression.py:78-86); here a batch may mix members row by row, and a
layer may have any width.  As everywhere: work is enqueued on torch's current stream of the operands' device, nothing synchronises, workspaces
belong to the call (under capture: to the graph).
"""
import ctypes as C
from collections import namedtuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as N

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INT8_MAX_INPUTS = 131072   # of 32-bit sums of products of 8-bit integers

_FLOATS = tuple(_TYPES)

# order int32 [pairs]: pair (row * copies + copy) at every grouped row; offsets int32 [members + 1]: first grouped row of every member;
# shape: that of the member indices, (rows,) or (rows, copies)
RowGroups = namedtuple("RowGroups", "order offsets shape")
# values int8 [..., K], scale float32 [...]: the numbers values * scale[..., None]
QuantRows = namedtuple("QuantRows", "values scale")


def _gpu(t, name, dtypes):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in dtypes:
        got = f"{t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise TypeError(f"{name}: expected a GPU tensor of {' / '.join(str(d) for d in dtypes)}, got {got}")
    return t


def _same_device(dev, name, t):
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, the rows are on cuda:{dev}")


def _no_tangents(**operands):
    """Refuse operands of forward-mode differentiation (a native call reads the values alone: the derivative would come out as zero)."""
    for name, t in operands.items():
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} carries a forward-mode tangent: these layers have no forward-mode derivative")


def _run(dev, fn, *args):
    """A native call with device `dev` current (one process may drive several), on torch's current stream of it."""
    if dev == N.current_device():
        rc = fn(*args, N.stream_ptr(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, N.stream_ptr(dev))
    if rc < 0:
        N.check(rc)


def _addr(t):
    return None if t is None else t.data_ptr()


def _rows2d(t):
    """t [n, K] with its elements side by side in a row, and how many elements its rows are apart (any distance: a slice, an expanded row)."""
    (row, col), (n, k) = t.stride(), t.shape
    if (col != 1 and k > 1) or row > 1 << 28:
        t, row = t.contiguous(), k
    return t, row if n > 1 else k


def _layers(w):
    """w [G, N, K]: elements side by side along K; members and output rows any distance apart (slices of the members' flat vectors)."""
    return w if w.shape[2] <= 1 or w.stride(2) == 1 else w.contiguous()


def group_rows(member, n_members):
    """Sort (row, copy) pairs by ensemble member, stably -> RowGroups(order, offsets, shape).

    member: int32 [rows] or [rows, copies], the member(s) that evaluate each row; values outside [0, n_members) mean nobody (padding): those
    pairs come last, and the layers below give them zeros.  n_members <= 4096.  One launch up to 4096 pairs, three beyond."""
    _gpu(member, "member", (torch.int32,))
    shape = tuple(member.shape)
    if len(shape) not in (1, 2):
        raise ValueError("member must be [rows] or [rows, copies]")
    n_members = int(n_members)
    if not 1 <= n_members <= 4096:
        raise ValueError("n_members must lie in 1 .. 4096")
    if len(shape) == 2 and shape[1] < 1:
        raise ValueError("member must hold at least one copy per row")
    P = member.numel()
    if P >= 1 << 30:
        raise ValueError("rows x copies must stay below 2^30")
    m = member.contiguous()
    order = m.new_empty(P)
    offsets = m.new_empty(n_members + 1)
    nbytes = 0 if P <= 4096 else N.lib().bnn_group_rows_workspace_bytes(P, n_members)
    ws = m.new_empty(nbytes // 4) if nbytes else None
    _run(m.get_device(), N.lib().bnn_group_rows_i32, m.data_ptr(), P, n_members, order.data_ptr(), offsets.data_ptr(), _addr(ws))
    return RowGroups(order, offsets, shape)


def _check_groups(groups, x, G, gather, what="x"):
    """-> (rows, copies) of the groups, after checking them against the row operand."""
    if not isinstance(groups, RowGroups):
        raise TypeError("groups must be the RowGroups that group_rows returns")
    order, offsets, shape = groups
    dev = x.get_device()
    if len(shape) == 2:
        rows, copies = shape
    elif len(shape) == 1:
        rows, copies = shape[0], 1
    else:
        raise ValueError("groups.shape must be (rows,) or (rows, copies)")
    try:   # at every call, also of what group_rows made: a named tuple is easily rebuilt around other tensors, and the kernels trust these
        fit = (order.dtype is torch.int32 and offsets.dtype is torch.int32 and order.get_device() == dev and offsets.get_device() == dev
               and order.numel() == rows * copies and order.is_contiguous() and offsets.is_contiguous())
    except AttributeError:
        fit = False
    if not fit:
        for name, t in (("groups.order", order), ("groups.offsets", offsets)):
            if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.device.type != x.device.type:
                raise TypeError(f"{name}: expected a torch.int32 tensor on the rows' device, got " + (f"{t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__))
            _same_device(dev, name, t)
        raise ValueError("groups.order must be contiguous and hold one entry per (row, copy) pair, groups.offsets contiguous")
    if offsets.numel() != G + 1:
        raise ValueError(f"groups are over {offsets.numel() - 1} members, the weights over {G}")
    want = rows if gather else rows * copies
    if x.shape[0] != want:
        raise ValueError(f"{what} must have {want} rows ({'the batch' if gather else 'one per grouped pair'}), got {x.shape[0]}")
    return rows, copies


def _out_shape(groups, pairs, n_out, scatter):
    return (*groups.shape, n_out) if scatter else (pairs, n_out)


def _check_linear(x, weight, groups, bias, gather):
    if forward_ad._current_level >= 0:   # (inside a dual_level; outside of one there are no tangents)
        _no_tangents(x=x, weight=weight, bias=bias)
    _gpu(x, "x", _FLOATS)
    dtype, dev = x.dtype, x.get_device()
    _gpu(weight, "weight", (dtype,))
    G, n_out, n_in = weight.shape if weight.dim() == 3 else (0, 0, 0)
    if x.dim() != 2 or n_in != x.shape[1] or G < 1 or n_out < 1 or n_in < 1:
        raise ValueError("x must be [rows, K] and weight [members, N, K]")
    if max(G, n_out, n_in) > 1 << 24:
        raise ValueError("members, inputs and outputs must stay below 2^24")
    _same_device(dev, "weight", weight)
    if bias is not None:
        _gpu(bias, "bias", (dtype,))
        if bias.shape != (G, n_out):
            raise ValueError(f"bias must be [{G}, {n_out}]")
        _same_device(dev, "bias", bias)
    return _check_groups(groups, x, G, gather)


def _descriptor(groups, rows, copies, dtype, weight, x_row, y_row, gather, scatter, relu=False):
    G, n_out, n_in = weight.shape
    member, row, _ = weight.stride()
    return N.BnnGrouped(rows, copies, G, n_in, n_out, _TYPES[dtype], 1 if gather else 0, 1 if scatter else 0, 1 if relu else 0, x_row, y_row,
                        member if G > 1 else 0, row if n_out > 1 else n_in, groups.order.data_ptr(), groups.offsets.data_ptr())


def _linear(x, weight, groups, bias, relu, gather, scatter, rows, copies):
    (x, x_row), weight = _rows2d(x), _layers(weight)
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    n_out = weight.shape[1]
    y = x.new_empty(_out_shape(groups, rows * copies, n_out, scatter))
    q = _descriptor(groups, rows, copies, x.dtype, weight, x_row, n_out, gather, scatter, relu)
    _run(x.get_device(), N.lib().bnn_grouped_linear, q, x.data_ptr(), weight.data_ptr(), _addr(bias), y.data_ptr())
    return y


def grouped_linear_grads(dy, x, weight, groups, y=None, gather=False, scatter=False, need=(True, True, True)):
    """Gradients of grouped_linear -> (dx, dweight, dbias), each None where `need` says so.

    dy: gradient of the layer's output, in its shape; y: that output, for a layer with relu=True (no gradient where y <= 0; a NaN output passes it, as in
    nn.ReLU), else None.
    A plain function without autograd: what grouped_linear's backward calls, and what a captured HIP graph of a training step may call.
    dweight and dbias of a member without rows are zero; sums are fp32 and do not depend on timing.
    Memory for the call: with gather and several copies dx takes rows x copies x K floats (a row's gradients meet in fp32), with y a masked copy of dy, and
    dbias is computed along with dweight."""
    if forward_ad._current_level >= 0:
        _no_tangents(dy=dy, y=y)
    rows, copies = _check_linear(x, weight, groups, None, gather)
    G, n_out, n_in = weight.shape
    shape = _out_shape(groups, rows * copies, n_out, scatter)
    dev = x.get_device()
    for name, t in (("dy", dy),) if y is None else (("dy", dy), ("y", y)):
        _gpu(t, name, (x.dtype,))
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must be {list(shape)}")
        _same_device(dev, name, t)
    (x, x_row), weight = _rows2d(x), _layers(weight)
    dy, dy_row = _rows2d(dy.reshape(-1, n_out))
    need_x, need_w, need_b = need
    L = N.lib()
    if y is not None:
        y2, y_row = _rows2d(y.reshape(-1, n_out))
        masked = x.new_empty((dy.shape[0], n_out))
        _run(dev, L.bnn_relu_grad, dy.data_ptr(), dy_row, y2.data_ptr(), y_row, dy.shape[0], n_out, _TYPES[x.dtype], masked.data_ptr())
        dy, dy_row = masked, n_out
    dx = dw = db = None
    if need_x:
        dx = x.new_empty((x.shape[0], n_in))
        q = _descriptor(groups, rows, copies, x.dtype, weight, n_in, dy_row, gather, scatter)
        nbytes = L.bnn_grouped_linear_dx_workspace_bytes(q)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        _run(dev, L.bnn_grouped_linear_dx, q, dy.data_ptr(), weight.data_ptr(), dx.data_ptr(), _addr(ws))
    if need_w or need_b:
        dw = x.new_empty((G, n_out, n_in))
        db = x.new_empty((G, n_out)) if need_b else None
        q = _descriptor(groups, rows, copies, x.dtype, weight, x_row, dy_row, gather, scatter)
        nbytes = L.bnn_grouped_linear_dw_workspace_bytes(q)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        _run(dev, L.bnn_grouped_linear_dw, q, dy.data_ptr(), x.data_ptr(), dw.data_ptr(), _addr(db), _addr(ws))
    return dx, dw if need_w else None, db


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, relu, gather, scatter, rows, copies):
        y = _linear(x, weight, groups, bias, relu, gather, scatter, rows, copies)
        ctx.save_for_backward(x, weight, groups.order, groups.offsets, y if relu else None)
        ctx.shape, ctx.gather, ctx.scatter = groups.shape, gather, scatter
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, order, offsets, y = ctx.saved_tensors
        dx, dw, db = grouped_linear_grads(dy, x, weight, RowGroups(order, offsets, ctx.shape), y, ctx.gather, ctx.scatter,
                                          need=ctx.needs_input_grad[:3])
        return dx, dw, db, None, None, None, None, None, None


def grouped_linear(x, weight, groups, bias=None, relu=False, gather=False, scatter=False):
    """y = act(W[m] x + b[m]) for every row of every member m's group; differentiable in x, weight and bias (once).

    x [rows, K] float32 / bfloat16 / float16; weight [members, N, K] and bias [members, N] of the same type; groups: group_rows(...).
    gather=True: x holds the batch's rows, each read by the member(s) its indices name; False: x [pairs, K] is already in grouped order.
    scatter=True: y comes in the batch's order, [rows, N] or [rows, copies, N]; False: in grouped order, [pairs, N] -- so a chain of layers
    gathers in the first, scatters in the last and permutes nothing in between.  Rows of nobody: zero.
    Under stream capture call it in torch.no_grad() (a captured training step: grouped_linear_grads for its backward pass).
    Forward-mode derivatives are refused.
    x and weight may be strided as long as the elements along K are neighbours (a layer's slice of flat parameter vectors [members, d]).
    Sums are fp32 (float32 operands: exact fp32 products), rounded once to the operands' type."""
    rows, copies = _check_linear(x, weight, groups, bias, gather)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("grouped_linear records no autograd graph under stream capture: autograd would join the capture with the streams of "
                               "earlier graphs of the same leaves.  Capture it under torch.no_grad() with grouped_linear_grads as the backward pass")
        return _GroupedLinear.apply(x, weight, bias, groups, relu, gather, scatter, rows, copies)
    return _linear(x, weight, groups, bias, relu, gather, scatter, rows, copies)


def _check_quantize(x):
    if forward_ad._current_level >= 0:
        _no_tangents(x=x)
    _gpu(x, "x", _FLOATS)
    K = x.shape[-1] if x.dim() else 0
    if K < 1:
        raise ValueError("x must be [..., K] with K >= 1")
    if K > 1 << 24 or x.numel() >= K << 31:
        raise ValueError("rows must stay below 2^31, their length below 2^24")
    if x.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("8-bit rows have no gradient: detach x")


def quantize_rows(x):
    """Rows to 8-bit integers -> QuantRows(values int8 [..., K], scale float32 [...]): scale = max |x| / 127 of the row (a token, or an output
    channel of a weight [N, K] / [members, N, K]), values = x / scale rounded half to even, exactly.  A row of zeros has scale 0; a row that holds
    NaN or an infinity has scale NaN, so that whatever is computed from it is NaN."""
    _check_quantize(x)
    shape = x.shape
    K = shape[-1]
    x2, x_row = _rows2d(x if len(shape) == 2 else x.reshape(-1, K))
    values = torch.empty(shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    _run(x.get_device(), N.lib().bnn_quantize_rows, x2.data_ptr(), _TYPES[x.dtype], x2.shape[0], K, x_row, values.data_ptr(), K, scale.data_ptr())
    return QuantRows(values, scale)


def int8_linear(x, weight, groups=None, bias=None, relu=False, gather=False, scatter=False, dtype=None):
    """The linear layer on 8-bit operands with a scale per row and per output channel; integer sums are exact.

    x [rows, K]: float rows (quantised here: quantize_rows) or QuantRows made earlier; weight: QuantRows of [N, K] (one matrix; groups=None) or of
    [members, N, K] with groups / gather / scatter as in grouped_linear.  bias [N] or [members, N] in the output's type `dtype` (default: x's
    type; float32 for QuantRows).  Inference only: operands that require a gradient are refused under grad mode.  K <= 131072."""
    quant = isinstance(x, QuantRows)
    if forward_ad._current_level >= 0:
        for name, t in (("x", x), ("weight", weight)):
            if isinstance(t, QuantRows):
                _no_tangents(**{f"{name}.scale": t.scale})
        _no_tangents(bias=bias)
    if quant:
        rows_of, xs = _gpu(x.values, "x.values", (torch.int8,)), _gpu(x.scale, "x.scale", (torch.float32,))
    else:
        _check_quantize(x)
        rows_of = x
    dtype = dtype or (torch.float32 if quant else x.dtype)
    if dtype not in _TYPES:
        raise TypeError(f"dtype must be one of {[str(d) for d in _TYPES]}")
    if not isinstance(weight, QuantRows):
        raise TypeError("weight must be the QuantRows that quantize_rows returns")
    wq, ws = _gpu(weight.values, "weight.values", (torch.int8,)), _gpu(weight.scale, "weight.scale", (torch.float32,))
    shape = wq.shape
    if len(shape) != (2 if groups is None else 3) or rows_of.dim() != 2 or shape[-1] != rows_of.shape[1] or min(shape) < 1:
        raise ValueError("x must be [rows, K], weight [N, K] without groups or [members, N, K] with them")
    if wq.stride(-1) != 1 and shape[-1] > 1:
        wq = wq.contiguous()
    if groups is None:
        (n_out, n_in), G, strides = shape, 1, (0, wq.stride(0))
    else:
        (G, n_out, n_in), strides = shape, wq.stride()
    if n_in > _INT8_MAX_INPUTS:
        raise ValueError(f"K must not exceed {_INT8_MAX_INPUTS}: the sums are 32-bit integers")
    if G > 1 << 24 or n_out > 1 << 24:
        raise ValueError("members and outputs must stay below 2^24")
    if torch.is_grad_enabled() and (ws.requires_grad or (quant and xs.requires_grad)):
        raise NotImplementedError(f"the 8-bit layer has no gradient: detach {'weight' if ws.requires_grad else 'x'}.scale")
    if ws.shape != shape[:-1] or (quant and xs.shape != rows_of.shape[:1]):
        raise ValueError("scales must have their values' shape without the last dimension")
    dev = rows_of.get_device()
    _same_device(dev, "weight.values", wq)
    _same_device(dev, "weight.scale", ws)
    if bias is not None:
        _gpu(bias, "bias", (dtype,))
        if bias.shape != shape[:-1]:
            raise ValueError(f"bias must be {list(shape[:-1])}")
        if bias.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("the 8-bit layer has no gradient: detach bias")
        _same_device(dev, "bias", bias)
        bias = bias.contiguous()
    if groups is None:
        if gather or scatter:
            raise ValueError("gather / scatter need groups")
        rows, copies, order, offsets = rows_of.shape[0], 1, None, None
        if rows >= 1 << 30:
            raise ValueError("rows must stay below 2^30")
        out = (rows, n_out)
    else:
        rows, copies = _check_groups(groups, rows_of, G, gather)
        order, offsets = groups.order.data_ptr(), groups.offsets.data_ptr()
        out = _out_shape(groups, rows * copies, n_out, scatter)
    (rows_of, x_row), ws = _rows2d(rows_of), ws.contiguous()
    y = rows_of.new_empty(out, dtype=dtype)
    q = N.BnnGrouped(rows, copies, G, n_in, n_out, _TYPES[dtype], 1 if gather else 0, 1 if scatter else 0, 1 if relu else 0, x_row, n_out,
                     strides[0] if G > 1 else 0, strides[1] if n_out > 1 else n_in, order, offsets)
    if quant:
        _same_device(dev, "x.scale", xs)
        xs = xs.contiguous()
        _run(dev, N.lib().bnn_int8_linear, q, rows_of.data_ptr(), xs.data_ptr(), wq.data_ptr(), ws.data_ptr(), _addr(bias), y.data_ptr())
    else:
        space = rows_of.new_empty(max(int8_rows_workspace(rows_of.shape[0], n_in), 1), dtype=torch.uint8)
        _run(dev, N.lib().bnn_int8_linear_rows, q, rows_of.data_ptr(), _TYPES[rows_of.dtype], space.data_ptr(), wq.data_ptr(), ws.data_ptr(), _addr(bias), y.data_ptr())
    return y


def int8_rows_workspace(rows, n_in):
    """Bytes that the codes and scales of `rows` rows take (bnn_int8_linear_rows_workspace_bytes, without the call)."""
    return rows * (-(-n_in // 16) * 16 + 4)
