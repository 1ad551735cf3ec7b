"""GPU: the calls of the linear layers over row groups that their documentation allows and that go wrong easily.

Bounds as in test_member_linear.py: a sum of n products in fp32 is off by at most (n + 1) 2^-23 sum |a b|, and one rounding to the output's type by half a
step."""
import numpy as np
import pytest
import torch

from test_member_linear import INT8_SLACK, _gen, int8_plain, make, ops  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- altered groups --------------------------------------------------------------------------------------------------------------------------
def test_altered_groups_are_refused_before_a_launch(ops):
    m, x, w, b = make(300, 3, 0, 24, 16, torch.float32, True)
    gr = ops.group_rows(m, 3)
    wq = ops.quantize_rows(w)
    dy = torch.ones(300, 16, device="cuda")
    longer = x.repeat(2, 1)
    for bad, rows, error in ((gr._replace(shape=(600,)), longer, ValueError), (gr._replace(offsets=gr.offsets.cpu()), x, TypeError), (gr._replace(order=gr.order.cpu()), x, TypeError),
                             (gr._replace(order=gr.order.long()), x, TypeError), (gr._replace(offsets=gr.offsets.long()), x, TypeError),
                             (gr._replace(order=gr.order.repeat_interleave(2)[::2]), x, ValueError), (gr._replace(offsets=gr.offsets.repeat_interleave(2)[::2]), x, ValueError)):
        with pytest.raises(error):
            ops.grouped_linear(rows, w, bad, bias=b, gather=True, scatter=True)
        with pytest.raises(error):
            ops.grouped_linear_grads(dy, rows, w, bad, gather=True, scatter=True)
        with pytest.raises(error):
            ops.int8_linear(rows, wq, groups=bad, bias=b, gather=True, scatter=True)
    same = gr._replace(shape=(300, 1))
    assert torch.equal(ops.grouped_linear(x, w, same, bias=b, gather=True, scatter=True)[:, 0], ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True))


# ---- forward-mode derivatives ------------------------------------------------------------------------------------------------------------------
def test_operands_with_a_tangent_are_refused(ops):
    from torch.autograd import forward_ad
    m, x, w, b = make(300, 3, 0, 24, 16, torch.float32, True)
    gr = ops.group_rows(m, 3)
    want = ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
    with forward_ad.dual_level():
        for i in range(3):
            for grad in (False, True):       # a dual tensor requires no gradient by itself
                t = [a.clone() for a in (x, w, b)]
                t[i] = forward_ad.make_dual(t[i].requires_grad_(grad), torch.ones_like(t[i]))
                with pytest.raises(NotImplementedError):
                    ops.grouped_linear(t[0], t[1], gr, bias=t[2], gather=True, scatter=True)
        leaf = x.clone().requires_grad_(True)
        y = ops.grouped_linear(leaf, w, gr, bias=b, gather=True, scatter=True)
        with pytest.raises(NotImplementedError):   # forward over reverse
            torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
        assert torch.equal(ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True), want)
    assert torch.equal(ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True), want)


# ---- 8 bits: no gradient is lost -----------------------------------------------------------------------------------------------------------------
def test_8_bit_operands_that_require_a_gradient_are_refused(ops):
    m, x, w, b = make(40, 3, 0, 24, 16, torch.float32, True)
    gr, xq, wq = ops.group_rows(m, 3), ops.quantize_rows(x), ops.quantize_rows(w)
    f = lambda xx, ww, bb: ops.int8_linear(xx, ww, groups=gr, bias=bb, gather=True, scatter=True)
    leaf = lambda t: t.clone().requires_grad_(True)
    for args in ((xq._replace(scale=leaf(xq.scale)), wq, b), (xq, wq._replace(scale=leaf(wq.scale)), b), (x, wq._replace(scale=leaf(wq.scale)), b), (leaf(x), wq, b), (xq, wq, leaf(b))):
        with pytest.raises(NotImplementedError, match="no gradient"):
            f(*args)
        with torch.no_grad():
            assert torch.equal(f(*args), f(xq, wq, b))
    dense = ops.QuantRows(wq.values[0], leaf(wq.scale[0]))
    with pytest.raises(NotImplementedError, match="weight.scale"):
        ops.int8_linear(x, dense)


# ---- 8 bits: the largest sum -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("K", [131072, 131071, 131056, 131057])
@pytest.mark.parametrize("n,N", [(3, 20), (3, 600), (200, 40), (200, 2048), (1100, 2050)])
def test_sums_of_the_lowest_code(ops, n, N, K):
    """Codes that a caller brings may be -128, which quantize_rows never gives: 2^17 products of two of them are 2^31.  Exact: a sum is
    rounded once, to a float32."""
    one = lambda k: torch.ones(k, device="cuda")
    q = torch.full((n, K), -128, dtype=torch.int8, device="cuda")
    w = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    w[N // 2:] = 127
    q[n // 2:] = 127
    y = ops.int8_linear(ops.QuantRows(q, one(n)), ops.QuantRows(w, one(N)))
    f = lambda a, b: float(np.float32(a * b * K))
    assert (y[:n // 2, :N // 2] == f(-128, -128)).all() and (y[:n // 2, N // 2:] == f(-128, 127)).all()
    assert (y[n // 2:, :N // 2] == f(127, -128)).all() and (y[n // 2:, N // 2:] == f(127, 127)).all()


# ---- 8 bits: rows of nobody ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,G,K,N", [(20, 3, 41, 40), (40, 1, 4096, 80), (300, 3, 256, 64), (3000, 9, 41, 40), (3000, 9, 61, 130), (4000, 2, 255, 200), (3000, 3, 511, 96), (700, 3, 2048, 2048)])
def test_rows_of_nobody_are_zero_next_to_weights_that_are_not_finite(ops, n, G, K, N):
    """A NaN in a channel of any member's matrix makes that output of the member's own rows NaN, and nothing else."""
    m, x, w, b = make(n, G, 0, K, N, torch.float32, True, seed=n + K)
    m[::7] = -1
    gr = ops.group_rows(m, G)
    clean = ops.int8_linear(x, ops.quantize_rows(w), groups=gr, bias=b, gather=True, scatter=True)
    for g in (0, G - 1):
        bad = w.clone()
        bad[g, ::5, 3] = float("nan")
        for relu in (False, True):
            y = ops.int8_linear(x, ops.quantize_rows(bad), groups=gr, bias=b, relu=relu, gather=True, scatter=True)
            want = clean.clamp_min(0) if relu else clean.clone()
            want[(m == g)[:, None] & (torch.arange(N, device="cuda") % 5 == 0)] = float("nan")
            assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y.nan_to_num(7.0), want.nan_to_num(7.0))
            assert (y[m < 0] == 0).all()


# ---- 8 bits: scales whose product no float holds -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,K,N", [(3, 4096, 20), (20, 200, 600), (3000, 41, 40), (3000, 201, 130), (300, 512, 64), (3000, 640, 384), (3001, 641, 383), (16384, 512, 4096), (16384, 513, 4095)])
@pytest.mark.parametrize("a,b", [(-22, -20), (-40, -4), (-20, -24), (30, 9), (5, 34), (38, -38), (-44, 30)])
def test_scales_whose_product_no_float_holds(ops, n, K, N, a, b):
    """The sum times the scales in 64 bits: where it is a float, the output is that float to four roundings (and half the smallest subnormal) although the
    scales' product under- or overflows; a sum of zero is zero, a result beyond the floats infinite.  Ready codes, and (rows of few inputs and many) float rows."""
    g = _gen(n + K)
    q = torch.randint(-127, 128, (n, K), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    q[::5] = 0                                    # sums of zero
    w[::7] = 0
    s = (0.5 + torch.rand(n, generator=g, device="cuda", dtype=torch.float64)).mul(10.0 ** a).float()
    ws = (0.5 + torch.rand(N, generator=g, device="cuda", dtype=torch.float64)).mul(10.0 ** b).float()
    assert torch.isfinite(s).all() and torch.isfinite(ws).all()
    cases = [(ops.QuantRows(q, s), q, s)]
    x = (q.double() * s.double()[:, None]).float()
    if torch.isfinite(x).all():
        cases.append((x, *ops.quantize_rows(x)))
    top = float(torch.finfo(torch.float32).max)
    for rows, codes, scale in cases:
        for relu in (False, True):
            y = ops.int8_linear(rows, ops.QuantRows(w, ws), relu=relu)
            want, _ = int8_plain(codes, scale, w, ws, None)
            if relu:
                want = want.clamp_min(0)
            sure = want.abs() * (1 + INT8_SLACK) < top
            assert (y[want == 0] == 0).all()
            assert ((y.double() - want).abs()[sure] <= (INT8_SLACK * want.abs() + 2.0 ** -149)[sure]).all()
            assert torch.isinf(y[want.abs() * (1 - INT8_SLACK) > top]).all() and (torch.sign(y.double()) == torch.sign(want))[~sure].all()
