"""GPU: every kernel form of the linear layers over row groups against the formula in 64 bits -- forward, gradients and 8 bits, with ReLU, rows in the batch's
and in the members' order, even members and very uneven ones.  test_member_linear_checks_cpu.py asserts that the sizes below reach every form.

Bounds as in test_member_linear.py."""
import numpy as np
import pytest
import torch

from test_member_linear import DT, INT8_SLACK, _gen, int8_plain, make, ops, pair_view, within  # noqa: F401

pytestmark = pytest.mark.gpu

# rows, members, copies, inputs, outputs
SIZES = [(84, 1, 3, 21, 337), (70, 1, 3, 608, 320), (267, 1, 0, 41, 563), (882, 2, 0, 88, 632), (3555, 16, 0, 1560, 10), (20098, 100, 0, 160, 16), (10, 8, 0, 18, 9),
         (8, 64, 0, 16, 16), (16, 2, 2, 23, 9), (32, 2, 0, 16, 16), (39, 1, 2, 22, 9), (9, 100, 0, 16, 928), (65, 64, 0, 18, 140), (22970, 100, 3, 19, 131), (5347, 64, 3, 336, 304),
         (68, 1, 0, 33, 14), (44, 1, 2, 65, 12), (13620, 100, 0, 225, 331), (10947, 3, 3, 76, 441), (1622, 30, 2, 34, 3475), (16346, 1, 0, 304, 800), (102, 1, 0, 50, 9),
         (33, 1, 2, 146, 8), (39, 1, 2, 107, 11), (62, 1, 2, 252, 10), (87, 1, 0, 56, 86), (42, 1, 2, 94, 69), (45, 2, 3, 103, 74), (34, 1, 3, 189, 67), (24, 30, 0, 615, 1361),
         (10980, 8, 0, 1120, 368), (10197, 100, 2, 648, 155), (6334, 2, 3, 768, 448), (4383, 100, 3, 54, 803), (39518, 100, 0, 117, 287), (7369, 100, 0, 142, 1638),
         (6895, 100, 0, 211, 1319), (140000, 1, 0, 41, 9), (70, 1, 0, 9, 12), (80, 1, 0, 13, 70), (6001, 30, 2, 15, 1303)]


def uneven(m, G, seed):
    """Nine rows in ten to the last member."""
    m[torch.rand(m.shape, generator=_gen(seed + 5), device="cuda") < 0.9] = G - 1
    return m


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,G,copies,K,N", SIZES)
def test_every_form(ops, n, G, copies, K, N, dtype):
    for moved, relu, skew in ((True, True, False), (False, False, True)):
        m, x, w, b = make(n, G, copies, K, N, DT[dtype], moved, seed=n + N)
        if skew:
            m = uneven(m, G, n)
        gr = ops.group_rows(m, G)
        xi, yi, mem = pair_view(gr, m, moved, moved)
        P = m.numel()
        y = ops.grouped_linear(x, w, gr, bias=b, relu=relu, gather=moved, scatter=moved)
        dy = torch.randn(y.shape, generator=_gen(n + 1), device="cuda").to(x.dtype)
        dx, dw, db = ops.grouped_linear_grads(dy, x, w, gr, y=y if relu else None, gather=moved, scatter=moved)
        wq, (q, s) = ops.quantize_rows(w), ops.quantize_rows(x)
        y8 = ops.int8_linear(ops.QuantRows(q, s), wq, groups=gr, bias=b, relu=relu, gather=moved, scatter=moved, dtype=x.dtype)
        assert torch.equal(ops.int8_linear(x, wq, groups=gr, bias=b, relu=relu, gather=moved, scatter=moved), y8)
        y, y8, d = y.reshape(-1, N), y8.reshape(-1, N), dy.double().reshape(-1, N)
        if relu:
            d = d * (y > 0)
        act = (lambda t: t.clamp_min(0)) if relu else (lambda t: t)
        seen = torch.zeros(P, dtype=torch.bool, device="cuda")
        wx, mx = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
        for g in range(G):
            sel = np.nonzero(mem == g)[0]
            a, t = torch.as_tensor(xi[sel], device="cuda"), torch.as_tensor(yi[sel], device="cuda")
            xg, wg, bg, dg = x[a].double(), w[g].double(), b[g].double(), d[t]
            seen[t] = True
            within(y[t], act(xg @ wg.t() + bg), (K + 2) * 2.0 ** -23 * (xg.abs() @ wg.abs().t() + bg.abs()))
            want, mag = int8_plain(q[a], s[a], wq.values[g], wq.scale[g], b[g])
            within(y8[t], act(want), INT8_SLACK * mag)
            within(dw[g], dg.t() @ xg, (sel.size + 2) * 2.0 ** -23 * (dg.abs().t() @ xg.abs()))
            within(db[g], dg.sum(0), (sel.size + 2) * 2.0 ** -23 * dg.abs().sum(0))
            wx.index_add_(0, a, dg @ wg)
            mx.index_add_(0, a, dg.abs() @ wg.abs())
        within(dx, wx, (N * max(copies, 1) + 2) * 2.0 ** -23 * mx)
        assert (y[~seen] == 0).all() and (y8[~seen] == 0).all()
