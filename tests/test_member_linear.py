"""GPU: rows sorted by member, the grouped linear layer with its gradients and its 8-bit form, against plain formulas in 64 bits.

Bounds.  A sum of n products in fp32, in any order, is off by at most (n + 1) u sum |a b| with u = 2^-24; the matrix pipe may round a step by
truncation, which doubles u.  The result is rounded once to the output's type: half a step, eps / 2 of the value (plus half the smallest
subnormal of fp16).  A bias adds one rounding."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from bnn_chaos_model_amd import ops
    return ops


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def members(n, G, copies=0, seed=0, nobody=True):
    g = _gen(seed + 77)
    m = torch.randint(-1 if nobody else 0, G, (n, max(copies, 1)), generator=g, device="cuda", dtype=torch.int32)
    if G > 3:
        m[m == 2] = 1                          # a member without rows
    return m if copies else m[:, 0].contiguous()


def within(got, want, slack):
    """|got - want| <= slack + half a step of got's type at that value."""
    got64 = got.double()
    half = torch.finfo(got.dtype).eps / 2
    bound = slack + half * (want.abs() + slack) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    bad = ~((got64 - want).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond the bound, worst {float((got64 - want).abs().max())}"


def pair_view(groups, member, gather, scatter):
    """(x row, y row, member) of every grouped row, from the definition."""
    m = member.reshape(-1).cpu().numpy()
    G = groups.offsets.numel() - 1
    key = np.where((m < 0) | (m >= G), G, m)
    order = np.argsort(key, kind="stable")
    copies = member.shape[1] if member.dim() == 2 else 1
    r = np.arange(m.size)
    return order // copies if gather else r, order if scatter else r, key[order]


def plain(x, w, b, xi, yi, mem, rows_out):
    """y and sum |x w| + |b| in 64 bits, [rows_out, N]."""
    x, w = x.double(), w.double()
    y = torch.zeros(rows_out, w.shape[1], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    for g in range(w.shape[0]):
        sel = np.nonzero(mem == g)[0]
        if sel.size == 0:
            continue
        a = x[torch.as_tensor(xi[sel], device=x.device)]
        t = torch.as_tensor(yi[sel], device=x.device)
        y[t] = a @ w[g].t() + (0 if b is None else b[g].double())
        mag[t] = a.abs() @ w[g].abs().t() + (0 if b is None else b[g].double().abs())
    return y, mag


# ---- group_rows --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,G,copies", [(0, 3, 0), (1, 1, 0), (1, 30, 0), (63, 30, 0), (64, 2, 2), (65, 7, 3), (4096, 30, 0), (4097, 30, 0), (8192, 30, 0), (8193, 30, 0), (50001, 1023, 0),
                                        (50001, 1024, 2), (20000, 4096, 0), (300007, 30, 4), (1000000, 1, 0)])
def test_group_rows_is_the_stable_sort(ops, n, G, copies):
    m = members(n, G, copies, seed=n)
    gr = ops.group_rows(m, G)
    key = m.reshape(-1).cpu().numpy()
    key = np.where((key < 0) | (key >= G), G, key)
    assert np.array_equal(gr.order.cpu().numpy(), np.argsort(key, kind="stable"))
    assert np.array_equal(gr.offsets.cpu().numpy(), np.searchsorted(np.sort(key), np.arange(G + 1)))
    assert gr.order.dtype == gr.offsets.dtype == torch.int32 and gr.shape == tuple(m.shape)


def test_group_rows_members_out_of_range_and_strided(ops):
    m = torch.tensor([5, -2147483648, 2147483647, 0, 4, -1, 5, 3], dtype=torch.int32, device="cuda")
    gr = ops.group_rows(m, 5)
    assert gr.order.tolist() == [3, 7, 4, 0, 1, 2, 5, 6] and gr.offsets.tolist() == [0, 1, 1, 1, 2, 3]
    wide = torch.zeros(8, 3, dtype=torch.int32, device="cuda")
    wide[:, 1] = m
    assert torch.equal(ops.group_rows(wide[:, 1], 5).order, gr.order)


# ---- the layer -----------------------------------------------------------------------------------------------------------------------------
SHAPES = [  # rows, members, copies, K, N
    (1, 1, 0, 1, 1), (1, 30, 0, 40, 40), (15, 30, 0, 40, 40), (17, 3, 2, 41, 40), (64, 1, 0, 64, 64), (65, 2, 0, 65, 63), (300, 5, 0, 128, 128),
    (257, 70, 0, 96, 130), (1000, 4, 3, 41, 128), (2000, 3, 0, 264, 520), (700, 2, 0, 512, 384), (3, 2, 0, 1000, 8), (130, 9, 4, 7, 3),
    (5000, 2, 0, 16, 1024), (40, 4, 0, 4096, 48)]


def make(n, G, copies, K, N, dt, gather, seed=1, nobody=True):
    g = _gen(seed)
    m = members(n, G, copies, seed, nobody)
    rows = n if gather else m.numel()
    x = torch.randn(rows, K, generator=g, device="cuda").to(dt)
    w = (torch.randn(G, N, K, generator=g, device="cuda") / K ** 0.5).to(dt)
    b = torch.randn(G, N, generator=g, device="cuda").to(dt)
    return m, x, w, b


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,G,copies,K,N", SHAPES)
def test_grouped_linear(ops, n, G, copies, K, N, dtype):
    for gather, scatter, relu, bias in ((True, True, True, True), (False, False, False, False), (True, False, False, True), (False, True, True, False)):
        m, x, w, b = make(n, G, copies, K, N, DT[dtype], gather, seed=n + K)
        gr = ops.group_rows(m, G)
        y = ops.grouped_linear(x, w, gr, bias=b if bias else None, relu=relu, gather=gather, scatter=scatter)
        assert tuple(y.shape) == ((*m.shape, N) if scatter else (m.numel(), N)) and y.dtype == x.dtype
        xi, yi, mem = pair_view(gr, m, gather, scatter)
        want, mag = plain(x, w, b if bias else None, xi, yi, mem, m.numel())
        if relu:
            want = want.clamp_min(0)
        within(y.reshape(-1, N), want, (K + 2) * 2.0 ** -23 * mag)
        nobody = torch.as_tensor(yi[mem == G], device="cuda")
        assert (y.reshape(-1, N)[nobody] == 0).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,G,copies,K,N", SHAPES)
def test_grouped_linear_grads(ops, n, G, copies, K, N, dtype):
    for gather, scatter, relu in ((True, True, False), (False, False, True), (True, False, True), (False, True, False)):
        m, x, w, b = make(n, G, copies, K, N, DT[dtype], gather, seed=n + N)
        gr = ops.group_rows(m, G)
        for t in (x, w, b):
            t.requires_grad_(True)
        y = ops.grouped_linear(x, w, gr, bias=b, relu=relu, gather=gather, scatter=scatter)
        dy = torch.randn(y.shape, generator=_gen(n + 5), device="cuda").to(x.dtype)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        d = dy.double().reshape(-1, N) * ((y.detach().reshape(-1, N) > 0) if relu else 1)
        xi, yi, mem = pair_view(gr, m, gather, scatter)
        wx, ww, wb = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(w, dtype=torch.float64), torch.zeros_like(b, dtype=torch.float64)
        mx, mw, mb = torch.zeros_like(wx), torch.zeros_like(ww), torch.zeros_like(wb)
        most = 0
        for g in range(G):
            sel = np.nonzero(mem == g)[0]
            most = max(most, sel.size)
            a, t = torch.as_tensor(xi[sel], device="cuda"), torch.as_tensor(yi[sel], device="cuda")
            wx.index_add_(0, a, d[t] @ w[g].double())
            mx.index_add_(0, a, d[t].abs() @ w[g].double().abs())
            ww[g], mw[g] = d[t].t() @ x[a].double(), d[t].abs().t() @ x[a].double().abs()
            wb[g], mb[g] = d[t].sum(0), d[t].abs().sum(0)
        assert dx.dtype == dw.dtype == db.dtype == x.dtype
        within(dx, wx, (N * max(copies, 1) + 2) * 2.0 ** -23 * mx)
        within(dw, ww, (most + 2) * 2.0 ** -23 * mw)
        within(db, wb, (most + 2) * 2.0 ** -23 * mb)
        only = ops.grouped_linear_grads(dy, x.detach(), w.detach(), gr, y=y.detach() if relu else None, gather=gather, scatter=scatter, need=(False, True, False))
        assert only[0] is None and only[2] is None and torch.equal(only[1], dw)


# Sizes at which each kernel form is the one chosen: tiles of 256 (with members whose last tile is a half one), 128 and 64, rows that can and cannot be
# loaded straight into LDS, few rows a member, short rows, and for dW tiles of 256, 128 and 64 with and without row splits.
FORMS = [(4000, 3, 264, 4096), (4001, 3, 263, 4095), (5000, 2, 264, 1024), (5001, 2, 263, 1022), (3000, 30, 64, 128), (700, 3, 2048, 2048), (701, 3, 2047, 2050),
         (900, 3, 1024, 1024), (901, 3, 1023, 1021), (90, 2, 512, 512), (40, 1, 4096, 80), (5, 4, 2000, 200), (6, 4, 2001, 201), (4000, 9, 17, 130), (4000, 9, 41, 40),
         (3000, 2, 9, 70), (3000, 2, 61, 200), (3001, 1, 4096, 264), (9000, 1, 72, 136)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,G,K,N", FORMS)
def test_every_form_of_the_layer(ops, n, G, K, N, dtype):
    """Forward, gradients (rows in the members' order and through the order) and the 8-bit layer at the sizes above."""
    for moved in (True, False):
        m, x, w, b = make(n, G, 0, K, N, DT[dtype], moved, seed=n + N)
        gr = ops.group_rows(m, G)
        xi, yi, mem = pair_view(gr, m, moved, moved)
        y = ops.grouped_linear(x, w, gr, bias=b, gather=moved, scatter=moved)
        want, mag = plain(x, w, b, xi, yi, mem, n)
        within(y, want, (K + 2) * 2.0 ** -23 * mag)
        dy = torch.randn(n, N, generator=_gen(n), device="cuda").to(x.dtype)
        dx, dw, db = ops.grouped_linear_grads(dy, x, w, gr, gather=moved, scatter=moved)
        wx, mx = torch.zeros(n, K, dtype=torch.float64, device="cuda"), torch.zeros(n, K, dtype=torch.float64, device="cuda")
        for g in range(G):
            sel = np.nonzero(mem == g)[0]
            a, t = torch.as_tensor(xi[sel], device="cuda"), torch.as_tensor(yi[sel], device="cuda")
            d, wg, xg = dy[t].double(), w[g].double(), x[a].double()
            wx[a], mx[a] = d @ wg, d.abs() @ wg.abs()
            within(dw[g], d.t() @ xg, (sel.size + 2) * 2.0 ** -23 * (d.abs().t() @ xg.abs()))
            within(db[g], d.sum(0), (sel.size + 2) * 2.0 ** -23 * d.abs().sum(0))
        within(dx, wx, (N + 2) * 2.0 ** -23 * mx)
        wq = ops.quantize_rows(w)
        q, s = ops.quantize_rows(x)
        y8 = ops.int8_linear(x, wq, groups=gr, bias=b, relu=True, gather=moved, scatter=moved)
        want, mag = torch.zeros(n, N, dtype=torch.float64, device="cuda"), torch.zeros(n, N, dtype=torch.float64, device="cuda")
        for g in range(G):
            sel = np.nonzero(mem == g)[0]
            a, t = torch.as_tensor(xi[sel], device="cuda"), torch.as_tensor(yi[sel], device="cuda")
            want[t], mag[t] = int8_plain(q[a], s[a], wq.values[g], wq.scale[g], b[g])
        within(y8, want.clamp_min(0), INT8_SLACK * mag)


def test_gradients_are_the_differences(ops):
    """Whole numbers: every sum is exact in fp32 and the layer is linear, so (L(t + h) - L(t - h)) / 2 equals the gradient's product with h exactly."""
    g = _gen(3)
    ri = lambda *s: torch.randint(-4, 5, s, generator=g, device="cuda").float()
    m = members(90, 4, 2, 9)
    gr = ops.group_rows(m, 4)
    t = [ri(90, 37), ri(4, 50, 37), ri(4, 50)]
    dy = ri(90, 2, 50)
    f = lambda x, w, b: ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
    leaves = [a.clone().requires_grad_(True) for a in t]
    grads = torch.autograd.grad(f(*leaves), leaves, dy)
    for i in range(3):
        h = ri(*t[i].shape)
        up, down = list(t), list(t)
        up[i], down[i] = t[i] + h, t[i] - h
        diff = ((f(*up).double() - f(*down).double()) * dy.double()).sum() / 2
        assert float(diff) == float((grads[i].double() * h.double()).sum())


def test_same_bits_every_call(ops):
    m, x, w, b = make(20000, 3, 2, 128, 72, torch.float32, True)
    gr = ops.group_rows(m, 3)
    for t in (x, w, b):
        t.requires_grad_(True)
    dy = torch.randn(20000, 2, 72, device="cuda")
    runs = []
    for _ in range(3):
        y = ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
        runs.append((y.detach(),) + torch.autograd.grad(y, (x, w, b), dy))
    for r in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(r, runs[0]))


def test_slices_of_flat_parameter_vectors_and_other_strides(ops):
    """The members' weights as they lie in the flat vectors [members, d] (d odd: rows of any alignment), x a slice of a wider matrix, an expanded
    row, an expanded weight, an expanded dy."""
    g = _gen(4)
    G, K, N, d, off = 5, 40, 40, 7583, 81 + 41 * 40 + 40
    flat = torch.randn(G, d, generator=g, device="cuda")
    w = flat[:, off:off + N * K].unflatten(1, (N, K))
    b = flat[:, off + N * K:off + N * K + N]
    assert w.data_ptr() == flat.data_ptr() + 4 * off
    m = members(333, G, 0, 5)
    gr = ops.group_rows(m, G)
    big = torch.randn(333, 97, generator=g, device="cuda")
    for x in (big[:, 3:43], big[:1, 3:43].expand(333, 40), big.t().contiguous().t()[:, 3:43]):
        y = ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
        xi, yi, mem = pair_view(gr, m, True, True)
        want, mag = plain(x, w, b, xi, yi, mem, 333)
        within(y, want, (K + 2) * 2.0 ** -23 * mag)
    one = torch.randn(1, N, K, generator=g, device="cuda").requires_grad_(True)
    x = big[:, 3:43].detach().requires_grad_(True)
    y = ops.grouped_linear(x, one.expand(G, N, K), gr, gather=True, scatter=True)
    y.sum().backward()                              # dy is an expanded one
    live = (m >= 0) & (m < G)
    within(one.grad[0], x.detach().double()[live].sum(0).expand(N, K), 400 * 2.0 ** -23 * x.detach().double()[live].abs().sum(0).expand(N, K) * 2)
    within(x.grad, one.detach().double()[0].sum(0) * live[:, None], (N + 2) * 2.0 ** -23 * one.detach().double()[0].abs().sum(0) * live[:, None])


def test_infinities_and_nan_stay_in_their_rows(ops):
    for dt in DT.values():
        m, x, w, b = make(200, 3, 0, 72, 40, dt, True, nobody=True)
        gr = ops.group_rows(m, 3)
        clean = ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
        live = torch.nonzero(m >= 0)[:, 0]
        bad = x.clone()
        r1, r2 = int(live[3]), int(live[7])
        bad[r1, 71] = float("nan")
        bad[r2, 0] = float("inf")
        none = torch.nonzero(m < 0)[:, 0]
        bad[none] = float("nan")                    # rows of nobody are never read
        y = ops.grouped_linear(bad, w, gr, bias=b, relu=False, gather=True, scatter=True)
        assert torch.isnan(y[r1]).all() and not torch.isfinite(y[r2]).any()
        keep = torch.ones(200, dtype=torch.bool, device="cuda")
        keep[[r1, r2]] = False
        assert torch.equal(y[keep], clean[keep]) and (y[none] == 0).all()
        assert torch.isnan(ops.grouped_linear(bad, w, gr, bias=b, relu=True, gather=True, scatter=True)[r1]).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,N", [(1, 1), (3, 5), (300, 8), (7, 64), (20000, 136), (20001, 41), (5, 40000), (1100000, 8)])
def test_relu_mask_of_the_gradient(ops, n, N, dtype):
    """db of one row a member is the masked dy itself: dense and strided operands, rows on 16-byte borders and not, more chunks than threads in the
    grid, outputs of zero, minus zero and NaN.  Exact: nothing is rounded."""
    g = _gen(n + N)
    y = torch.randint(-2, 3, (n, N), generator=g, device="cuda").to(DT[dtype])
    dy = torch.randint(1, 9, (n, N), generator=g, device="cuda").to(DT[dtype])
    y.view(-1)[::7] = -0.0
    y.view(-1)[::11] = float("nan")
    want = torch.where(y <= 0, 0.0, dy.float())          # (a comparison with NaN is false: dy passes)
    wide_y, wide_dy = torch.zeros(n, N + 3, dtype=DT[dtype], device="cuda"), torch.zeros(n, N + 8, dtype=DT[dtype], device="cuda")
    wide_y[:, 3:], wide_dy[:, :N] = y, dy
    x = torch.ones(n, 1, dtype=DT[dtype], device="cuda")
    w = torch.ones(1, N, 1, dtype=DT[dtype], device="cuda")
    gr = ops.group_rows(torch.zeros(n, dtype=torch.int32, device="cuda"), 1)
    for yy, dd in ((y, dy), (wide_y[:, 3:], dy), (y, wide_dy[:, :N]), (wide_y[:, 3:], wide_dy[:, :N])):
        dx, _, db = ops.grouped_linear_grads(dd, x, w, gr, y=yy)
        rows, cols = want.double().sum(1), want.double().sum(0)   # (sums of positive whole numbers)
        for got, sums, terms in ((dx[:, 0], rows, N), (db[0], cols, n)):
            slack = (terms + 2) * 2.0 ** -23 * sums
            # The largest fp16 number is 65504 and its step there is 32, so that 65520 and more round to infinity: a sum that is certainly beyond
            # (here 40 000 terms of 1.8 on average) has to be infinite, any other lies within the bound or, next to the border, on either side.
            top = 65520.0 if got.dtype == torch.float16 else float("inf")
            assert torch.isinf(got[sums - slack >= top]).all()
            sure = sums + slack < top
            within(got[sure], sums[sure], slack[sure])


def test_nan_output_passes_the_gradient_as_in_relu(ops):
    x = torch.tensor([[float("nan")], [1.0], [-1.0], [0.0]], device="cuda", requires_grad=True)
    w = torch.full((1, 1, 1), 2.0, device="cuda")
    gr = ops.group_rows(torch.zeros(4, dtype=torch.int32, device="cuda"), 1)
    y = ops.grouped_linear(x, w, gr, relu=True, gather=True, scatter=True)
    got, = torch.autograd.grad(y.sum(), x)
    z = x.detach().clone().requires_grad_(True)
    want, = torch.autograd.grad(torch.relu(z * 2.0).sum(), z)
    assert torch.equal(got, want) and float(got[0]) == 2.0


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,copies,K", [(1, 2, 1), (3, 3, 5), (4, 2, 8), (2000, 5, 64), (30001, 2, 136), (3001, 3, 41), (2, 4, 20000)])
def test_copies_of_a_row_add_up(ops, n, copies, K, dtype):
    """dx of a row is the sum over its copies, those of nobody left out: whole numbers below 256 with one output, so exact in every type."""
    g = _gen(n + K)
    m = torch.randint(-1, 3, (n, copies), generator=g, device="cuda", dtype=torch.int32)
    w = torch.randint(-3, 4, (3, 1, K), generator=g, device="cuda").to(DT[dtype])
    dy = torch.randint(-4, 5, (n, copies, 1), generator=g, device="cuda").to(DT[dtype])
    x = torch.zeros(n, K, dtype=DT[dtype], device="cuda")
    dx, _, _ = ops.grouped_linear_grads(dy, x, w, ops.group_rows(m, 3), gather=True, scatter=True, need=(True, False, False))
    want = torch.zeros(n, K, device="cuda")
    for c in range(copies):
        live = m[:, c] >= 0
        want[live] += dy[live, c].float() * w[m[live, c].long(), 0].float()
    assert float(want.abs().max()) <= 60 and torch.equal(dx.float(), want)


def test_offsets_beyond_32_bits(ops):
    """Batches, outputs and weights of more than 2^32 elements: their last rows come out as those rows do alone."""
    n, K = 131077, 32776
    assert n * K > 1 << 32
    x = torch.empty(n, K, dtype=torch.bfloat16, device="cuda").normal_(generator=_gen(1))
    m = torch.zeros(n, dtype=torch.int32, device="cuda")
    m[::3] = 1
    gr = ops.group_rows(m, 2)
    w = torch.randn(2, 24, K, generator=_gen(2), device="cuda").bfloat16()
    far = torch.tensor([0, 1, n // 2, n - 3, n - 2, n - 1], device="cuda")
    xf, mf = x[far].double(), m[far].long()

    def rows_of(a, wm):   # a [6, k] times each row's own matrix [6, n, k]
        return (wm * a[:, None]).sum(-1), (wm * a[:, None]).abs().sum(-1)
    y = ops.grouped_linear(x, w, gr, gather=True, scatter=True)
    want, mag = rows_of(xf, w.double()[mf])
    within(y[far], want, (K + 2) * 2.0 ** -23 * mag)
    # dW: only the last three rows have a gradient (products of bf16 are exact in fp32, sums of at most three: two roundings)
    dy = torch.zeros(n, 24, dtype=torch.bfloat16, device="cuda")
    dy[far[3:]] = torch.randn(3, 24, generator=_gen(3), device="cuda").bfloat16()
    dx, dw, _ = ops.grouped_linear_grads(dy, x, w, gr, gather=True, scatter=True)
    want, mag = rows_of(dy[far].double(), w.double()[mf].transpose(1, 2))
    within(dx[far], want, 26 * 2.0 ** -23 * mag)
    for g in (0, 1):
        pick = far[3:][m[far[3:]] == g]
        d, a = dy[pick].double(), x[pick].double()
        within(dw[g], d.t() @ a, 5 * 2.0 ** -23 * (d.abs().t() @ a.abs()))
    del dx, dw
    # 8 bits
    q = ops.quantize_rows(x)
    near = ops.quantize_rows(x[far])
    assert torch.equal(q.values[far], near.values) and torch.equal(q.scale[far], near.scale)
    wq = ops.quantize_rows(w)
    y8 = ops.int8_linear(q, wq, groups=gr, gather=True, scatter=True)
    want, mag = rows_of(near.values.double() * near.scale.double()[:, None], wq.values.double()[mf] * wq.scale.double()[mf][..., None])
    within(y8[far], want, 4 * 2.0 ** -24 * want.abs())   # the integer sum's conversion, the scales' product, theirs
    del x, q, y, dy
    # the outputs, and the mask over them
    a = torch.randn(n, 16, generator=_gen(4), device="cuda").bfloat16()
    v = torch.randn(2, K, 16, generator=_gen(5), device="cuda").bfloat16()
    y = ops.grouped_linear(a, v, gr, relu=True, gather=True, scatter=True)
    want, mag = rows_of(a[far].double(), v.double()[mf])
    within(y[far], want.clamp_min(0), 18 * 2.0 ** -23 * mag)
    dy = torch.zeros_like(y)
    dy[far] = 1.0
    dx, _, _ = ops.grouped_linear_grads(dy, a, v, gr, y=y, gather=True, scatter=True, need=(True, False, False))
    want, mag = rows_of((y[far] > 0).double(), v.double()[mf].transpose(1, 2))
    within(dx[far], want, (K + 2) * 2.0 ** -23 * mag)
    del y, dy
    big = torch.empty(3, 40000, 40000, dtype=torch.bfloat16, device="cuda").normal_(generator=_gen(6))
    assert big.numel() > 1 << 32
    a = torch.randn(5, 40000, generator=_gen(7), device="cuda").bfloat16()
    y = ops.grouped_linear(a, big, ops.group_rows(torch.full((5,), 2, dtype=torch.int32, device="cuda"), 3), gather=True, scatter=True)
    last = big[2, -8:].double()
    within(y[:, -8:], (a.double()[:, None] * last).sum(-1), 40002 * 2.0 ** -23 * (a.double()[:, None] * last).abs().sum(-1))


def test_no_rows(ops):
    m = torch.empty(0, dtype=torch.int32, device="cuda")
    gr = ops.group_rows(m, 3)
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    w = torch.randn(3, 4, 8, device="cuda", requires_grad=True)
    b = torch.randn(3, 4, device="cuda", requires_grad=True)
    y = ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
    assert tuple(y.shape) == (0, 4)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 4, device="cuda"))
    assert tuple(dx.shape) == (0, 8) and (dw == 0).all() and (db == 0).all()
    q = ops.quantize_rows(x.detach())
    assert tuple(q.values.shape) == (0, 8) and ops.int8_linear(q, ops.quantize_rows(w[0].detach())).shape == (0, 4)


def test_everybody_nobody(ops):
    m = torch.full((100,), -1, dtype=torch.int32, device="cuda")
    gr = ops.group_rows(m, 2)
    _, x, w, b = make(100, 2, 0, 24, 40, torch.bfloat16, True)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
    grads = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert all((t == 0).all() for t in (y, *grads))


# ---- 8 bits ----------------------------------------------------------------------------------------------------------------------------------
def plain_quantize(x):
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    return torch.round(127 * x / torch.where(amax > 0, amax, 1.0)), divide_127(amax[..., 0])


def divide_127(amax):
    """amax / 127 rounded once to float32 (numpy: torch may multiply by a rounded reciprocal)."""
    return torch.as_tensor(amax.cpu().numpy().astype(np.float32) / np.float32(127))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,K", [(1, 1), (1, 4096), (15, 41), (64, 40), (1000, 257), (33, 5000), (3, 20001), (2500, 128), (2100, 41), (2100, 511), (2100, 1030), (7, 16), (5000, 3)])
def test_quantize_rows_is_exact(ops, n, K, dtype):
    x = torch.randn(n, K, generator=_gen(K), device="cuda").to(DT[dtype])
    q, s = ops.quantize_rows(x)
    wq, ws = plain_quantize(x)
    assert q.dtype == torch.int8 and torch.equal(q.double(), wq)
    assert torch.equal(s.cpu(), ws)


def test_quantize_rows_at_the_borders(ops):
    """Values in the middle between two integers (ties to even), next to it, tiny and huge rows, rows of zeros."""
    mid = torch.arange(-126, 127, device="cuda").double() + 0.5
    row = torch.cat([mid, torch.tensor([127.0], device="cuda")])
    rows = [row.float() * s for s in (1.0, 2.0 ** -120, 2.0 ** -140, 2.0 ** 120, 2.0 ** -7)]
    up, down = torch.nextafter(row.float(), torch.tensor(1e9, device="cuda")), torch.nextafter(row.float(), torch.tensor(-1e9, device="cuda"))
    up[-1] = down[-1] = 127.0
    third = torch.cat([(mid / 3).float(), torch.tensor([127.0 / 3], device="cuda")])
    x = torch.stack(rows + [up, down, third, torch.zeros_like(up)])
    q, s = ops.quantize_rows(x)
    wq, _ = plain_quantize(x)
    assert torch.equal(q.double(), wq)
    assert torch.equal(s.cpu(), divide_127(x.abs().amax(1))) and float(s[-1]) == 0


def test_quantize_rows_shapes_and_strides(ops):
    w = torch.randn(3, 10, 48, device="cuda")
    q, s = ops.quantize_rows(w)
    assert tuple(q.shape) == (3, 10, 48) and tuple(s.shape) == (3, 10)
    for v in (w[:, :, 3:40], w.transpose(0, 1), w[0].t(), w[:, ::2]):
        a, b = ops.quantize_rows(v), ops.quantize_rows(v.contiguous())
        assert torch.equal(a.values, b.values) and torch.equal(a.scale, b.scale)


def test_rows_that_are_not_finite_give_nan(ops):
    x = torch.randn(40, 64, device="cuda")
    x[3, 5], x[9, 63], x[11, 0] = float("nan"), float("inf"), -float("inf")
    w = ops.quantize_rows(torch.randn(24, 64, device="cuda"))
    q = ops.quantize_rows(x)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[3, 9, 11]] = True
    assert torch.equal(torch.isnan(q.scale), bad) and (q.values[bad] == 0).all()
    y = ops.int8_linear(x, w, relu=True)
    assert torch.equal(torch.isnan(y).any(1), bad) and torch.isnan(y[bad]).all()


def int8_plain(q, s, wq, ws, b):
    """One matrix, in 64 bits -> (y, |sum| scale + |b|); the sums are whole numbers below 2^53."""
    acc = q.double() @ wq.double().t()
    sc = s.double()[:, None] * ws.double()[None]
    bb = 0 if b is None else b.double()
    return acc * sc + bb, (acc * sc).abs() + (0 if b is None else b.double().abs())


INT8_SLACK = 4 * 2.0 ** -24   # the sum to fp32, the product of the scales, their product, the bias


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("n,K,N", [(1, 1, 1), (2, 100, 33), (3, 4096, 64), (4, 15, 16), (9, 4095, 40), (33, 512, 64), (1, 70000, 24), (1, 4096, 512), (1, 41, 40), (5, 128, 130), (16, 1040, 64), (17, 4096, 96), (64, 64, 64), (129, 257, 255), (3000, 640, 384), (300, 4099, 16)])
def test_int8_linear_dense(ops, n, K, N, out):
    g = _gen(n + K)
    x = (torch.randn(n, K, generator=g, device="cuda") * 3).to(DT[out])
    w = ops.quantize_rows(torch.randn(N, K, generator=g, device="cuda"))
    b = torch.randn(N, generator=g, device="cuda").to(DT[out])
    q, s = ops.quantize_rows(x)
    for relu, bias in ((True, b), (False, None)):
        want, mag = int8_plain(q, s, w.values, w.scale, bias)
        if relu:
            want = want.clamp_min(0)
        y = ops.int8_linear(x, w, bias=bias, relu=relu)
        assert y.dtype == x.dtype
        within(y, want, INT8_SLACK * mag)
        assert torch.equal(y, ops.int8_linear(ops.QuantRows(q, s), w, bias=bias, relu=relu, dtype=DT[out]))


def test_int8_sums_are_exact_at_their_largest(ops):
    for K in (131072, 131056):
        q = torch.full((3, K), 127, dtype=torch.int8, device="cuda")
        w = torch.full((20, K), -127, dtype=torch.int8, device="cuda")
        one = lambda n: torch.ones(n, device="cuda")
        y = ops.int8_linear(ops.QuantRows(q, one(3)), ops.QuantRows(w, one(20)))
        assert (y == float(np.float32(-127 * 127 * K))).all()


@pytest.mark.parametrize("n,G,copies,K,N", SHAPES)
def test_int8_linear_grouped(ops, n, G, copies, K, N):
    for gather, scatter, relu, dt in ((True, True, True, torch.bfloat16), (False, False, False, torch.float32), (True, False, False, torch.float16)):
        m, x, w, b = make(n, G, copies, K, N, dt, gather, seed=n + K)
        gr, wq = ops.group_rows(m, G), ops.quantize_rows(w)
        y = ops.int8_linear(x, wq, groups=gr, bias=b, relu=relu, gather=gather, scatter=scatter)
        q, s = ops.quantize_rows(x)
        xi, yi, mem = pair_view(gr, m, gather, scatter)
        want = torch.zeros(m.numel(), N, dtype=torch.float64, device="cuda")
        mag = torch.zeros_like(want)
        for g in range(G):
            sel = np.nonzero(mem == g)[0]
            a, t = torch.as_tensor(xi[sel], device="cuda"), torch.as_tensor(yi[sel], device="cuda")
            want[t], mag[t] = int8_plain(q[a], s[a], wq.values[g], wq.scale[g], b[g])
        within(y.reshape(-1, N), want.clamp_min(0) if relu else want, INT8_SLACK * mag)


# ---- together ----------------------------------------------------------------------------------------------------------------------------------
def chain(ops, x, gr, ws, bs):
    h = ops.grouped_linear(x, ws[0], gr, bias=bs[0], relu=True, gather=True)
    h = ops.grouped_linear(h, ws[1], gr, bias=bs[1], relu=True)
    return ops.grouped_linear(h, ws[2], gr, bias=bs[2], scatter=True)


def test_feature_network_of_random_members_and_its_saliency(ops):
    """feature_nn of the pretrained members (41 -> 40 -> 40 -> 20, straight from their flat vectors), every row through two random members: equal
    to the per-member evaluation by plain products, and its gradient by autograd through them, in 64 bits."""
    from conftest import load_golden
    flat = torch.as_tensor(np.stack([load_golden(f"swag_v50_{i}.npz")["w_avg"] for i in (0, 12)])).float().cuda()
    ws, bs, at = [], [], 81
    for k, n in ((41, 40), (40, 40), (40, 20)):
        ws.append(flat[:, at:at + n * k].unflatten(1, (n, k)))
        bs.append(flat[:, at + n * k:at + n * k + n])
        at += n * k + n
    x = torch.as_tensor(load_golden("inputs.npz")["x_slow"]).float().cuda().reshape(-1, 41)[:1500].contiguous().requires_grad_(True)
    m = torch.stack([torch.arange(1500, device="cuda") % 2, (torch.arange(1500, device="cuda") // 3) % 2], 1).int()
    m[7, 1] = -1
    gr = ops.group_rows(m, 2)
    y = chain(ops, x, gr, ws, bs)
    (dx,) = torch.autograd.grad(y.square().sum(), (x,))
    # per member, in 64 bits: values h, pre-activations z and their error bound e (a layer adds (K + 2) 2^-23 of its magnitudes and passes on |W| e)
    rows = torch.arange(1500, device="cuda")
    want, bound = torch.zeros(1500, 2, 20, dtype=torch.float64, device="cuda"), torch.zeros(1500, 2, 20, dtype=torch.float64, device="cuda")
    dwant, dbound = torch.zeros(1500, 41, dtype=torch.float64, device="cuda"), torch.zeros(1500, 41, dtype=torch.float64, device="cuda")
    clear = torch.ones(1500, dtype=torch.bool, device="cuda")       # no ReLU's side within the error: its gradient is determined
    for c in range(2):
        for g in range(2):
            r = rows[m[:, c] == g]
            h, e = x.detach().double()[r], torch.zeros(r.numel(), 41, dtype=torch.float64, device="cuda")
            sides = []
            for l in range(3):
                w, b = ws[l][g].double(), bs[l][g].double()
                z = h @ w.t() + b
                e = e @ w.abs().t() + (w.shape[1] + 2) * 2.0 ** -23 * ((h.abs() + e) @ w.abs().t() + b.abs())
                if l < 2:
                    sides.append(z > 0)
                    clear[r] &= (z.abs() > e).all(1)
                    h = z.clamp_min(0)
            want[r, c], bound[r, c] = z, e
            d, de = 2 * z, 2 * e + 2.0 ** -22 * z.abs()
            for l in (2, 1, 0):
                w = ws[l][g].double()
                de = de @ w.abs() + (w.shape[0] + 2) * 2.0 ** -23 * ((d.abs() + de) @ w.abs())
                d = d @ w
                if l:
                    d, de = d * sides[l - 1], de * sides[l - 1]
            dwant[r] += d
            dbound[r] += de + 2.0 ** -22 * d.abs()
    within(y, want, bound)
    assert int(clear.sum()) > 750
    within(dx[clear], dwant[clear], dbound[clear])


def test_captured_and_replayed_next_to_eager_work(ops):
    """Forward, gradients and the 8-bit layer in two graphs on their own streams' pools, replayed several times with new inputs and eager work between."""
    G, K, N, n = 3, 64, 48, 500
    m, x, w, b = make(n, G, 2, K, N, torch.bfloat16, True)
    dy = torch.randn(n, 2, N, device="cuda").to(torch.bfloat16)
    wq = ops.quantize_rows(w)

    def step():
        gr = ops.group_rows(m, G)
        y = ops.grouped_linear(x, w, gr, bias=b, relu=True, gather=True, scatter=True)
        return (y, ops.int8_linear(x, wq, groups=gr, bias=b, gather=True, scatter=True)) + ops.grouped_linear_grads(dy, x, w, gr, y=y, gather=True, scatter=True)

    step()
    graphs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = step()
        graphs.append((g, out))
    for r in range(4):
        m.copy_(members(n, G, 2, seed=100 + r))
        x.copy_(torch.randn(n, K, generator=_gen(r), device="cuda"))
        want = [t.clone() for t in step()]
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_autograd_under_capture_is_refused(ops):
    """... also while an eager graph of the same leaves lives; the process and the leaves stay usable, and the plain functions capture."""
    m, x, w, b = make(64, 3, 0, 16, 24, torch.float32, True)
    for t in (x, w, b):
        t.requires_grad_(True)
    gr = ops.group_rows(m, 3)
    alive = ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="capture"):
            ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
        with torch.no_grad():
            y = ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
            grads = ops.grouped_linear_grads(torch.ones_like(y), x, w, gr, gather=True, scatter=True)
    want = torch.autograd.grad(alive, (x, w, b), torch.ones_like(alive))
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, alive) and all(torch.equal(a, c) for a, c in zip(grads, want))


def test_on_another_stream(ops):
    m, x, w, b = make(3000, 5, 0, 128, 64, torch.float32, True)
    gr = ops.group_rows(m, 5)
    want = ops.grouped_linear(x, w, gr, bias=b, gather=True, scatter=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.grouped_linear(x, w, ops.group_rows(m, 5), bias=b, gather=True, scatter=True)
    s.synchronize()
    assert torch.equal(got, want)
