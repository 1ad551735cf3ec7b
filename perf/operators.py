"""The ensemble's grouped and 8-bit linear layers as they are measured: cases, inputs, a plain form of each operator in elementary torch
operations, the calls a user makes of this package's own operators, and the definitions in 64 bits.

Five operators (`kind` of a case):
  group     rows sorted by the ensemble member that evaluates them: `order` (stable) and `offsets`
  linear    y_r = act(W[g] x_r + b[g]) for the rows of every member g, gathered from / scattered to the batch's own order
  train     the same layer (no activation) with its gradients dx, dW, db
  quantize  rows to 8-bit integers with one scale each
  int8      the linear layer on 8-bit operands, a scale per row and per output channel; one matrix, or one per member
A row whose member is -1 (padding of a batch) belongs to nobody: its output and its gradient are zero.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _case(kind, n, G=0, K=0, N=0, dtype="f32", copies=1, relu=False, moved=True, name=None):
    c = {"kind": kind, "rows": n, "members": G, "inputs": K, "outputs": N, "dtype": dtype, "copies": copies, "relu": relu, "moved": moved}
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one validation batch of 3 000 rows over the 30 members
        _case("group", 3000, G=30, name="group-batch"),
        # a million systems with four random members each
        _case("group", 1000000, G=30, copies=4, name="group-systems"),
        # one 15-row chunk of the evaluation scripts, every row its own member, through a 40-wide hidden layer: latency
        _case("linear", 15, G=30, K=40, N=40, relu=True, name="linear-chunk"),
        # the first layer on 1 500 systems x 100 time steps of 41 features (rows of 164 bytes)
        _case("linear", 150000, G=30, K=41, N=128, relu=True, name="linear-series"),
        # a wide hidden layer of eight members, two members a row, gathered and scattered back
        _case("linear", 32768, G=8, K=4096, N=4096, dtype="bf16", copies=2, relu=True, name="linear-wide"),
        # a training step of a 128-wide layer over 30 members
        _case("train", 30000, G=30, K=128, N=128, name="train-series"),
        # a training step of a wide layer, rows already in the members' order
        _case("train", 32768, G=16, K=2048, N=2048, dtype="bf16", moved=False, name="train-wide"),
        # one row, as before a product for a single system
        _case("quantize", 1, K=4096, dtype="bf16", name="quantize-row"),
        # the activations of a large batch
        _case("quantize", 65536, K=4096, dtype="bf16", name="quantize-batch"),
        # a single row through a wide layer: the weights' 16 MiB are what is read
        _case("int8", 1, K=4096, N=4096, dtype="bf16", name="int8-row"),
        # the validation batch over the members' own matrices
        _case("int8", 3000, G=30, K=1024, N=1024, dtype="f32", relu=True, name="int8-members"),
        # a large batch through one wide layer
        _case("int8", 16384, K=4096, N=8192, dtype="bf16", relu=True, name="int8-wide"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    w = _log_int(rng, lo, hi)
    if rng.random() < 0.6 and w >= 16:      # most layers have widths of a multiple of 16, some are odd
        w = max(16, w // 16 * 16)
    return w


def draw(rng):
    kind = rng.choice(["group", "linear", "linear", "train", "quantize", "int8", "int8"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "group":
        copies = rng.choice([1, 1, 2, 4])
        return _case(kind, _log_int(rng, 1, 1000000), G=_log_int(rng, 1, 256), copies=copies)
    if kind == "quantize":
        return _case(kind, _log_int(rng, 1, 65536), K=_width(rng, 1, 4096), dtype=dtype)
    limit = {"linear": 1.09e12, "train": 1.37e11, "int8": 5.4e11}[kind]     # multiply-adds of the largest listed case of the kind
    if dtype == "f32" and kind != "int8":
        limit /= 16
    if kind == "int8" and rng.random() < 0.5:
        G, copies = 0, 1
    else:
        G, copies = _log_int(rng, 1, 64), rng.choice([1, 1, 2, 4])
    K, N = _width(rng, 8, 4096), _width(rng, 8, 4096)
    n = _log_int(rng, 1, max(1, min(65536 // copies, int(limit / (K * N * copies)))))
    return _case(kind, n, G=G, K=K, N=N, dtype=dtype, copies=copies, relu=kind != "train" and rng.random() < 0.5, moved=rng.random() < 0.7)


def _members(case, gen):
    """The member of every (row, copy): uneven shares, one member without rows, some padded rows."""
    n, G, k = case["rows"], case["members"], case["copies"]
    share = torch.softmax(0.7 * torch.randn(G, generator=gen, device="cuda"), 0)
    if G >= 3:
        share[int(torch.randint(0, G, (1,), generator=gen, device="cuda"))] = 0.0
    m = torch.multinomial(share, n * k, replacement=True, generator=gen).to(torch.int32)
    if n >= 64:
        m[torch.rand(n * k, generator=gen, device="cuda") < 1.0 / 64] = -1
    return m.view(n, k) if k > 1 else m


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    gen = torch.Generator("cuda").manual_seed(int(seed) * 7919 + 17)
    n, G, K, N, k, kind = case["rows"], case["members"], case["inputs"], case["outputs"], case["copies"], case["kind"]
    dt = DTYPES[case["dtype"]]
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")
    t = {"member": _members(case, gen) if G else None}
    if kind == "group":
        return t
    rows = n if (case["moved"] or not G) else n * k
    x = rnd(rows, K)
    if kind in ("quantize", "int8"):        # activations with a few channels that stand out
        x = x * torch.where(torch.rand(K, generator=gen, device="cuda") < 0.02, 8.0, 1.0)
    t["x"] = x.to(dt)
    if kind == "quantize":
        return t
    shape = (G, N, K) if G else (N, K)
    if kind == "int8":
        t["wq"] = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
        t["ws"] = (0.5 + torch.rand(shape[:-1], generator=gen, device="cuda")) / (64.0 * math.sqrt(K))
    else:
        t["w"] = torch.empty(shape, dtype=dt, device="cuda")
        for g in range(G):
            t["w"][g] = rnd(N, K) / math.sqrt(K)
    t["b"] = (0.5 * rnd(*shape[:-1])).to(dt)
    if kind == "train":
        t["dy"] = (rnd(n, k, N) if k > 1 else rnd(n, N)).to(dt) if case["moved"] else rnd(n * k, N).to(dt)
    return t


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["members"] and case["kind"] != "group":
        if own:
            from bnn_chaos_model_amd import ops
            s["groups"] = ops.group_rows(s["member"], case["members"])
        else:
            s["order"], off = _plain_group(s["member"], case["members"])
            s["off"] = off.tolist()
    if own and case["kind"] == "int8":
        from bnn_chaos_model_amd import ops
        s["weight"] = ops.QuantRows(s["wq"], s["ws"])
    if own and case["kind"] == "train":
        for name in ("x", "w", "b"):
            s[name].requires_grad_(True)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------------
def _plain_group(member, G):
    key = member.reshape(-1).long()
    key = torch.where((key < 0) | (key >= G), G, key)
    order = torch.argsort(key, stable=True).int()
    count = torch.zeros(G + 1, dtype=torch.long, device=key.device).scatter_add_(0, key, torch.ones_like(key))
    off = torch.zeros(G + 1, dtype=torch.long, device=key.device)
    off[1:] = count[:G].cumsum(0)
    return order, off.int()


def _plain_quantize(x):
    x = x.double()                                   # the border between two integers is met exactly in 64 bits
    amax = x.abs().amax(1, keepdim=True)
    q = torch.round(x * 127.0 / torch.where(amax > 0, amax, 1.0))
    return q, (amax[:, 0] / 127.0).float()


def _pairs(s):
    """The grouped rows' positions in x (rows of members only)."""
    return s["order"][:s["off"][-1]].long()


def _plain_take(s, x):
    case = s["case"]
    return x[_pairs(s) // case["copies"]] if case["moved"] else x[:s["off"][-1]]


def _plain_put(s, y):
    """Grouped rows y back to where the caller has them; rows without a member are zero."""
    case = s["case"]
    P, k = case["rows"] * case["copies"], case["copies"]
    out = torch.zeros((P, y.shape[1]), dtype=y.dtype, device=y.device)
    if not case["moved"]:
        out[:y.shape[0]] = y
        return out
    out[_pairs(s)] = y
    return out.view(case["rows"], k, -1) if k > 1 else out


def _plain_linear(s):
    case, off = s["case"], s["off"]
    x = _plain_take(s, s["x"].float())
    y = torch.empty((off[-1], case["outputs"]), device=x.device)
    for g in range(case["members"]):
        a, e = off[g], off[g + 1]
        if e > a:
            y[a:e] = x[a:e] @ s["w"][g].float().t() + s["b"][g].float()
    if case["relu"]:
        y = y.clamp_min(0)
    return _plain_put(s, y.to(s["x"].dtype))


def _plain_train(s):
    case, off, dt = s["case"], s["off"], s["x"].dtype
    x, k = _plain_take(s, s["x"].float()), case["copies"]
    dy = s["dy"].float().reshape(-1, case["outputs"])
    dy = dy[_pairs(s)] if case["moved"] else dy[:off[-1]]
    dx, dw, db = torch.empty_like(x), torch.zeros_like(s["w"]), torch.zeros_like(s["b"])
    for g in range(case["members"]):
        a, e = off[g], off[g + 1]
        if e > a:
            dx[a:e] = dy[a:e] @ s["w"][g].float()
            dw[g] = (dy[a:e].t() @ x[a:e]).to(dt)
            db[g] = dy[a:e].sum(0).to(dt)
    dx = _plain_put(s, dx)
    if case["moved"] and k > 1:
        dx = dx.sum(1)
    return _plain_linear(s), dx.to(dt), dw, db


def _plain_int8(s):
    case, dt = s["case"], s["x"].dtype
    q, xs = _plain_quantize(s["x"])
    scale = lambda acc, a, w: (acc * a.double()[:, None] * w.double()[None, :])
    if not case["members"]:
        y = scale(q @ s["wq"].double().t(), xs, s["ws"]) + s["b"].double()
        return (y.clamp_min(0) if case["relu"] else y).to(dt)
    q, xs, off = _plain_take(s, q), _plain_take(s, xs), s["off"]
    y = torch.empty((off[-1], case["outputs"]), dtype=torch.float64, device=q.device)
    for g in range(case["members"]):
        a, e = off[g], off[g + 1]
        if e > a:
            y[a:e] = scale(q[a:e] @ s["wq"][g].double().t(), xs[a:e], s["ws"][g]) + s["b"][g].double()
    if case["relu"]:
        y = y.clamp_min(0)
    return _plain_put(s, y.to(dt))


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "group":
            return _plain_group(s["member"], case["members"])
        if kind == "quantize":
            q, scale = _plain_quantize(s["x"])
            return q.float() * scale[:, None], scale
        return {"linear": _plain_linear, "train": _plain_train, "int8": _plain_int8}[kind](s)
    from bnn_chaos_model_amd import ops
    if kind == "group":
        groups = ops.group_rows(s["member"], case["members"])
        return groups.order, groups.offsets
    if kind == "quantize":
        q, scale = ops.quantize_rows(s["x"])
        return q * scale[:, None], scale
    if kind == "int8":
        moved = bool(case["members"]) and case["moved"]
        return ops.int8_linear(s["x"], s["weight"], groups=s.get("groups"), bias=s["b"], relu=case["relu"], gather=moved, scatter=moved)
    y = ops.grouped_linear(s["x"], s["w"], s["groups"], bias=s["b"], relu=case["relu"], gather=case["moved"], scatter=case["moved"])
    if kind == "linear":
        return y
    return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])


def work(case):
    kind, n, k, K, N, es = case["kind"], case["rows"], case["copies"], case["inputs"], case["outputs"], SIZE[case["dtype"]]
    P = n * k
    if kind == "group":
        return {"bytes": 8 * P, "flops": 0}
    if kind == "quantize":
        return {"bytes": n * K * (es + 4) + 4 * n, "flops": 3 * n * K}
    used = min(max(case["members"], 1), P)           # matrices that any row needs
    rows_in = n if (case["moved"] or not case["members"]) else P
    wb = 1 if kind == "int8" else es
    nbytes = rows_in * K * es + used * N * K * wb + P * N * es + used * N * (es + (4 if kind == "int8" else 0))
    if kind != "train":
        return {"bytes": nbytes, "flops": 2 * P * N * K}
    back = P * N * es + rows_in * K * es + max(case["members"], 1) * N * (K + 1) * es
    return {"bytes": nbytes + back, "flops": 6 * P * N * K}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------------
def exact(case, seed):
    kind, k, N = case["kind"], case["copies"], case["outputs"]
    if kind == "group":
        return None
    t = _inputs(case, seed)
    x = t["x"].double()
    if kind in ("quantize", "int8"):
        amax = x.abs().max(dim=1).values
        step = amax / 127.0
        codes = torch.zeros_like(x)
        some = amax > 0
        codes[some] = torch.round(x[some] / amax[some, None] * 127.0)
        if kind == "quantize":
            return codes * step[:, None], step
        x = codes * step[:, None]
        w = t["wq"].double() * t["ws"].double().unsqueeze(-1)
    else:
        w = t["w"].double()
    b = t["b"].double()
    act = (lambda v: torch.relu(v)) if case["relu"] else (lambda v: v)
    if not case["members"]:
        return act(torch.addmm(b, x, w.t()))
    P = case["rows"] * k
    member = t["member"].reshape(-1)
    lists = [torch.nonzero(member == g)[:, 0] for g in range(case["members"])]     # (row, copy) pairs of every member, in the batch's order
    start = [0]
    for idx in lists:
        start.append(start[-1] + idx.numel())
    y = torch.zeros((P, N), dtype=torch.float64, device=x.device)
    dx = torch.zeros_like(x)
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    dy = t["dy"].double().reshape(P, N) if kind == "train" else None
    for g, idx in enumerate(lists):
        if idx.numel() == 0:
            continue
        if case["moved"]:
            src, dst = torch.div(idx, k, rounding_mode="floor"), idx
        else:
            src = dst = torch.arange(start[g], start[g + 1], device=x.device)
        xg = x[src]
        y[dst] = act(torch.addmm(b[g], xg, w[g].t()))
        if kind == "train":
            dx.index_add_(0, src, dy[dst] @ w[g])
            dw[g] = torch.mm(dy[dst].t(), xg)
            db[g] = dy[dst].sum(0)
    if case["moved"] and k > 1:
        y = y.view(case["rows"], k, N)
    return y if kind != "train" else (y, dx, dw, db)
