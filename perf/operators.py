"""Cases of the operators over a fitted tree's leaves, for measuring them.

``leaf_embedding`` looks up one learned vector per row by the row's leaf (and sums its gradient by
leaf); ``leaf_linear`` multiplies every row with the matrix of its leaf (a linear model per leaf, or
the experts behind a router), with the gradients of rows, matrices and biases. Each pass starts
from the bare leaf indices: the sort of the rows by leaf is part of it.

``own`` false computes the plain form in elementary torch operations; true calls the framework.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
# for the comparison of two cases' sizes only: seconds a byte and a multiply-add cost, roughly
RATE = {"f32": 1.0e14, "f16": 1.0e15, "bf16": 1.0e15}


def listed():
    """The listed cases. ``op``: embed / linear; ``grad``: with the backward pass. ``n`` rows,
    ``leaves`` leaves (experts, or a vocabulary), ``skew``: leaf r is met with weight
    (r + 1)^-skew, ``pad``: share of the rows without a leaf (-1)."""
    def embed(name, n, leaves, d, dtype, grad, scale=1.0, skew=0.0, pad=0.0):
        return {"name": name, "op": "embed", "n": n, "leaves": leaves, "d": d, "dtype": dtype,
                "grad": grad, "scale": scale, "skew": skew, "pad": pad}

    def linear(name, n, leaves, k, m, dtype, grad, bias=False, skew=0.0, pad=0.0):
        return {"name": name, "op": "linear", "n": n, "leaves": leaves, "k": k, "m": m,
                "dtype": dtype, "grad": grad, "bias": bias, "skew": skew, "pad": pad}

    return [
        # answering for one row: latency alone
        embed("embed_one", 1, 93_500, 1024, "bf16", False, scale=32.0),
        # the leaves of 1M training rows under a full-depth tree, short vectors
        embed("embed_rows", 1_000_000, 93_500, 16, "f32", False, scale=0.25, skew=0.5),
        # a training step on a batch with a skewed vocabulary and padding
        embed("embed_train", 16_384, 50_001, 1024, "bf16", True, scale=32.0, skew=1.0, pad=0.05),
        # a depth-6 tree: few leaves with very many rows each, odd width
        embed("embed_train_few", 1_000_000, 64, 63, "f32", True, skew=0.5),
        # a large table and a large batch
        embed("embed_train_large", 200_000, 120_000, 2048, "f16", True, scale=4.0, skew=0.5),
        # one row through its leaf's matrix: latency and one matrix read
        linear("linear_one", 1, 64, 2048, 1024, "bf16", False),
        # a small serving batch: about one row a matrix, bound by reading the matrices
        linear("linear_batch", 64, 64, 2048, 1024, "bf16", False, bias=True),
        # a long prompt's worth of rows over 32 matrices, bound by the matrix cores
        linear("linear_prompt", 32_768, 32, 2048, 4096, "bf16", False, skew=0.5),
        # odd sizes, leaves of very different sizes, rows without a leaf
        linear("linear_train_odd", 10_007, 12, 1000, 601, "f16", True, bias=True, skew=1.0,
               pad=0.05),
        # linear leaves for regression: 100k x 32 rows under a depth-limited tree, one output
        linear("linear_train_reg", 100_000, 1_500, 32, 1, "f32", True, bias=True, skew=0.5),
        # linear leaves for 64 classes: 1M x 64 rows under a depth-12 tree
        linear("linear_train_rows", 1_000_000, 4_096, 64, 64, "f32", True, bias=True, skew=0.5),
        # a large training step
        linear("linear_train_large", 65_536, 64, 2048, 2048, "bf16", True, skew=0.5),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 4.0e12 + w["flops"] / RATE[case["dtype"]]


def draw(rng):
    """One more case of the listed ones' ranges."""
    cap = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("embed", "linear")}
    while True:
        op = rng.choice(("embed", "linear"))
        case = {"op": op, "n": _log(rng, 1, 1_000_000), "dtype": rng.choice(("f32", "f16", "bf16")),
                "grad": rng.random() < 0.6, "skew": rng.choice((0.0, 0.5, 1.0)),
                "pad": rng.choice((0.0, 0.0, 0.05))}
        if op == "embed":
            case.update(leaves=_log(rng, 2, 200_000), d=_log(rng, 1, 4096),
                        scale=rng.choice((1.0, 0.25, 32.0)))
        else:
            case.update(leaves=_log(rng, 1, 4096), k=_log(rng, 1, 4096), m=_log(rng, 1, 4096),
                        bias=rng.random() < 0.5)
            if case["leaves"] * case["k"] * case["m"] > 2 ** 29:
                continue
        if _cost(case) <= cap[op]:
            return case


def _weights(case):
    p = (np.arange(case["leaves"], dtype=np.float64) + 1.0) ** -case["skew"]
    return p / p.sum()


def work(case):
    """Bytes and operations of one pass: inputs read once (of a table or the matrices the expected
    share that some row meets), outputs written once."""
    n, leaves, sz = case["n"], case["leaves"], BYTES[case["dtype"]]
    rows = n * (1.0 - case["pad"])
    met = float((1.0 - np.exp(rows * np.log1p(-np.minimum(_weights(case), 1 - 1e-12)))).sum())
    if case["op"] == "embed":
        d = case["d"]
        nbytes = 8 * n + met * d * sz + n * d * sz
        flops = rows * d
        if case["grad"]:
            nbytes += rows * d * sz + leaves * d * sz
            flops += rows * d
    else:
        k, m = case["k"], case["m"]
        bias = case["bias"]
        nbytes = 8 * n + (rows * k + met * m * (k + bias) + n * m) * sz
        flops = 2.0 * rows * k * m
        if case["grad"]:
            nbytes += (rows * m + n * k + leaves * m * (k + bias)) * sz
            flops *= 3.0
    return {"bytes": int(nbytes), "flops": int(flops)}


def prepare(case, seed):
    """Leaf indices as a tree's walk gives them, the parameters, and the incoming gradient."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    n, dt = case["n"], DTYPES[case["dtype"]]

    def normal(shape, std):
        out = torch.empty(shape, dtype=dt, device=dev)
        flat = out.view(-1)
        for a in range(0, flat.numel(), 2 ** 27):  # in parts: large matrices in one type only
            part = flat[a : a + 2 ** 27]
            part.copy_(torch.randn(part.numel(), generator=g, device=dev) * std)
        return out

    cdf = torch.from_numpy(np.cumsum(_weights(case))).to(dev)
    u = torch.rand(n, generator=g, device=dev, dtype=torch.float64)
    rank = torch.searchsorted(cdf, u).clamp_(max=case["leaves"] - 1)
    leaves = torch.randperm(case["leaves"], generator=g, device=dev)[rank]
    if case["pad"]:
        leaves[torch.rand(n, generator=g, device=dev) < case["pad"]] = -1
    st = {"case": case, "leaves": leaves}
    if case["op"] == "embed":
        st["table"] = normal((case["leaves"], case["d"]), 0.02)
        if case["grad"]:
            st["dy"] = normal((n, case["d"]), 0.1)
    else:
        st["x"] = normal((n, case["k"]), 1.0)
        st["weight"] = normal((case["leaves"], case["m"], case["k"]), case["k"] ** -0.5)
        st["bias"] = normal((case["leaves"], case["m"]), 0.1) if case["bias"] else None
        if case["grad"]:
            st["dy"] = normal((n, case["m"]), 0.1)
    if own and case["grad"]:
        for name in ("table", "x", "weight", "bias"):
            if st.get(name) is not None:
                st[name].requires_grad_()
    return st


def run(st):
    """One pass: the outputs, and the gradients of every float input where there is a backward."""
    embed = st["case"]["op"] == "embed"
    if own:
        return _own_embed(st) if embed else _own_linear(st)
    return _plain_embed(st) if embed else _plain_linear(st)


def _own_embed(st):
    from mpitree_amd import leaf_embedding

    y = leaf_embedding(st["leaves"], st["table"], scale=st["case"]["scale"])
    if not st["case"]["grad"]:
        return y
    (dtable,) = torch.autograd.grad(y, (st["table"],), st["dy"])
    return y.detach(), dtable


def _own_linear(st):
    from mpitree_amd import leaf_linear

    y = leaf_linear(st["x"], st["leaves"], st["weight"], st["bias"])
    if not st["case"]["grad"]:
        return y
    wrt = [st["x"], st["weight"]] + ([st["bias"]] if st["bias"] is not None else [])
    return (y.detach(), *torch.autograd.grad(y, wrt, st["dy"]))


def _plain_embed(st):
    case, leaves, table = st["case"], st["leaves"], st["table"]
    none = (leaves < 0)[:, None]
    y = table[leaves.clamp(min=0)].float() * case["scale"]
    y = y.masked_fill_(none, 0.0).to(table.dtype)
    if not case["grad"]:
        return y
    # sums over the rows of a leaf in 64 bits: a leaf may hold most of a million rows
    dtable = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
    dtable.index_add_(0, leaves.clamp(min=0), st["dy"].double().masked_fill_(none, 0.0))
    return y, (dtable * case["scale"]).to(table.dtype)


def _plain_linear(st):
    case, leaves, x, w, b = st["case"], st["leaves"], st["x"], st["weight"], st["bias"]
    n, m, grad = case["n"], case["m"], case["grad"]
    key, order = torch.sort(leaves)
    ends = torch.searchsorted(key, torch.arange(-1, case["leaves"], device=key.device), right=True)
    ends = ends.tolist()
    y = torch.zeros((n, m), dtype=torch.float32, device=x.device)
    if grad:
        dx = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
        dw = torch.zeros(w.shape, dtype=torch.float32, device=x.device)
        db = torch.zeros((case["leaves"], m), dtype=torch.float32, device=x.device)
    for g in range(case["leaves"]):
        if ends[g] == ends[g + 1]:
            continue
        rows = order[ends[g] : ends[g + 1]]
        xg, wg = x[rows].float(), w[g].float()
        yg = xg @ wg.t()
        y[rows] = yg if b is None else yg + b[g].float()
        if grad:
            dyg = st["dy"][rows].float()
            dx[rows] = dyg @ wg
            dw[g] = dyg.t() @ xg
            if b is not None:
                db[g] = dyg.double().sum(0).float()
    dt = x.dtype
    if not grad:
        return y.to(dt)
    out = (y.to(dt), dx.to(dt), dw.to(dt))
    return out if b is None else (*out, db.to(dt))


def exact(case, seed):
    """The outputs from the definitions in 64 bits, one leaf after the other."""
    st = prepare(case, seed)
    leaves = st["leaves"]
    if case["op"] == "embed":
        table, d = st["table"].detach().double(), case["d"]
        kept = torch.nonzero(leaves >= 0).flatten()
        y = torch.zeros((case["n"], d), dtype=torch.float64, device=leaves.device)
        y[kept] = table.index_select(0, leaves[kept]) * case["scale"]
        if not case["grad"]:
            return y
        # one column block at a time: a sorted running sum would lose digits, a scatter does not
        dtable = torch.zeros_like(table)
        for a in range(0, d, 256):
            part = st["dy"][kept, a : a + 256].double() * case["scale"]
            where = leaves[kept][:, None].expand(-1, part.shape[1]).contiguous()
            block = torch.zeros((case["leaves"], part.shape[1]), dtype=torch.float64,
                                device=leaves.device)
            dtable[:, a : a + 256] = block.scatter_add_(0, where, part)
        return y, dtable
    x, w = st["x"].detach(), st["weight"].detach()
    b = None if st["bias"] is None else st["bias"].detach()
    f64 = {"dtype": torch.float64, "device": x.device}
    y = torch.zeros((case["n"], case["m"]), **f64)
    if case["grad"]:
        dx, dw = torch.zeros(x.shape, **f64), torch.zeros(w.shape, **f64)
        db = torch.zeros((case["leaves"], case["m"]), **f64)
    for g in range(case["leaves"]):
        rows = torch.nonzero(leaves == g).flatten()
        if rows.numel() == 0:
            continue
        wt = w[g].double().t().contiguous()
        xg = x.index_select(0, rows).double()
        yg = torch.mm(xg, wt)
        if b is not None:
            yg += b[g].double()
        y.index_copy_(0, rows, yg)
        if case["grad"]:
            dyg = st["dy"].index_select(0, rows).double()
            dx.index_copy_(0, rows, torch.mm(dyg, w[g].double()))
            dw[g] = torch.mm(xg.t().contiguous(), dyg).t()
            db[g] = dyg.sum(0)
    if not case["grad"]:
        return y
    return (y, dx, dw) if b is None else (y, dx, dw, db)
