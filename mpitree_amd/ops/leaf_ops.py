"""Operators over a tree's leaves: what a leaf holds, beyond the class counts of ``predict``.

A fitted tree sends every row to a leaf (:meth:`apply`). These operators let the leaves hold
learned parameters, in training and in answering:

* :func:`leaf_embedding` -- one vector per leaf, looked up by each row's leaf and scaled; its
  gradient sums the rows of each leaf;
* :func:`leaf_linear` -- one matrix (and bias) per leaf, each row multiplied with its leaf's: linear
  models in the leaves, or the experts behind a router; with the gradients of rows, matrices and
  biases;
* :func:`leaf_route` -- the rows sorted by leaf, which both need for their gradients. A fitted
  tree's rows do not change leaves, so a training loop may keep the route and pass it in place of
  the leaf indices; passed the indices, the operators sort on every call.

``leaves`` is an integer tensor (int32 or int64) of any shape, numbering leaves from 0, or a
:class:`LeafRoute`. A row whose number is outside ``[0, n_leaves)`` has no leaf (padding): its
outputs are zeros and it contributes to no gradient. Parameters and rows are float32, float16 or
bfloat16, all of one type; sums are held in 32 bits (float32: 64 bits where only sums are formed)
and rounded once. Gradients do not depend on the launch: the same inputs give the same bits.

CUDA tensors run the gfx950 kernels (``ops/csrc/leaf_*.hip``) on the tensors' device and its current
stream, without host synchronisation, so calls can be captured into a graph; CPU tensors take a
plain path of the same results.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import native

__all__ = ["LeafRoute", "leaf_route", "leaf_embedding", "leaf_linear"]

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MAX_ROWS = 2 ** 31 - 1
_MAX_WIDTH = 2 ** 20


@dataclass(frozen=True)
class LeafRoute:
    """Rows sorted by leaf: ``order[offsets[g]:offsets[g + 1]]`` are leaf ``g``'s rows in their
    order, for ``g == n_leaves`` the rows without a leaf."""

    leaves: torch.Tensor  # the leaf numbers, as given
    n_leaves: int
    order: torch.Tensor  # int32 [n]
    keys: torch.Tensor  # int32 [n], the leaf at each sorted position (n_leaves: none)
    offsets: torch.Tensor  # int32 [n_leaves + 2]

    @property
    def counts(self) -> torch.Tensor:
        """Rows of each leaf, int32 [n_leaves]."""
        return self.offsets[1 : self.n_leaves + 1] - self.offsets[: self.n_leaves]


def _check_leaves(leaves) -> torch.Tensor:
    if not isinstance(leaves, torch.Tensor):
        raise TypeError(f"leaves must be a tensor or a LeafRoute, got {type(leaves).__name__}")
    if leaves.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"leaves must be int32 or int64, got {leaves.dtype}")
    if leaves.numel() > _MAX_ROWS:
        raise ValueError(f"at most {_MAX_ROWS} rows, got {leaves.numel()}")
    return leaves


def _check_n_leaves(n_leaves) -> int:
    n_leaves = int(n_leaves)
    if not 1 <= n_leaves <= _MAX_ROWS - 1:
        raise ValueError(f"n_leaves must be in [1, {_MAX_ROWS - 1}], got {n_leaves}")
    return n_leaves


def _check_params(what: str, t, like=None, ndim=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.dtype not in _TYPES:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{what} must have {ndim} dimensions, got shape {tuple(t.shape)}")
    if like is not None and t.dtype != like.dtype:
        raise TypeError(f"{what} is {t.dtype}, expected {like.dtype} as the other operands")
    return t


def _check_width(what: str, width: int):
    if not 1 <= width <= _MAX_WIDTH:
        raise ValueError(f"{what} must be in [1, {_MAX_WIDTH}], got {width}")


def _check_device(*tensors):
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        raise ValueError(f"operands on different devices: {sorted(map(str, devices))}")


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., C] as [rows, C] with unit column stride (any row stride)."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 and t.stride(0) >= 0 else t.contiguous()


# -------------------------------------------------------------------------------- route
def leaf_route(leaves: torch.Tensor, n_leaves: int) -> LeafRoute:
    """Sort the rows by leaf (stable). ``leaves``: int32 or int64 of any shape."""
    leaves = _check_leaves(leaves)
    n_leaves = _check_n_leaves(n_leaves)
    ids = leaves.detach().reshape(-1)
    n, dev = ids.numel(), ids.device
    if not ids.is_cuda:
        key = torch.where((ids >= 0) & (ids < n_leaves), ids, n_leaves).to(torch.int64)
        key, order = torch.sort(key, stable=True)
        bounds = torch.arange(n_leaves + 1, dtype=torch.int64)
        offsets = torch.cat([torch.searchsorted(key, bounds), torch.tensor([n])])
        return LeafRoute(leaves, n_leaves, order.int(), key.int(), offsets.int())
    hip = native.hip()
    with torch.cuda.device(dev):
        ids = ids.contiguous()
        buf = torch.empty(2 * n + n_leaves + 2, dtype=torch.int32, device=dev)
        order, keys, offsets = buf[:n], buf[n : 2 * n], buf[2 * n :]
        work = torch.empty(hip.leaf_route_words(n, n_leaves), dtype=torch.int32, device=dev)
        hip.leaf_route(_stream(ids), ids.data_ptr(), ids.dtype == torch.int64, n, n_leaves,
                       order.data_ptr(), keys.data_ptr(), offsets.data_ptr(), work.data_ptr())
    return LeafRoute(leaves, n_leaves, order, keys, offsets)


# ---------------------------------------------------------------------------- embedding
def _embed_forward(ids: torch.Tensor, table: torch.Tensor, scale: float) -> torch.Tensor:
    D = table.shape[1]
    if not ids.is_cuda:
        flat = ids.reshape(-1)
        has = (flat >= 0) & (flat < table.shape[0])
        y = table[torch.where(has, flat, 0)].float() * scale
        return torch.where(has[:, None], y, 0.0).to(table.dtype).reshape(*ids.shape, D)
    y = torch.empty((*ids.shape, D), dtype=table.dtype, device=ids.device)
    if table.stride(1) != 1 and D > 1:
        table = table.contiguous()
    ids = ids.contiguous()
    with torch.cuda.device(ids.device):
        native.hip().leaf_embed(_stream(ids), _TYPES[table.dtype], ids.data_ptr(),
                                ids.dtype == torch.int64, table.data_ptr(), table.stride(0),
                                ids.numel(), table.shape[0], D, scale, y.data_ptr())
    return y


def _sum_by_leaf(dy: torch.Tensor, route: LeafRoute, scale: float) -> torch.Tensor:
    """scale * the sum of dy's rows of each leaf, [n_leaves, D]."""
    V, D = route.n_leaves, dy.shape[-1]
    dy = dy.reshape(-1, D)
    if not dy.is_cuda:
        out = torch.zeros((V + 1, D), dtype=torch.float64)
        out.index_add_(0, route.keys.long(), dy[route.order.long()].double())
        return (out[:V] * scale).to(dy.dtype)
    dy = dy.contiguous()
    hip, n, kind = native.hip(), dy.shape[0], _TYPES[dy.dtype]
    with torch.cuda.device(dy.device):
        out = torch.empty((V, D), dtype=dy.dtype, device=dy.device)
        work = torch.empty(hip.leaf_embed_grad_bytes(kind, n, D), dtype=torch.uint8,
                           device=dy.device)
        hip.leaf_embed_grad(_stream(dy), kind, dy.data_ptr(), route.order.data_ptr(),
                            route.keys.data_ptr(), route.offsets.data_ptr(), n, V, D, scale,
                            out.data_ptr(), work.data_ptr())
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, route, scale):
        ctx.route, ctx.scale, ctx.n_leaves = route, scale, table.shape[0]
        ctx.save_for_backward(ids)
        return _embed_forward(ids, table, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        route = ctx.route if ctx.route is not None else leaf_route(ids, ctx.n_leaves)
        return _sum_by_leaf(dy, route, ctx.scale), None, None, None


def leaf_embedding(leaves, table: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[leaves]``: one row of ``table`` [n_leaves, D] per leaf number.

    Returns ``leaves.shape + (D,)`` in the table's type. The gradient of ``table`` is dense: for
    each leaf ``scale`` times the sum over its rows, zeros for a leaf that no row reached."""
    table = _check_params("table", table, ndim=2)
    route = leaves if isinstance(leaves, LeafRoute) else None
    ids = _check_leaves(leaves if route is None else route.leaves)
    n_leaves = _check_n_leaves(table.shape[0])
    if route is not None and route.n_leaves != n_leaves:
        raise ValueError(f"table has {n_leaves} rows, the route {route.n_leaves} leaves")
    _check_width("the table's width", table.shape[1])
    _check_device(ids, table)
    scale = float(scale)
    if scale - scale != 0.0:
        raise ValueError(f"scale must be finite, got {scale}")
    if table.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(table, ids, route, scale)
    return _embed_forward(ids, table, scale)


# ------------------------------------------------------------------------------- linear
def _linear_plain(x, route, w, b):
    y = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float32)
    bounds = route.offsets.tolist()
    for g in torch.unique(route.keys).tolist():
        if g < route.n_leaves:
            rows = route.order[bounds[g] : bounds[g + 1]].long()
            out = x[rows].float() @ w[g].float().t()
            y[rows] = out if b is None else out + b[g].float()
    return y.to(x.dtype)


def _linear_plain_grad(dy, x, route, w, need_x, need_w):
    dx = torch.zeros(x.shape, dtype=torch.float32) if need_x else None
    dw = torch.zeros(w.shape, dtype=torch.float32) if need_w else None
    bounds = route.offsets.tolist()
    for g in torch.unique(route.keys).tolist():
        if g < route.n_leaves:
            rows = route.order[bounds[g] : bounds[g + 1]].long()
            d = dy[rows].float()
            if need_x:
                dx[rows] = d @ w[g].float()
            if need_w:
                dw[g] = d.t() @ x[rows].float()
    return (dx.to(x.dtype) if need_x else None), (dw.to(w.dtype) if need_w else None)


def _linear_tile(dx: bool, src, route, w, bias) -> torch.Tensor:
    G, N, K = w.shape
    hip, n = native.hip(), src.shape[0]
    out = torch.empty((n, K if dx else N), dtype=src.dtype, device=src.device)
    work = torch.empty(hip.leaf_linear_tile_bytes(n, G), dtype=torch.uint8, device=src.device)
    hip.leaf_linear_tile(
        _stream(src), _TYPES[src.dtype], dx, src.data_ptr(), src.stride(0),
        route.order.data_ptr(), route.offsets.data_ptr(), n, G, w.data_ptr(),
        0 if bias is None else bias.data_ptr(), K, N, out.data_ptr(), work.data_ptr())
    return out


def _linear_forward(x, ids, route, w, b):
    """Returns (y, route): the route is built where the kernel needs one."""
    if not x.is_cuda:
        route = route if route is not None else leaf_route(ids, w.shape[0])
        return _linear_plain(x, route, w, b), route
    hip = native.hip()
    n, (G, N, K) = x.shape[0], w.shape
    with torch.cuda.device(x.device):
        if n <= hip.leaf_linear_small_rows():
            y = torch.empty((n, N), dtype=x.dtype, device=x.device)
            ids = ids.contiguous()
            hip.leaf_linear_small(_stream(x), _TYPES[x.dtype], x.data_ptr(), x.stride(0),
                                  ids.data_ptr(), ids.dtype == torch.int64, n, G, w.data_ptr(),
                                  0 if b is None else b.data_ptr(), K, N, y.data_ptr())
            return y, route
        route = route if route is not None else leaf_route(ids, G)
        return _linear_tile(False, x, route, w, b), route


def _linear_grad_weight(dy, x, route, w) -> torch.Tensor:
    G, N, K = w.shape
    hip, n = native.hip(), x.shape[0]
    dw = torch.empty((G, N, K), dtype=x.dtype, device=x.device)
    work = torch.empty(hip.leaf_linear_grad_bytes(_TYPES[x.dtype], n, G, K, N), dtype=torch.uint8,
                       device=x.device)
    hip.leaf_linear_grad(_stream(x), _TYPES[x.dtype], x.data_ptr(), x.stride(0), dy.data_ptr(),
                         dy.stride(0), route.order.data_ptr(), route.keys.data_ptr(),
                         route.offsets.data_ptr(), n, G, K, N, dw.data_ptr(), work.data_ptr())
    return dw


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, ids, route):
        y, ctx.route = _linear_forward(x, ids, route, w, b)
        ctx.save_for_backward(x, w, ids)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, ids = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        route = ctx.route if ctx.route is not None else leaf_route(ids, w.shape[0])
        if not x.is_cuda:
            dx, dw = _linear_plain_grad(dy, x, route, w, need_x, need_w)
        else:
            with torch.cuda.device(x.device):
                dy = _rows(dy)
                dx = _linear_tile(True, dy, route, w, None) if need_x else None
                dw = _linear_grad_weight(dy, x, route, w) if need_w else None
        db = _sum_by_leaf(dy, route, 1.0) if need_b else None
        return dx, dw, db, None, None


def leaf_linear(inputs: torch.Tensor, leaves, weight: torch.Tensor, bias=None) -> torch.Tensor:
    """``inputs[i] @ weight[g].T + bias[g]`` for the leaf ``g = leaves[i]`` of each row.

    ``inputs`` is ``leaves.shape + (K,)``, ``weight`` [n_leaves, N, K], ``bias`` [n_leaves, N] or
    None; returns ``leaves.shape + (N,)``. Rows may be strided as long as their columns are not."""
    weight = _check_params("weight", weight, ndim=3)
    inputs = _check_params("inputs", inputs, like=weight)
    route = leaves if isinstance(leaves, LeafRoute) else None
    ids = _check_leaves(leaves if route is None else route.leaves)
    G, N, K = weight.shape
    _check_n_leaves(G)
    _check_width("weight's rows", N)
    _check_width("weight's columns", K)
    if route is not None and route.n_leaves != G:
        raise ValueError(f"weight has {G} leaves, the route {route.n_leaves}")
    if inputs.shape != (*ids.shape, K):
        raise ValueError(f"inputs have shape {tuple(inputs.shape)}, expected "
                         f"{(*ids.shape, K)} for leaves {tuple(ids.shape)} and weight "
                         f"{tuple(weight.shape)}")
    if bias is not None:
        bias = _check_params("bias", bias, like=weight, ndim=2)
        if bias.shape != (G, N):
            raise ValueError(f"bias has shape {tuple(bias.shape)}, expected {(G, N)}")
        bias = bias.contiguous()
    _check_device(inputs, ids, weight, bias)
    x, weight, flat = _rows(inputs), weight.contiguous(), ids.reshape(-1)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or bias is not None and bias.requires_grad):
        y = _Linear.apply(x, weight, bias, flat, route)
    else:
        y = _linear_forward(x, flat, route, weight, bias)[0]
    return y.reshape(*ids.shape, N)
