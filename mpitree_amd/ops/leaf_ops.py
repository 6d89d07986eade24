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
stream, without host synchronisation, so calls can be captured into a graph (one with a backward
pass: while no eager autograd graph of the same parameters is alive, as for every operator of
torch). They give first derivatives in reverse mode; operands with a forward-mode tangent, tensors
without memory of their own (fake, functional or wrapped ones) and tracing (``make_fx``,
``torch.jit.trace``) are refused. CPU tensors take a plain path of the same results.
"""

from __future__ import annotations

import torch
import torch.autograd.forward_ad as fwad

from . import native

__all__ = ["LeafRoute", "leaf_route", "leaf_embedding", "leaf_linear"]

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MAX_ROWS = 2 ** 31 - 1
_MAX_LEAVES = 2 ** 30
_MAX_WIDTH = 2 ** 20
_MAX_F32 = torch.finfo(torch.float32).max


class LeafRoute:
    """Rows sorted by leaf, from :func:`leaf_route`: ``order[offsets[g]:offsets[g + 1]]`` are leaf
    ``g``'s rows in their order, for ``g == n_leaves`` the rows without a leaf.

    ``leaves`` is its own copy of the leaf numbers it was made from, ``keys`` [n] the leaf at each
    sorted position (``n_leaves``: none), ``order`` [n] and ``offsets`` [n_leaves + 2]: int32
    tensors, not to be written. It stays as it is when the numbers are changed later."""

    __slots__ = ("leaves", "n_leaves", "_buf")

    def __init__(self, leaves: torch.Tensor, n_leaves: int, buf: torch.Tensor):
        self.leaves, self.n_leaves, self._buf = leaves, n_leaves, buf

    @property
    def order(self) -> torch.Tensor:
        return self._buf[: self.leaves.numel()]

    @property
    def keys(self) -> torch.Tensor:
        n = self.leaves.numel()
        return self._buf[n : 2 * n]

    @property
    def offsets(self) -> torch.Tensor:
        return self._buf[2 * self.leaves.numel() :]

    @property
    def counts(self) -> torch.Tensor:
        """Rows of each leaf, int32 [n_leaves]."""
        off = self.offsets
        return off[1 : self.n_leaves + 1] - off[: self.n_leaves]

    def __repr__(self):
        return (f"LeafRoute({self.leaves.numel()} rows, {self.n_leaves} leaves, "
                f"device={self.leaves.device})")


def _check_leaves(leaves) -> torch.Tensor:
    if not isinstance(leaves, torch.Tensor):
        raise TypeError(f"leaves must be a tensor or a LeafRoute, got {type(leaves).__name__}")
    if leaves.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"leaves must be int32 or int64, got {leaves.dtype}")
    if leaves.numel() > _MAX_ROWS:
        raise ValueError(f"at most {_MAX_ROWS} rows, got {leaves.numel()}")
    return leaves


def _check_n_leaves(n_leaves) -> int:
    if type(n_leaves) is not int:
        try:
            whole = int(n_leaves) == n_leaves
        except (TypeError, ValueError, OverflowError):
            whole = False
        if not whole:
            raise TypeError(f"n_leaves must be a whole number, got {n_leaves!r}")
        n_leaves = int(n_leaves)
    if not 1 <= n_leaves <= _MAX_LEAVES:
        raise ValueError(f"n_leaves must be in [1, {_MAX_LEAVES}], got {n_leaves}")
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
    return t.resolve_neg() if t.is_neg() else t


def _check_width(what: str, width: int):
    if not 1 <= width <= _MAX_WIDTH:
        raise ValueError(f"{what} must be in [1, {_MAX_WIDTH}], got {width}")


def _check_device(first, *others):
    dev = first.get_device()  # (numbers: a third of the time; the same one for all but GPUs)
    for t in others:
        if t is not None and (t.get_device() != dev or dev < 0 and t.device != first.device):
            raise ValueError(f"operands on different devices: {first.device}, {t.device}")


def _check_launch(*operands):
    """The kernels take addresses, which say nothing of what torch keeps beside a tensor."""
    native.check_memory(*operands)
    if fwad._current_level >= 0:
        for t in operands:
            if t is not None and fwad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the leaf operators have no forward-mode derivative on CUDA "
                                   "tensors: an operand has a tangent")


def _stream(dev: int) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


# (the same handle without a Stream object around it, where this torch has it: 1.7 us a call)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream)


def _scratch(nbytes: int, like: torch.Tensor) -> torch.Tensor:
    return like.new_empty(nbytes, dtype=torch.uint8)


def _flat(t: torch.Tensor) -> torch.Tensor:
    """[..., C] as [rows, C] with unit column stride (any row stride)."""
    if t.dim() != 2:  # (a view would be one more node for autograd to walk)
        t = t.reshape(-1, t.shape[-1])
    stride, step = t.stride()
    return t if step == 1 or t.shape[1] == 1 and stride >= 0 else t.contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The same of an incoming gradient, whose sign may be known to the tensor only (the imaginary
    part of a conjugate)."""
    return _flat(t.resolve_neg() if t.is_neg() else t)


# -------------------------------------------------------------------------------- route
def leaf_route(leaves: torch.Tensor, n_leaves: int) -> LeafRoute:
    """Sort the rows by leaf (stable). ``leaves``: int32 or int64 of any shape."""
    leaves = _check_leaves(leaves).clone(memory_format=torch.contiguous_format)
    n_leaves = _check_n_leaves(n_leaves)
    return LeafRoute(leaves, n_leaves, _sort(leaves, n_leaves))


def _sort(leaves: torch.Tensor, n_leaves: int) -> torch.Tensor:
    """A route's buffer: order [n], keys [n], offsets [n_leaves + 2], int32."""
    ids = leaves if leaves.dim() == 1 else leaves.reshape(-1)
    n = ids.numel()
    if not ids.is_cuda:
        key = torch.where((ids >= 0) & (ids < n_leaves), ids, n_leaves).to(torch.int64)
        key, order = torch.sort(key, stable=True)
        bounds = torch.arange(n_leaves + 1, dtype=torch.int64)
        offsets = torch.cat([torch.searchsorted(key, bounds), torch.tensor([n])])
        return torch.cat([order, key, offsets]).int()
    _check_launch(ids)
    hip, dev, ids = native.hip(), ids.get_device(), ids.contiguous()
    buf = ids.new_empty(hip.leaf_route_len(n, n_leaves), dtype=torch.int32)
    work = _scratch(4 * hip.leaf_route_words(n, n_leaves), ids)
    hip.leaf_route(dev, _stream(dev), ids.data_ptr(), ids.dtype == torch.int64, n, n_leaves,
                   buf.data_ptr(), work.data_ptr())
    return buf


# ---------------------------------------------------------------------------- embedding
def _embed_forward(ids: torch.Tensor, table: torch.Tensor, scale: float) -> torch.Tensor:
    V, D = table.shape
    if not ids.is_cuda:
        flat = ids.reshape(-1)
        has = (flat >= 0) & (flat < V)
        y = table[torch.where(has, flat, 0)].float() * scale
        return torch.where(has[:, None], y, 0.0).to(table.dtype).reshape(*ids.shape, D)
    _check_launch(table, ids)
    n = ids.numel()
    y = table.new_empty((n, D) if ids.dim() == 1 else (*ids.shape, D))
    stride, step = table.stride()
    if D > 1 and step != 1:
        table, stride = table.contiguous(), D
    ids, dev = ids.contiguous(), table.get_device()
    native.hip().leaf_embed(dev, _stream(dev), _TYPES[table.dtype], ids.data_ptr(),
                            ids.dtype == torch.int64, table.data_ptr(), stride, n, V, D, scale,
                            y.data_ptr())
    return y


def _sum_by_leaf_plain(dy, buf, V: int, scale: float) -> torch.Tensor:
    n = dy.shape[0]
    out = torch.zeros((V + 1, dy.shape[1]), dtype=torch.float64)
    out.index_add_(0, buf[n : 2 * n].long(), dy[buf[:n].long()].double())
    scale = torch.tensor(scale, dtype=torch.float32).double()  # as the forward pass has it
    return (out[:V] * scale).to(dy.dtype)


def _embed_grad(dy, ids, buf, n_leaves: int, scale: float) -> torch.Tensor:
    """scale * the sum of dy's rows of each leaf, [n_leaves, D], from the leaf numbers or a route's
    buffer."""
    n, D = dy.shape if dy.dim() == 2 else (dy.numel() // dy.shape[-1], dy.shape[-1])
    if not dy.is_cuda:
        buf = buf if buf is not None else _sort(ids, n_leaves)
        return _sum_by_leaf_plain(dy.reshape(-1, D), buf, n_leaves, scale)
    _check_launch(dy)
    _check_device(dy, ids, buf)  # (saved tensors come back as their hooks leave them)
    hip, kind, dev, dy = native.hip(), _TYPES[dy.dtype], dy.get_device(), _rows(dy)
    out = dy.new_empty((n_leaves, D))
    work = _scratch(hip.leaf_embed_grad_bytes(kind, n, n_leaves, D, buf is not None), dy)
    if buf is None:
        ids = ids.contiguous()
        at, wide, sorted_ = ids.data_ptr(), ids.dtype == torch.int64, 0
    else:
        at, wide, sorted_ = 0, False, buf.data_ptr()
    hip.leaf_embed_grad(dev, _stream(dev), kind, dy.data_ptr(), dy.stride()[0], at, wide, sorted_,
                        n, n_leaves, D, scale, out.data_ptr(), work.data_ptr())
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, buf, scale):
        ctx.rest = buf is not None, table.shape[0], scale
        ctx.save_for_backward(ids if buf is None else buf)
        return _embed_forward(ids, table, scale)

    @staticmethod
    def _first(ctx, dy):
        (kept,), (routed, n_leaves, scale) = ctx.saved_tensors, ctx.rest
        ids, buf = (None, kept) if routed else (kept, None)
        return _embed_grad(dy, ids, buf, n_leaves, scale), None, None, None

    _marked = torch.autograd.function.once_differentiable(_first.__func__)

    @staticmethod
    def backward(ctx, dy):
        # (with create_graph only: the marking costs 4 us)
        return (_Embedding._marked if torch.is_grad_enabled() else _Embedding._first)(ctx, dy)


def leaf_embedding(leaves, table: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[leaves]``: one row of ``table`` [n_leaves, D] per leaf number.

    Returns ``leaves.shape + (D,)`` in the table's type. The gradient of ``table`` is dense: for
    each leaf ``scale`` times the sum over its rows, zeros for a leaf that no row reached.
    ``scale`` is taken in float32, where it has to be finite."""
    table = _check_params("table", table, ndim=2)
    route = leaves if isinstance(leaves, LeafRoute) else None
    ids = _check_leaves(leaves) if route is None else route.leaves
    n_leaves, D = table.shape
    _check_n_leaves(n_leaves)
    if route is not None and route.n_leaves != n_leaves:
        raise ValueError(f"table has {n_leaves} rows, the route {route.n_leaves} leaves")
    _check_width("the table's width", D)
    _check_device(ids, table)
    scale = float(scale)
    if not -_MAX_F32 <= scale <= _MAX_F32:
        raise ValueError(f"scale must be finite in float32, got {scale}")
    if table.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(table, ids, None if route is None else route._buf, scale)
    return _embed_forward(ids, table, scale)


# ------------------------------------------------------------------------------- linear
def _leaf_rows(buf, n: int, G: int):
    """(leaf, its rows) of the leaves that have rows."""
    order, bounds = buf[:n].long(), buf[2 * n :].tolist()
    for g in torch.unique(buf[n : 2 * n]).tolist():
        if g < G:
            yield g, order[bounds[g] : bounds[g + 1]]


def _linear_plain(x, buf, w, b):
    y = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float32)
    for g, rows in _leaf_rows(buf, x.shape[0], w.shape[0]):
        out = x[rows].float() @ w[g].float().t()
        y[rows] = out if b is None else out + b[g].float()
    return y.to(x.dtype)


def _linear_plain_grad(dy, x, buf, w, need_x, need_w):
    dx = torch.zeros(x.shape, dtype=torch.float32) if need_x else None
    dw = torch.zeros(w.shape, dtype=torch.float32) if need_w else None
    for g, rows in _leaf_rows(buf, x.shape[0], w.shape[0]):
        d = dy[rows].float()
        if need_x:
            dx[rows] = d @ w[g].float()
        if need_w:
            dw[g] = d.t() @ x[rows].float()
    return (dx.to(x.dtype) if need_x else None), (dw.to(w.dtype) if need_w else None)


def _linear_forward(x, ids, buf, w, b):
    """Returns (y, the route's buffer); it is made where the kernel needs one and none is given."""
    (n, K), (G, N, _) = x.shape, w.shape
    if not x.is_cuda:
        buf = buf if buf is not None else _sort(ids, G)
        with torch.autocast("cpu", enabled=False):  # (32-bit products, as the kernels')
            return _linear_plain(x, buf, w, b), buf
    _check_launch(x, w, b, ids)
    hip, kind, dev, ids = native.hip(), _TYPES[x.dtype], x.get_device(), ids.contiguous()
    wide, bias = ids.dtype == torch.int64, 0 if b is None else b.data_ptr()
    y, (stride, _) = x.new_empty((n, N)), x.stride()
    if n <= hip.LEAF_LINEAR_SMALL_ROWS:
        hip.leaf_linear_small(dev, _stream(dev), kind, x.data_ptr(), stride, ids.data_ptr(), wide,
                              n, G, w.data_ptr(), bias, K, N, y.data_ptr())
        return y, buf
    work = _scratch(hip.leaf_linear_bytes(kind, x.data_ptr(), stride, w.data_ptr(), n, G, K, N,
                                          buf is not None), x)
    sort = 0
    if buf is None:
        sort = ids.data_ptr()
        buf = ids.new_empty(hip.leaf_route_len(n, G), dtype=torch.int32)
    hip.leaf_linear(dev, _stream(dev), kind, x.data_ptr(), stride, sort, wide, buf.data_ptr(), n,
                    G, w.data_ptr(), bias, K, N, y.data_ptr(), work.data_ptr())
    return y, buf


def _linear_grad(dy, x, buf, w, need_x, need_w, need_b):
    _check_launch(dy, x, w)
    _check_device(dy, x, w, buf)  # (saved tensors come back as their hooks leave them)
    if not x.dtype == w.dtype == dy.dtype:
        raise TypeError(f"saved tensors are {x.dtype} and {w.dtype}, the gradient {dy.dtype}")
    dy, x, w = _rows(dy), _flat(x), w.contiguous()
    (n, K), (G, N, _) = x.shape, w.shape
    hip, kind, dev = native.hip(), _TYPES[x.dtype], x.get_device()
    dx = x.new_empty((n, K)) if need_x else None
    dw = x.new_empty((G, N, K)) if need_w else None
    db = x.new_empty((G, N)) if need_b else None
    ops = kind, x.data_ptr(), x.stride()[0], dy.data_ptr(), dy.stride()[0]
    at = w.data_ptr()
    work = _scratch(hip.leaf_linear_grad_bytes(*ops, at, n, G, K, N, need_x, need_w, need_b), x)
    hip.leaf_linear_grad(dev, _stream(dev), *ops, buf.data_ptr(), n, G, at, K, N,
                         0 if dx is None else dx.data_ptr(), 0 if dw is None else dw.data_ptr(),
                         0 if db is None else db.data_ptr(), work.data_ptr())
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, ids, buf):
        y, buf = _linear_forward(x, ids, buf, w, b)
        ctx.routed = buf is not None
        ctx.save_for_backward(x, w, buf if ctx.routed else ids)
        return y

    @staticmethod
    def _first(ctx, dy):
        x, w, kept = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        buf = kept if ctx.routed else _sort(kept, w.shape[0])
        if dy.is_cuda:
            grads = _linear_grad(dy, x, buf, w, need_x, need_w, need_b)
        else:
            with torch.autocast("cpu", enabled=False):
                grads = _linear_plain_grad(dy, x, buf, w, need_x, need_w)
            grads += (_sum_by_leaf_plain(dy, buf, w.shape[0], 1.0) if need_b else None,)
        return (*grads, None, None)

    _marked = torch.autograd.function.once_differentiable(_first.__func__)

    @staticmethod
    def backward(ctx, dy):
        return (_Linear._marked if torch.is_grad_enabled() else _Linear._first)(ctx, dy)


def leaf_linear(inputs: torch.Tensor, leaves, weight: torch.Tensor, bias=None) -> torch.Tensor:
    """``inputs[i] @ weight[g].T + bias[g]`` for the leaf ``g = leaves[i]`` of each row.

    ``inputs`` is ``leaves.shape + (K,)``, ``weight`` [n_leaves, N, K], ``bias`` [n_leaves, N] or
    None; returns ``leaves.shape + (N,)``. Rows may be strided as long as their columns are not."""
    weight = _check_params("weight", weight, ndim=3)
    inputs = _check_params("inputs", inputs, like=weight)
    route = leaves if isinstance(leaves, LeafRoute) else None
    ids = _check_leaves(leaves) if route is None else route.leaves
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
    x, weight = _flat(inputs), weight.contiguous()
    buf = None if route is None else route._buf
    one = ids.dim() == 1
    flat = ids if one else ids.reshape(-1)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or bias is not None and bias.requires_grad):
        y = _Linear.apply(x, weight, bias, flat, buf)
    else:
        y = _linear_forward(x, flat, buf, weight, bias)[0]
    return y if one else y.reshape(*ids.shape, N)
