"""Calls of the operators over a tree's leaves that have to be right or refused."""

import gc
import warnings

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.checkpoint import checkpoint
from torch.utils.flop_counter import FlopCounterMode

from mpitree_amd import (DecisionTreeClassifier, LeafRoute, leaf_embedding, leaf_linear,
                         leaf_route)
from mpitree_amd.ops import leaf_ops, native

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.float16, torch.bfloat16]
F32_MAX = torch.finfo(torch.float32).max


# ------------------------------------------------------------------------------- scale
@pytest.mark.parametrize("scale", [1e39, -1e39, 2 * F32_MAX, float("nan"), float("-inf")])
def test_scale_is_finite_in_32_bits(scale):
    # the operator multiplies in 32 bits: an infinite factor would make NaN of a row of zeros
    ids, t = torch.tensor([0, -1, 2]), torch.zeros(3, 5)
    with pytest.raises(ValueError, match="finite"):
        leaf_embedding(ids, t, scale=scale)
    with pytest.raises(ValueError, match="finite"):
        leaf_embedding(ids, t.requires_grad_(), scale=scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [F32_MAX, -F32_MAX, 2.0 ** -149, 1e-60])
def test_scale_at_the_ends_of_32_bits(device, scale):
    t = torch.tensor([[0.0, 1.0], [0.5, -0.25]], device=device, requires_grad=True)
    y = leaf_embedding(torch.tensor([0, 5, 1, 1], device=device), t, scale=scale)
    s = torch.tensor(scale, dtype=torch.float32)  # 1e-60: zero
    want = torch.tensor([[0.0, 1.0], [0.0, 0.0], [0.5, -0.25], [0.5, -0.25]]) * s
    assert torch.equal(y.detach().cpu(), want)
    (dt,) = torch.autograd.grad(y, t, torch.full_like(y, 0.25))
    assert torch.equal(dt.cpu(), torch.tensor([[0.25, 0.25], [0.5, 0.5]]) * s)


@pytest.mark.parametrize("device", DEVICES)
def test_scale_is_the_same_number_in_both_directions(device):
    # 0.1 rounded to 32 bits, in the forward pass and on the gradient's sum
    d = torch.randn(400, 3, generator=torch.Generator().manual_seed(1))
    t = d.clone().to(device).requires_grad_()
    y = leaf_embedding(torch.arange(400, device=device), t, scale=0.1)
    (dt,) = torch.autograd.grad(y, t, d.to(device))
    want = (d.double() * torch.tensor(0.1, dtype=torch.float32).double()).float()
    assert torch.equal(y.detach().cpu(), want)
    assert torch.equal(dt.cpu(), want)


# --------------------------------------------------------------------- forward-mode tangents
def operands(device, n=9, G=3, K=4, N=2):
    g = torch.Generator().manual_seed(n)
    return (torch.randint(-1, G, (n,), generator=g).to(device),
            *(torch.randn(*s, generator=g).to(device) for s in ((n, K), (G, N, K), (G, N))))


def forward_calls(device):
    """(call, its operands that may have a tangent) of each operator."""
    for n in (9, 90):  # the form for few rows and the tiles
        ids, x, w, b = operands(device, n)
        yield from calls_of(ids, x, w, b)
        yield from calls_of(leaf_route(ids, 3), x, w, b)


def calls_of(leaves, x, w, b):
    yield (lambda t: leaf_embedding(leaves, t, scale=0.5)), [b]
    yield (lambda x, w, b: leaf_linear(x, leaves, w, b)), [x, w, b]


@pytest.mark.gpu
def test_tangents_are_refused_on_the_gpu():
    # the kernels know nothing of them: the derivative would read as zero
    for call, args in forward_calls("cuda"):
        for k in range(len(args)):
            with fwad.dual_level():
                dual = list(args)
                dual[k] = fwad.make_dual(args[k], torch.ones_like(args[k]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*dual)
                with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                    call(*dual)
                call(*args)  # operands without one pass
        call(*args)


@pytest.mark.gpu
def test_tangents_of_an_incoming_gradient_are_refused_on_the_gpu():
    for call, args in forward_calls("cuda"):
        args = [a.clone().requires_grad_() for a in args]
        y = call(*args)
        with fwad.dual_level():
            dy = fwad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, args, dy)


def test_tangents_are_refused_before_a_launch():
    # what the calls above check first, here without a GPU
    t = torch.randn(3, 4)
    leaf_ops._check_launch(t, None)
    with fwad.dual_level():
        leaf_ops._check_launch(t, None)
        with pytest.raises(RuntimeError, match="forward-mode"):
            leaf_ops._check_launch(torch.arange(3), fwad.make_dual(t, t), None)
    leaf_ops._check_launch(t, None)


def test_tangents_on_the_cpu():
    # plain torch operations: the operators are linear in each operand
    for call, args in forward_calls("cpu"):
        for k in range(len(args)):
            with fwad.dual_level():
                dual = list(args)
                tangent = torch.ones_like(args[k])
                dual[k] = fwad.make_dual(args[k], tangent)
                got = fwad.unpack_dual(call(*dual)).tangent
            zero = list(args)
            zero[k] = torch.zeros_like(tangent)
            one = list(args)
            one[k] = tangent
            assert torch.allclose(got, call(*one) - call(*zero), atol=1e-5)


# ------------------------------------------- tensors without memory of their own, and tracing
def all_calls(device):
    ids = operands(device)[0]
    yield (lambda ids: leaf_route(ids, 3)), [ids]
    for call, args in forward_calls(device):
        yield call, args


class Wrapped(torch.Tensor):
    """A tensor whose operations are answered by its class."""

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        return NotImplemented


def test_fake_tensors_of_the_gpu_are_refused():
    # their address is 0
    with FakeTensorMode():
        ids = torch.zeros(100, dtype=torch.int64, device="cuda")
        x, w, b = (torch.zeros(*s, device="cuda") for s in ((100, 4), (3, 2, 4), (3, 2)))
        for call in (lambda: leaf_route(ids, 3), lambda: leaf_embedding(ids, b),
                     lambda: leaf_embedding(ids, b.requires_grad_()),
                     lambda: leaf_linear(x, ids, w, b), lambda: leaf_linear(x[:9], ids[:9], w)):
            with pytest.raises(TypeError, match="plain tensors"):
                call()
    for call in (lambda: leaf_embedding(ids, b), lambda: leaf_linear(x, ids, w)):
        with pytest.raises(TypeError, match="plain tensors"):
            call()


@pytest.mark.parametrize("device", DEVICES)
def test_what_a_launch_would_do_wrongly_is_refused(device):
    t = torch.zeros(3, 4, device=device)
    native.check_memory(t, None, torch.nn.Parameter(t))
    with pytest.raises(TypeError, match="plain tensors"):
        native.check_memory(t, t.as_subclass(Wrapped))
    with FakeTensorMode(), pytest.raises(RuntimeError, match="traced"):
        native.check_memory(t)
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises((RuntimeError, TypeError), match="traced|plain tensors"):
            make_fx(lambda x: (native.check_memory(x), x + 1)[1], tracing_mode=mode)(t)
    with pytest.raises(RuntimeError, match="jit.trace"):
        torch.jit.trace(lambda x: (native.check_memory(x), x + 1)[1], (t,))
    with FlopCounterMode(display=False):  # it watches and changes nothing
        native.check_memory(t)
    native.check_memory(t.as_subclass(type("Named", (torch.Tensor,), {})))


def test_null_addresses_are_refused():
    hip = native.hip()
    for call in (lambda: hip.leaf_route(0, 0, 0, True, 5, 3, 64, 0),
                 lambda: hip.leaf_route(0, 0, 64, True, 5, 3, 0, 0),
                 lambda: hip.leaf_embed(0, 0, 0, 64, True, 0, 4, 5, 3, 4, 1.0, 64),
                 lambda: hip.leaf_embed(0, 0, 0, 64, True, 64, 4, 5, 3, 4, 1.0, 0),
                 lambda: hip.leaf_embed_grad(0, 0, 0, 0, 4, 64, True, 0, 5, 3, 4, 1.0, 64, 64),
                 lambda: hip.leaf_embed_grad(0, 0, 0, 64, 4, 0, True, 0, 5, 3, 4, 1.0, 64, 64),
                 lambda: hip.leaf_linear_small(0, 0, 0, 0, 4, 64, True, 5, 3, 64, 0, 4, 2, 64),
                 lambda: hip.leaf_linear(0, 0, 0, 64, 4, 0, True, 64, 99, 3, 64, 0, 4, 2, 0, 64),
                 lambda: hip.leaf_linear_grad(0, 0, 0, 64, 4, 0, 2, 64, 99, 3, 64, 4, 2, 64, 64, 0,
                                              64)):
        with pytest.raises(RuntimeError, match="no memory of its own"):
            call()


@pytest.mark.gpu
def test_traced_and_wrapped_calls_are_refused_on_the_gpu():
    for call, args in all_calls("cuda"):
        want = call(*args)
        for mode in ("real", "fake", "symbolic"):
            with pytest.raises((RuntimeError, TypeError), match="traced|plain tensors"):
                make_fx(call, tracing_mode=mode)(*args)
        with pytest.raises(RuntimeError, match="jit.trace"):
            torch.jit.trace(call, tuple(args))
        # (wrappers that torch itself makes: an address of 0, or no address)
        with pytest.raises(RuntimeError, match="memory|storage"):
            torch.func.functionalize(call)(*args)
        with pytest.raises(RuntimeError, match="memory|storage"):
            torch.func.vmap(call)(*(a[None] for a in args))
        with FlopCounterMode(display=False):
            got = call(*args)
        if isinstance(want, torch.Tensor):
            assert torch.equal(got, want)


@pytest.mark.gpu
def test_traced_and_faked_gradients_are_refused_on_the_gpu():
    for call, args in forward_calls("cuda"):
        args = [a.clone().requires_grad_() for a in args]
        y = call(*args)
        dy = torch.ones_like(y)
        want = torch.autograd.grad(y, args, dy, retain_graph=True)
        with pytest.raises((RuntimeError, TypeError), match="traced|plain tensors"):
            make_fx(lambda d: torch.autograd.grad(y, args, d, retain_graph=True))(dy)
        for a, b in zip(want, torch.autograd.grad(y, args, dy)):
            assert torch.equal(a, b)


def test_an_estimator_refuses_fake_rows():
    X = torch.randn(80, 3, generator=torch.Generator().manual_seed(0))
    est = DecisionTreeClassifier(max_depth=3, device="cpu").fit(X.numpy(), (X[:, 0] > 0).long())
    with FakeTensorMode(), pytest.raises(TypeError, match="plain tensors"):
        est.leaf_route(torch.zeros(4, 3, device="cuda"))
    assert est.leaf_route(X).leaves.shape == (80,)


@pytest.mark.parametrize("device", DEVICES)
def test_inside_a_compiled_function(device):
    # torch.compile breaks its graph at the launches and calls them as they are
    for call, args in forward_calls(device):
        args = [a.clone().requires_grad_() for a in args]

        def step(*args):
            return call(*(a * 2 for a in args)) + 1

        y, want = torch.compile(step, backend="eager")(*args), step(*args)
        assert torch.equal(y, want)
        for a, b in zip(*(torch.autograd.grad(out.sum(), args) for out in (y, want))):
            assert torch.equal(a, b)
        torch._dynamo.reset()


# --------------------------------------------------------- views that torch negates when read
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [9, 90])
def test_lazily_negated_operands(device, n):
    # the imaginary part of a conjugate holds the other sign in memory
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-1, 3, (n,), generator=g).to(device)

    def pair(*shape):
        z = torch.randn(*shape, dtype=torch.complex64, generator=g).to(device)
        view = z.conj().imag
        assert view.is_neg()
        return view, view.clone()

    for K, N in ((1, 1), (1, 6), (6, 1), (6, 6)):
        (x, x0), (w, w0), (b, b0) = pair(n, K), pair(3, N, K), pair(3, N)
        dy, dy0 = pair(n, N)
        w1, b1 = torch._neg_view(-w0), torch._neg_view(-b0)  # (contiguous ones)
        assert torch.equal(w1, w0) and w1.is_contiguous()
        want = leaf_linear(x0, ids, w0, b0)
        assert torch.equal(leaf_linear(x, ids, w, b), want)
        assert torch.equal(leaf_linear(torch._neg_view(-x0), ids, w1, b1), want)
        assert torch.equal(leaf_embedding(ids, b), leaf_embedding(ids, b0))
        assert torch.equal(leaf_embedding(ids, b1), leaf_embedding(ids, b0))
        args = [a.requires_grad_() for a in (x0, w0, b0)]
        for op, wrt in ((lambda: leaf_linear(args[0], ids, *args[1:]), args),
                        (lambda: leaf_embedding(ids, args[2]), args[2:])):
            for got, ref in zip(torch.autograd.grad(op(), wrt, dy),
                                torch.autograd.grad(op(), wrt, dy0)):
                assert torch.equal(got, ref)


def test_rows_and_parameters_of_negated_views_are_materialised():
    # what reaches a launch, here without a GPU
    v = torch.randn(5, 1, dtype=torch.complex64).conj().imag
    assert v.is_neg() and not leaf_ops._rows(v).is_neg()
    assert torch.equal(leaf_ops._rows(v), v)
    assert not leaf_ops._check_params("table", v, ndim=2).is_neg()


# ------------------------------------------------------------------------- whole numbers
@pytest.mark.parametrize("n_leaves", [2.5, 0.9, "3", None, float("nan"), float("inf")])
def test_the_number_of_leaves_is_whole(n_leaves):
    with pytest.raises((TypeError, ValueError), match="n_leaves"):
        leaf_route(torch.zeros(4, dtype=torch.int64), n_leaves)


@pytest.mark.parametrize("n_leaves", [3, 3.0, np.int32(3), torch.tensor(3)])
def test_whole_numbers_of_any_type(n_leaves):
    r = leaf_route(torch.tensor([2, 0]), n_leaves)
    assert r.n_leaves == 3 and type(r.n_leaves) is int


# ----------------------------------------------------------------- what a graph keeps
def kept_by_hooks(call, args, device):
    """Runs call with its saved tensors moved to the host; their types and shapes, the gradients."""
    seen = []

    def pack(t):
        seen.append((t.dtype, t.numel()))
        return t.cpu().clone()

    args = [a.detach().clone().requires_grad_() for a in args]
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(device)):
        y = call(*args)
    routes = sum(type(o) is LeafRoute for o in gc.get_objects())
    return seen, routes, [y, *torch.autograd.grad(y.sum(), args)]


@pytest.mark.parametrize("device", DEVICES)
def test_saved_tensors_are_all_that_a_graph_keeps(device):
    # a route made inside a call too: hooks see it, and it goes with the saved tensors
    gc.collect()
    before = sum(type(o) is LeafRoute for o in gc.get_objects())
    ids, x, w, b = operands(device, 90)
    route = leaf_route(ids, 3)
    size = 2 * 90 + 3 + 2
    for leaves in (ids, route):
        for call, args, want in (
                (lambda t: leaf_embedding(leaves, t), [b],
                 [(torch.int32, size) if leaves is route else (torch.int64, 90)]),
                (lambda x, w, b: leaf_linear(x, leaves, w, b), [x, w, b],
                 [(torch.float32, x.numel()), (torch.float32, w.numel()), (torch.int32, size)])):
            seen, routes, got = kept_by_hooks(call, args, device)
            assert seen == want and routes == before + 1
            args = [a.detach().clone().requires_grad_() for a in args]
            y = call(*args)
            for p, q in zip(got, (y, *torch.autograd.grad(y.sum(), args))):
                assert torch.equal(p, q)


def test_a_rewritten_route_is_noticed():
    ids, x, w, b = operands("cpu", 90)
    route, b = leaf_route(ids, 3), b.requires_grad_()
    y, z = leaf_embedding(route, b), leaf_linear(x, route, w, b)
    route.order.zero_()
    for out in (y, z):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


@pytest.mark.gpu
def test_saved_tensors_that_come_back_elsewhere():
    # a hook that leaves them on the host is refused, one that returns other strides is not
    ids, x, w, b = operands("cuda", 90)
    for call, args in ((lambda t: leaf_embedding(ids, t), [b]),
                       (lambda x, w, b: leaf_linear(x, ids, w, b), [x, w, b])):
        args = [a.detach().clone().requires_grad_() for a in args]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
            y = call(*args)
        with pytest.raises((ValueError, RuntimeError), match="device"):
            torch.autograd.grad(y.sum(), args)
        with torch.autograd.graph.saved_tensors_hooks(
                lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
            y = call(*args)
        got = torch.autograd.grad(y.sum(), args)
        for p, q in zip(got, torch.autograd.grad(call(*args).sum(), args)):
            assert torch.equal(p, q)


# ----------------------------------------------------------------------------- scratch
def test_scratch_is_of_what_a_call_makes():
    # 65536 rows, 64 leaves, 2048 -> 2048 bf16: partial matrices with a weight gradient only
    h, at = native.hip(), 1 << 20
    n, G, K, N = 65_536, 64, 2048, 2048

    def grad(dx, dw, db):
        return h.leaf_linear_grad_bytes(2, at, K, at, N, at, n, G, K, N, dx, dw, db)

    assert grad(True, False, False) < 2 ** 14  # the tile list: 8 bytes for each 256 rows and leaf
    assert grad(False, False, False) == 0
    assert 0 < grad(False, False, True) == h.leaf_embed_grad_bytes(2, n, G, N, True)
    assert grad(True, True, False) >= 2 * N * K * 4
    assert grad(True, False, True) == max(grad(True, False, False), grad(False, False, True))
    assert grad(True, True, True) == max(grad(True, True, False), grad(False, False, True))

    def forward(n, K, N, routed):
        return h.leaf_linear_bytes(0, at, K, at, n, 4096, K, N, routed)

    assert forward(10 ** 6, 64, 64, True) == 0  # nothing is sorted, no tiles listed
    assert forward(10 ** 6, 64, 64, False) == 4 * h.leaf_route_words(10 ** 6, 4096)
    # operands that are copied into whole chunks are so in every call
    odd = [h.leaf_linear_grad_bytes(2, at, 2047, at, 2049, at, n, G, 2047, 2049, dx, dw, False)
           for dx, dw in ((True, False), (False, True))]
    assert odd[0] >= n * 2056 * 2 + G * 2049 * 2048 * 2 and odd[1] >= n * (2048 + 2056) * 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,G,K,N", [(90, 3, 6, 5), (5000, 4, 24, 40), (9000, 3, 200, 129),
                                     (9000, 3, 1032, 520), (1000, 2500, 64, 64)])
def test_every_subset_of_the_gradients(dtype, n, G, K, N):
    # each with the scratch that is its own; from leaf numbers and from a route
    g = torch.Generator().manual_seed(n + K)
    ids = torch.randint(-1, G, (n,), generator=g).cuda()
    # whole numbers of few bits: sums in any order are exact
    x, w, b, dy = (torch.randint(-2, 3, s, generator=g).to(dtype).cuda()
                   for s in ((n, K), (G, N, K), (G, N), (n, N)))
    for leaves in (ids, leaf_route(ids, G)):
        full = None
        for need in ("xwb", "x", "w", "b", "xw", "wb", "xb"):
            args = {k: t.detach().clone().requires_grad_(k in need)
                    for k, t in zip("xwb", (x, w, b))}
            y = leaf_linear(args["x"], leaves, args["w"], args["b"])
            got = dict(zip(need, torch.autograd.grad(y, [args[k] for k in need], dy)))
            full = full or (y, got)
            assert torch.equal(y, full[0])
            for k in need:
                assert torch.equal(got[k], full[1][k]), (need, k)


# ------------------------------------------------------------------ rows of an estimator
@pytest.mark.parametrize("device", DEVICES)
def test_an_estimator_takes_rows_of_any_layout(device):
    # what apply() takes: reversed, read-only, strided, lists, other types
    X = np.random.default_rng(0).normal(size=(90, 3)).astype(np.float32)
    est = DecisionTreeClassifier(max_depth=3, device="cpu").fit(X, X[:, 0] + X[:, 1] > 0)
    w = torch.randn(est.get_n_leaves(), 2, 3, device=device)
    fixed = X.copy()
    fixed.flags.writeable = False
    wide = np.zeros((90, 6), np.float32)
    wide[:, ::2] = X
    want = est.leaf_linear(X, w)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert torch.equal(est.leaf_linear(X[::-1], w), want.flip(0))
        assert torch.equal(est.leaf_linear(fixed, w), want)
        assert torch.equal(est.leaf_linear(np.asfortranarray(X), w), want)
        assert torch.equal(est.leaf_linear(wide[:, ::2], w), want)
        assert torch.equal(est.leaf_linear(X.tolist(), w), want)
        assert torch.equal(est.leaf_linear(X.astype(object), w), want)
        assert torch.equal(est.leaf_linear(torch.from_numpy(X), w), want)
        # (numpy's own bytes the other way round)
        assert torch.equal(est.leaf_linear(X.astype(">f4"), w), want)


# ------------------------------------------------------- inside torch's other machinery
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [9, 90])
def test_recomputed_in_the_backward_pass(device, n):
    ids, x, w, b = operands(device, n)
    for leaves in (ids, leaf_route(ids, 3)):
        args = [t.clone().requires_grad_() for t in (x, w, b)]

        def step(x, w, b):
            return leaf_linear(x, leaves, w, b) * leaf_embedding(leaves, b, scale=0.5)

        want = torch.autograd.grad(step(*args).sum(), args)
        y = checkpoint(step, *args, use_reentrant=False)
        for p, q in zip(torch.autograd.grad(y.sum(), args), want):
            assert torch.equal(p, q)


@pytest.mark.parametrize("device", DEVICES)
def test_in_inference_mode_and_autocast(device):
    for call, args in forward_calls(device):
        want = call(*args)
        with torch.inference_mode():
            assert torch.equal(call(*args), want)
        with torch.autocast(device, dtype=torch.bfloat16):  # the operands' types stay
            got = call(*args)
        assert got.dtype == want.dtype and torch.equal(got, want)
        args = [a.clone().requires_grad_() for a in args]
        want = torch.autograd.grad(call(*args).sum(), args)
        with torch.autocast(device, dtype=torch.bfloat16):
            for p, q in zip(torch.autograd.grad(call(*args).sum(), args), want):
                assert torch.equal(p, q)


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_kept_for_a_second_backward(device):
    for call, args in forward_calls(device):
        args = [a.clone().requires_grad_() for a in args]
        y = call(*args).square().sum()
        first = torch.autograd.grad(y, args, retain_graph=True)
        for p, q in zip(first, torch.autograd.grad(y, args)):
            assert torch.equal(p, q)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, args)
