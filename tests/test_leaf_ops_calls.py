"""Calls of the operators over a tree's leaves that have to be right or refused."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from mpitree_amd import leaf_embedding, leaf_linear, leaf_route
from mpitree_amd.ops import leaf_ops

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
        for leaves in (ids, leaf_route(ids, 3)):
            yield (lambda t, leaves=leaves: leaf_embedding(leaves, t, scale=0.5)), [b]
            yield (lambda x, w, b, leaves=leaves: leaf_linear(x, leaves, w, b)), [x, w, b]


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
