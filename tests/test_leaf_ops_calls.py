"""Calls of the operators over a tree's leaves that have to be right or refused."""

import pytest
import torch

from mpitree_amd import leaf_embedding

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
