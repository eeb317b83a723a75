"""Group norm in FP32: each token by itself to a few roundings, and the activations and
their slopes."""

from __future__ import annotations

import pytest
import torch

from test_group_norm import _act, _formula, _inputs


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((4000, 8), 2), ((2000, 100), 4), ((500, 768), 1), ((700, 30), 3), ((200, 1000), 2)])
def test_fp32_tokens(native, shape, groups) -> None:
    """xhat of a group of n: its mean by a tree of sums of 32 and fewer values a lane, of
    which each rounding (rms 2^-24 / sqrt(3) / 2 of a partial sum) reaches xhat by at most
    1 / sqrt(n); then a difference, 1 / sqrt of the variance (whose own sum adds less
    than one rounding more) and two products: about six roundings of rms 2^-25 each, 7.3e-8
    of the norm, where the mean is half of the spread.  dx: two more means and as many
    products again, 1.1e-7 of the terms that dx is a sum of: dn, its mean, and xhat times
    the mean of dn xhat, in which x and the mean are rounded before their difference.
    (Of a group of four, dx is half of its terms' size and less.)"""

    x, weight, bias, dy, _ = _inputs(shape, torch.float32)
    leaf = x.cuda().requires_grad_()
    y = native.group_norm(leaf, groups)
    (grad,) = torch.autograd.grad(y, leaf, dy.cuda())
    end = x.double().requires_grad_()
    ones, zeros = torch.ones(shape[1]).double(), torch.zeros(shape[1]).double()
    expected = _formula(end, groups, ones, zeros, 1e-5, None, None)
    (exact,) = torch.autograd.grad(expected, end, dy.double())
    expected = expected.detach()
    assert float((y.detach().cpu().double() - expected).norm() / expected.norm()) <= 7.3e-8
    parts, dn = (t.double().unflatten(-1, (groups, -1)) for t in (x, dy))
    mean = parts.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((parts - mean).square().mean(-1, keepdim=True) + 1e-5)
    normal = (parts - mean) * rstd
    rounded = (parts.abs() + mean.abs()) * rstd
    terms = dn.abs() + dn.mean(-1, keepdim=True).abs() + rounded * (dn * normal).mean(-1, keepdim=True).abs()
    terms = (rstd * terms).flatten(-2)
    assert float((grad.cpu().double() - exact).norm() / terms.norm()) <= 1.1e-7


@pytest.mark.gpu
@pytest.mark.parametrize("size", (122, 126, 252, 504, 510))
def test_fp32_variances_are_divided(native, size) -> None:
    """Values of 3 and -3 by turns: a mean of 0 and a variance of 9, both exact, and 3
    times the rounded third is 1.  The sum times a rounded reciprocal is not 9 here."""

    x = torch.tensor([3.0, -3.0]).repeat(5, size // 2)
    y = native.group_norm(x.cuda(), 1, eps=0.0)
    assert torch.equal(y.cpu(), x / 3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ("silu", "gelu"))
@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("length", (None, 3))
def test_activations(native, activation, dtype, length) -> None:
    """Weights of zero make z the bias: act(z) and, as the bias' gradient for dy of one,
    act'(z), from -14 to 14.  FP32: a few roundings, and an exponential's of its argument
    (z^2 / 2 of GELU's density); 16-bit types: 1e-5 of the value before their rounding."""

    channels = 2048
    z = torch.linspace(-14.0, 14.0, channels)
    shape = (2, channels) if length is None else (1, length, channels)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    bias = z.cuda().requires_grad_()
    y = native.group_norm(x, 4, torch.zeros(channels, device="cuda"), bias, activation=activation)
    rows = y.numel() // channels
    (grad,) = torch.autograd.grad(y, bias, torch.ones_like(y))
    exact = z.double().requires_grad_()
    value = _act(exact, activation)
    (slope,) = torch.autograd.grad(value.sum(), exact)
    value = value.detach()
    fast = 0.0 if dtype == torch.float32 else 1e-5
    half = torch.finfo(dtype).eps / 2
    size = z.double().square() + 8
    bound = (half + fast + 2.0**-24 * size) * value.abs() + 2.0**-25
    assert ((y.detach().cpu().double().reshape(rows, -1) - value).abs() <= bound).all()
    # s + y (1 - s), Phi + z phi(z): terms of up to 1.2 that cancel.
    terms = 1.2 * (torch.sigmoid(exact) if activation == "silu" else torch.special.ndtr(exact)).detach() + (slope.abs())
    bound = (2.0**-24 * size + fast) * terms + 2.0**-24
    assert ((grad.cpu().double() / rows - slope).abs() <= bound).all()
