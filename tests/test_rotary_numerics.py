"""Rotary positions in FP32: sines of 64 bits, rounded once."""

from __future__ import annotations

import pytest
import torch

from lsso_amd.ball import rotary_frequencies
from test_rotary import _turned


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ("interleaved", "half"))
@pytest.mark.parametrize("far", (0, 10**6))
def test_fp32_is_rounded_as_its_sum(native, layout, far) -> None:
    """A sine and a cosine of half a rounding each (2^-25 of x and of x'), a product and
    the sum (2^-24 of the larger term and of y).  Angles rounded to 32 bits were off by
    up to 3 * 2^-25 alone."""

    generator = torch.Generator().manual_seed(3)
    x = torch.randn(2, 600, 3, 64, generator=generator)
    ids = far + torch.arange(600)
    f = rotary_frequencies(64)
    y, _ = native.rotary(x.cuda(), None, ids.cuda(), f.cuda(), layout=layout)
    expected = _turned(x, ids, f, layout)
    pairs = x.double().abs()
    pairs = pairs.unflatten(-1, (2, -1)).mT if layout == "half" else pairs.unflatten(-1, (-1, 2))
    terms = 2.0**-25 * pairs.sum(-1, keepdim=True) + 2.0**-24 * pairs.amax(-1, keepdim=True)
    terms = terms.expand(pairs.shape)
    bound = (terms.mT if layout == "half" else terms).flatten(-2) + 2.0**-24 * expected.abs()
    off = (y.cpu().double() - expected).abs()
    assert (off <= bound * (1 + 2.0**-20)).all()
    assert float((y.cpu().double() - expected).norm() / expected.norm()) <= 4.6e-8
