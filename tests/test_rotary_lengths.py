"""Rotary positions of more tokens than 32 bits count."""

from __future__ import annotations

import pytest
import torch

from lsso_amd.ball import rotary_frequencies
from test_rotary import _bound, _turned


@pytest.mark.gpu
@pytest.mark.parametrize("length", (2**32, 2**32 + 3))
def test_more_tokens_than_32_bits(native, length) -> None:
    """One pair of features, broadcast over 2^32 tokens and more (16 GiB of output): the
    first, those about 2^32 and the last keep their own positions."""

    one = torch.tensor([1.0, -0.5], dtype=torch.float16, device="cuda").view(1, 1, 1, 2)
    f = rotary_frequencies(2).cuda()
    y, _ = native.rotary(one.expand(1, length, 1, 2), None, None, f)
    for first in (0, 2**31 - 3, length - 9):
        rows = torch.arange(first, first + 9)
        x = one.expand(1, 9, 1, 2)
        expected = _turned(x, rows, f, "interleaved")
        found = y[:, first:first + 9].cpu().double()
        assert ((found - expected).abs() <= _bound(expected, x, f, "interleaved", 1.0, torch.float16)).all()
