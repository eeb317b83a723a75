"""Group norm of tokens of more channels than a wave holds: by a workgroup each, with
workspaces of their parameter gradients alone."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lsso_amd.ball import causal, hip
from test_group_norm import ACTIVATIONS, TYPES, _check, _inputs


@pytest.mark.parametrize("channels,groups", [(2048, 1), (4096, 1), (8192, 1), (16384, 2), (1023, 1), (4098, 2)])
def test_workspaces_do_not_grow_with_the_tokens(channels, groups) -> None:
    """Nothing forward; backward two rows of channels of each of up to 1,024 workgroups."""

    library = hip.open_library()
    sizes = [ctypes.c_size_t() for _ in range(3)]
    shape = causal.GroupNormShape(65536, 1, channels, groups, 1, 3, 0, 1e-5)
    assert library.lsso_hip_group_norm_sizes(ctypes.byref(shape), *map(ctypes.byref, sizes)) == 0
    assert sizes[0].value == 0 and sizes[1].value == 0 and sizes[2].value <= 1024 * 2 * 4 * channels + 256


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("shape,groups", [((5, 2056), 1), ((3, 4096), 1), ((2, 8192), 1), ((3, 5000), 1), ((7, 515), 1),
                                          ((2, 1023), 1), ((3, 4098), 2), ((2, 12288), 3), ((2, 8200), 1)])
@pytest.mark.parametrize("masked", (False, True))
def test_wide_tokens(native, dtype, activation, shape, groups, masked) -> None:
    x, weight, bias, dy, generator = _inputs(shape, dtype, seed=4)
    mask = torch.rand(shape[0], generator=generator) < 0.6 if masked else None
    _check(native, x, groups, weight, bias, dy, activation, mask)


@pytest.mark.gpu
def test_more_wide_tokens_than_workgroups(native) -> None:
    x, weight, bias, dy, generator = _inputs((2100, 2064), torch.bfloat16, seed=5)
    _check(native, x, 1, weight, bias, dy, "silu", torch.rand(2100, generator=generator) < 0.6)


@pytest.mark.gpu
def test_wide_tokens_repeat(native) -> None:
    x, weight, bias, dy, _ = _inputs((3000, 4096), torch.bfloat16)
    leaves = [t.cuda().requires_grad_() for t in (x, weight, bias)]
    dy = dy.cuda()
    results = []
    for _ in range(4):
        y = native.group_norm(leaves[0], 1, *leaves[1:], activation="silu")
        results.append([y, *torch.autograd.grad(y, leaves, dy)])
    for result in results[1:]:
        for a, b in zip(results[0], result):
            assert torch.equal(a, b)
