"""Batches without a sequence and sequences without a token, through the causal mixer
and group norm, as the other sizes."""

from __future__ import annotations

import pytest
import torch

from lsso_amd.ball import CausalMixer, GroupNorm


def _run(device, implementation, dtype):
    torch.manual_seed(0)
    mixer = CausalMixer(64, 4, kv_heads=2).to(device)
    for shape in ((0, 3, 64), (2, 0, 64), (0, 0, 64)):
        x = torch.zeros(shape, dtype=dtype, device=device, requires_grad=True)
        for mask in (None, torch.ones(shape[:2], dtype=torch.bool, device=device)):
            y, state = mixer(x, mask, return_state=True, implementation=implementation)
            assert y.shape == shape and state.shape == (shape[0], 4, 16, 16) and not state.any()
            assert torch.autograd.grad(y.sum(), x)[0].shape == shape
    state = mixer.initial_state(0)
    none = torch.zeros(0, dtype=torch.int64, device=device)
    assert mixer.step(torch.zeros(0, 64, dtype=dtype, device=device), state, none,
                      implementation=implementation).shape == (0, 64)
    norm = GroupNorm(4, 64).to(device)
    for shape in ((0, 64), (0, 3, 64), (2, 0, 64), (0, 2, 3, 64)):
        y = norm(torch.zeros(shape, dtype=dtype, device=device), implementation=implementation)
        grads = torch.autograd.grad(y.sum(), tuple(norm.parameters()))
        assert y.shape == shape and not any(grad.any() for grad in grads)


def test_a_state_that_no_token_changes_is_a_copy() -> None:
    """Steps change the state that a prompt returned in place, an empty one's too."""

    mixer = CausalMixer(64, 4, kv_heads=2)
    first = torch.randn(1, 4, 16, 16)
    kept = first.clone()
    with torch.no_grad():
        _, state = mixer(torch.zeros(1, 0, 64), state=first, return_state=True)
        assert torch.equal(state, first)
        mixer.step(torch.randn(1, 64), state, torch.zeros(1, dtype=torch.int64))
    assert torch.equal(first, kept) and not torch.equal(state, kept)


def test_reference() -> None:
    _run("cpu", "reference", torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_native(native, dtype) -> None:
    _run("cuda", "hip", dtype)
