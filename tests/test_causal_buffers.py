"""The causal mixer's frequencies and decays through moves of the module."""

from __future__ import annotations

import copy

import pytest
import torch

from lsso_amd.ball import CausalMixer, rotary_frequencies


def test_what_a_program_writes_is_kept() -> None:
    given = rotary_frequencies(8)
    mixer = CausalMixer(64, 4, frequencies=given)
    mixer.log_decay.fill_(-0.5)
    mixer.frequencies.mul_(0.25)
    for moved in (copy.deepcopy(mixer).half(), copy.deepcopy(mixer).double(), copy.deepcopy(mixer).to("cpu").float()):
        assert moved.log_decay.dtype == torch.float32 and torch.equal(moved.log_decay, torch.full((4,), -0.5))
        assert moved.frequencies.dtype == torch.float64 and torch.equal(moved.frequencies, given / 4)
    assert torch.equal(given, rotary_frequencies(8))   # the caller's own tensor
    copied = copy.deepcopy(mixer)
    copied.half().log_decay.fill_(-1.0)
    assert torch.equal(mixer.log_decay, torch.full((4,), -0.5))


def test_values_are_not_made_up() -> None:
    """A module without storage has no decays to move: it says so."""

    with torch.device("meta"):
        mixer = CausalMixer(64, 4)
    assert mixer.frequencies.is_meta and mixer.w_o.weight.is_meta
    with pytest.raises(NotImplementedError):
        mixer.to_empty(device="cpu")


@pytest.mark.gpu
def test_made_on_the_device(native) -> None:
    with torch.device("cuda"):
        mixer = CausalMixer(64, 4)
    assert mixer.frequencies.is_cuda and mixer.log_decay.is_cuda
    x = torch.randn(1, 5, 64, device="cuda").half()
    torch.manual_seed(0)
    other = CausalMixer(64, 4)
    other.load_state_dict({name: value.cpu() for name, value in mixer.state_dict().items()})
    assert torch.equal(other.cuda()(x, implementation="hip"), mixer(x, implementation="hip"))
