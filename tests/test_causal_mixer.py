"""The causal mixer: its operators as one run, over whole sequences, from a prompt on
and token by token; trained, captured and moved; and its kernels' registers."""

from __future__ import annotations

import copy

import pytest
import torch

from lsso_amd import LSSO, LSSOConfig, build
from lsso_amd.ball import CausalMixer, GatedFeedForward, TokenEmbedding, rotary_frequencies
from test_kernel_resources import _code_objects, _kernels


def _mixer(**keywords):
    torch.manual_seed(0)
    return CausalMixer(64, 4, kv_heads=2, **keywords)


def test_is_causal_and_goes_on_from_a_state() -> None:
    mixer = _mixer(layout="half").double()
    x = torch.randn(2, 90, 64, dtype=torch.float64)
    whole, last = mixer(x, return_state=True)
    changed = x.clone()
    changed[:, 50:] = 0.0
    torch.testing.assert_close(mixer(changed)[:, :50], whole[:, :50])
    first, state = mixer(x[:, :70], return_state=True)
    rest, after = mixer(x[:, 70:], position_ids=torch.arange(70, 90), state=state, return_state=True)
    torch.testing.assert_close(torch.cat((first, rest), dim=1), whole)
    torch.testing.assert_close(after, last)
    state = state.double()
    for t in range(70, 90):
        y = mixer.step(x[:, t], state, torch.full((2,), t))
        torch.testing.assert_close(y, whole[:, t])
    torch.testing.assert_close(state, last)


def test_excluded_tokens_are_as_if_not_there() -> None:
    mixer = _mixer().double()
    x = torch.randn(1, 8, 64, dtype=torch.float64)
    kept = torch.tensor([[False, True, True, False, True, False, True, True]])
    y = mixer(x, kept)
    assert not y[~kept].any()
    expected = mixer(x[kept][None], position_ids=kept.nonzero()[:, 1])
    torch.testing.assert_close(y[kept], expected[0])


def test_moves_keep_what_is_fixed() -> None:
    mixer = _mixer(frequencies=rotary_frequencies(8, scaling="linear", factor=4.0))
    for moved in (copy.deepcopy(mixer).half(), copy.deepcopy(mixer).double(), copy.deepcopy(mixer).to(torch.bfloat16)):
        assert torch.equal(moved.frequencies, mixer.frequencies) and moved.frequencies.dtype == torch.float64
        assert torch.equal(moved.log_decay, mixer.log_decay) and moved.log_decay.dtype == torch.float32
    assert set(mixer.state_dict()) == {"w_in.weight", "w_o.weight", "norm.weight", "norm.bias"}
    assert (mixer.log_decay < 0).all() and mixer.initial_state(3).shape == (3, 4, 16, 16)
    for wrong in ({"dim": 65, "num_heads": 4}, {"dim": 64, "num_heads": 4, "kv_heads": 3},
                  {"dim": 64, "num_heads": 4, "layout": "other"}, {"dim": 64, "num_heads": 4, "shortest": 1.0},
                  {"dim": 64, "num_heads": 4, "frequencies": rotary_frequencies(32)}, {"dim": 4, "num_heads": 4}):
        with pytest.raises(ValueError):
            CausalMixer(**wrong)


CAUSAL_KERNELS = ("11walk_kernel", "12carry_kernel", "21attention_step_kernel", "13rotary_kernel", "16team_norm_kernel",
                  "22norm_statistics_kernel", "17norm_apply_kernel", "16norm_grad_kernel", "15head_sum_kernel")


def test_causal_kernels_do_not_spill() -> None:
    path = build.library_path()
    if not path.is_file():
        import __graft_entry__

        __graft_entry__.build()
    found = {}
    for image in _code_objects(path.read_bytes()):
        for kernel in _kernels(image):
            if any(part in kernel[".name"] for part in CAUSAL_KERNELS):
                found[kernel[".name"]] = (kernel[".vgpr_spill_count"], kernel[".private_segment_fixed_size"])
    assert all(any(part in name for name in found) for part in CAUSAL_KERNELS)
    assert {name: count for name, count in found.items() if any(count)} == {}


def _relative(actual, expected):
    actual, expected = actual.detach().double().cpu(), expected.detach().double().cpu()
    return float((actual - expected).norm() / expected.norm())


# A chain of five operators, each of which rounds its output (and the projections
# their inputs to BF16) once: at most 12 roundings of 2^-8 or 2^-11 and 2^-8 on the
# way, added up as independent ones, and twice that on the way back.
FORWARD, BACKWARD = 12**0.5 * 2.0**-8, 2 * 12**0.5 * 2.0**-8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("layout", ("interleaved", "half"))
def test_trains_as_the_reference(native, dtype, layout) -> None:
    mixer = _mixer(layout=layout).cuda()
    x = torch.randn(3, 200, 64, device="cuda").to(dtype).requires_grad_()
    kept = torch.arange(200, device="cuda")[None, :] < torch.tensor([200, 77, 0], device="cuda")[:, None]
    dy = torch.randn(3, 200, 64, device="cuda").to(dtype)
    leaves = [x, *mixer.parameters()]
    y = mixer(x, kept, implementation="hip")
    assert y.dtype == dtype and not y[~kept].any()
    grads = torch.autograd.grad(y, leaves, dy)
    exact = copy.deepcopy(mixer).double()
    ends = [x.detach().double().requires_grad_(), *exact.parameters()]
    expected = exact(ends[0], kept)
    assert _relative(y, expected) <= FORWARD
    for a, e in zip(grads, torch.autograd.grad(expected, ends, dy.double())):
        assert _relative(a, e) <= BACKWARD
    assert not grads[0][~kept].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_prompt_and_steps(native, dtype) -> None:
    """A batch of padded prompts, then single tokens, one sequence ending early."""

    mixer = _mixer().cuda()
    exact = copy.deepcopy(mixer).double()
    lengths = torch.tensor([40, 9, 64], device="cuda")
    kept = torch.arange(64, device="cuda")[None, :] < lengths[:, None]
    x = torch.randn(3, 64, 64, device="cuda").to(dtype)
    with torch.no_grad():
        y, state = mixer(x, kept, return_state=True, implementation="hip")
        expected, exact_state = exact(x.double(), kept, return_state=True)
        assert _relative(y, expected) <= FORWARD and _relative(state, exact_state) <= FORWARD
        for t in range(6):
            token = torch.randn(3, 64, device="cuda").to(dtype)
            alive = torch.tensor([True, t < 3, True], device="cuda")
            before = state.clone()
            y = mixer.step(token, state, lengths + t, alive, implementation="hip")
            expected = exact.step(token.double(), exact_state, lengths + t, alive)
            assert _relative(y, expected) <= FORWARD and _relative(state, exact_state) <= FORWARD
            if t >= 3:
                assert not y[1].any() and torch.equal(state[1], before[1])


@pytest.mark.gpu
def test_captured_serving(native) -> None:
    """The step of a serving loop as one graph, its state and positions moving on."""

    mixer = _mixer().cuda()
    state, other = mixer.initial_state(2), mixer.initial_state(2)
    token = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)
    position = torch.zeros(2, dtype=torch.int64, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        mixer.step(token, state, position, implementation="hip")
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mixer.step(token, state, position, implementation="hip")
        position += 1
    state.zero_()
    position.zero_()
    for t in range(5):
        token.copy_(torch.randn(2, 64))
        graph.replay()
        expected = mixer.step(token, other, torch.full((2,), t, device="cuda"), implementation="hip")
        assert torch.equal(y, expected) and torch.equal(state, other)


@pytest.mark.gpu
def test_captured_training_of_a_stack(native) -> None:
    """Embedding, LSSO, causal mixer and feed-forward block: one training step."""

    torch.manual_seed(0)
    embed = TokenEmbedding(50, 64).cuda()
    context = LSSO(LSSOConfig(dim=64, num_heads=2, rank=16)).cuda()
    mixer, feed = _mixer().cuda(), GatedFeedForward(64, 160).cuda()
    leaves = [p for m in (embed, context, mixer, feed) for p in m.parameters()]
    tokens = torch.randint(0, 50, (2, 80), device="cuda")
    dy = torch.randn(2, 80, 64, device="cuda").bfloat16()

    def step():
        x = embed(tokens, dtype=torch.bfloat16, implementation="hip")
        x = x + context(x, implementation="hip")
        x = x + mixer(x, implementation="hip")
        y = x + feed(x, implementation="hip")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        torch.manual_seed(seed)
        tokens.copy_(torch.randint(0, 50, (2, 80)))
        graph.replay()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_optimizer_step_moves_every_parameter(native) -> None:
    mixer = _mixer().cuda()
    before = [p.detach().clone() for p in mixer.parameters()]
    optimizer = torch.optim.SGD(mixer.parameters(), lr=0.1)
    x = torch.randn(2, 33, 64, device="cuda").bfloat16()
    mixer(x, implementation="hip").float().square().mean().backward()
    optimizer.step()
    for a, b in zip(mixer.parameters(), before):
        assert torch.isfinite(a).all() and not torch.equal(a, b)
