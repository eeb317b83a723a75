"""The operators around the mixer as a program uses them: tokens -> embedding ->
blocks of (mixer, residual dropout, feed-forward, residual dropout), trained,
decoded and captured."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn
from torch.autograd import forward_ad

from lsso_amd.ball import LSSO, GatedFeedForward, LSSOConfig, ResidualDropout, TokenEmbedding, hip

VOCABULARY, DIM, HIDDEN, PROBABILITY = 37, 64, 136, 0.1


class Stack(nn.Module):
    def __init__(self, layers: int, dim: int = DIM, hidden: int = HIDDEN, heads: int = 2, rank: int = 16) -> None:
        super().__init__()
        # A table of variance 1 / dim times sqrt(dim): a stream of variance 1.
        self.embed = TokenEmbedding(VOCABULARY, dim, scale=dim**0.5, padding_index=0)
        self.mixers = nn.ModuleList(LSSO(LSSOConfig(dim=dim, num_heads=heads, rank=rank)) for _ in range(layers))
        self.blocks = nn.ModuleList(GatedFeedForward(dim, hidden) for _ in range(layers))
        self.join = ResidualDropout(PROBABILITY)

    def forward(self, tokens, mask, seed, *, dtype, implementation, keep=None):
        x = self.embed(tokens, mask, dtype=dtype, implementation=implementation)
        for layer, (mixer, block) in enumerate(zip(self.mixers, self.blocks)):
            for part, step in enumerate((mixer, block)):
                y = step(x, mask, implementation=implementation)
                if keep is not None:
                    keep.append((x, y))
                x = self.join(y, x, seed=seed, offset=2 * layer + part, implementation=implementation)
        return x


def _stack(layers, device, **sizes):
    torch.manual_seed(5)
    stack = Stack(layers, **sizes)
    with torch.no_grad():
        for mixer in stack.mixers:   # zero as constructed
            mixer.core_base_raw.normal_(0, 0.2)
            mixer.core_drive_weight.normal_(0, 0.2)
    return stack.to(device)


def _batch(device, batch=3, length=70):
    generator = torch.Generator().manual_seed(11)
    tokens = torch.randint(0, VOCABULARY, (batch, length), generator=generator)
    mask = torch.ones(batch, length, dtype=torch.bool)
    mask[1, length // 2:] = False
    mask[2, :] = False   # a sequence of padding alone
    tokens[~mask] = 10**6
    dy = torch.randn(batch, length, DIM, generator=generator)
    return tokens.to(device), mask.to(device), dy.to(device)


def test_reference_run_against_differences() -> None:
    stack = _stack(1, "cpu", dim=8, hidden=8, heads=1, rank=4).double()
    tokens = torch.tensor([[1, 2, 0, 1, 5]])
    mask = torch.tensor([[True, True, True, True, False]])
    names, values = zip(*((name, value.detach()) for name, value in stack.named_parameters()))

    def run(*parameters):
        return torch.func.functional_call(
            stack, dict(zip(names, parameters)), (tokens, mask, 3), {"dtype": torch.float64, "implementation": "reference"}
        )

    # The padding row feeds the output and has no gradient: differences of the
    # table are taken of its other rows.
    table = values[names.index("embed.weight")]
    free = table[1:].clone().requires_grad_()
    others = [value.clone().requires_grad_() for name, value in zip(names, values) if name != "embed.weight"]

    def whole(rows, *rest):
        at = names.index("embed.weight")
        return run(*rest[:at], torch.cat((table[:1], rows)), *rest[at:])

    assert torch.autograd.gradcheck(whole, (free, *others), eps=1e-6, atol=1e-6, rtol=1e-5, fast_mode=True)


def test_forward_mode_derivatives_are_refused(monkeypatch) -> None:
    """With and without a reverse-mode graph; the check comes before the device's."""

    monkeypatch.setattr(hip, "require_available", lambda: None)
    x, weight = torch.randn(3, 4), torch.randn(4, 4)
    tokens = torch.tensor([0, 1])
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(weight, torch.ones(4, 4))
        rows = forward_ad.make_dual(x, torch.ones(3, 4))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: hip.embedding(tokens, dual), lambda: hip.dropout_add(rows, None, 0.1, 1),
                             lambda: hip.dropout_add(x, rows, 0.1, 1),
                             lambda: hip.gated_feed_forward(rows, weight, weight, weight),
                             lambda: hip.gated_feed_forward(x, weight, dual, weight),
                             lambda: hip.gated_feed_forward(x, weight, weight, dual)):
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call()
        with pytest.raises(RuntimeError, match="CUDA"):   # without a tangent
            hip.dropout_add(x, None, 0.1, 1)


def test_the_mixer_refuses_forward_mode_derivatives(monkeypatch) -> None:
    monkeypatch.setattr(hip, "require_available", lambda: None)
    x, weight, mixed = torch.randn(1, 4, 8), torch.randn(8, 8), torch.zeros(1, 4, 24)
    base, drive, eta = torch.zeros(1, 16, 16), torch.zeros(1, 8, 16), torch.zeros(1)
    core = (base, drive, eta)
    with torch.no_grad(), forward_ad.dual_level():
        rows = forward_ad.make_dual(x, torch.ones_like(x))
        dual = forward_ad.make_dual(eta, torch.ones_like(eta))
        for call in (lambda: hip.linear(rows, weight, None, torch.bfloat16),
                     lambda: hip.linear(x, weight, dual, torch.bfloat16),
                     lambda: hip.fast_mix(mixed, base, drive, dual),
                     lambda: hip.forward_inference(mixed, base, drive, dual),
                     lambda: hip.forward_train(mixed, base, drive, dual),
                     lambda: hip.project_mix(rows, weight, None, *core),
                     lambda: hip.mix_project(mixed, base, drive, dual, None, None, weight, None, torch.bfloat16),
                     lambda: hip.layer_forward(rows, weight, None, *core, None, None, weight, None),
                     lambda: hip.layer_train(rows, weight, None, *core, weight, None)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


@pytest.mark.gpu
def test_a_layer_refuses_forward_mode_derivatives(native) -> None:
    layer = LSSO(LSSOConfig(dim=64, num_heads=2, rank=16)).cuda()
    for dim, length in ((64, 33), (64, 1)):
        x = torch.randn(1, length, dim, device="cuda").bfloat16()
        expected = layer(x, implementation="hip")
        with forward_ad.dual_level():
            assert torch.equal(layer(x, implementation="hip"), expected)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                layer(forward_ad.make_dual(x, torch.ones_like(x)), implementation="hip")


@pytest.mark.gpu
def test_forward_mode_leaves_plain_calls_alone(native) -> None:
    x = torch.randn(5, 8, device="cuda")
    weights = [torch.randn(8, 8, device="cuda") for _ in range(3)]
    calls = (lambda: native.embedding(torch.tensor([0, 4, 2], device="cuda"), x),
             lambda: native.dropout_add(x, x, 0.3, 5),
             lambda: native.gated_feed_forward(x.bfloat16(), *weights))
    expected = [call() for call in calls]
    with forward_ad.dual_level():
        forward_ad.make_dual(torch.randn(2, device="cuda"), torch.ones(2, device="cuda"))
        for call, value in zip(calls, expected):
            assert torch.equal(call(), value)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            native.dropout_add(forward_ad.make_dual(x, torch.ones_like(x)), None, 0.1, 1)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: native.dropout_add(v, None, 0.1, 1), (x,), (torch.ones_like(x),))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("masked", (True, False))
def test_training_run_against_the_formulas(native, dtype, masked) -> None:
    """Against the reference path in FP64.

    Every rounding moves the stream, or its gradient, by at most half a step of
    bfloat16 (the mixer computes in it for both types), 2^-8, of what is
    rounded, and the branches' gains are below 1.  A path from a token to a
    gradient meets, per block and direction, up to 8 of them in the mixer
    (projection, weights, content, output and their gradients), 2 in the sums
    and 6 in the feed-forward block (weights, h, factors, dg, du, y): 16 x 2
    blocks x 2 directions x 2^-8 = 0.25 of each output's norm if all of them
    agreed."""

    stack = _stack(2, "cuda")
    tokens, mask, dy = _batch("cuda")
    if not masked:
        tokens, mask = tokens.clamp(max=VOCABULARY - 1), None
    dy = dy.to(dtype)
    y = stack(tokens, mask, 17, dtype=dtype, implementation="hip")
    parameters = dict(stack.named_parameters())
    grads = torch.autograd.grad(y, list(parameters.values()), dy)
    exact = _stack(2, "cuda").double()
    z = exact(tokens, mask, 17, dtype=torch.float64, implementation="reference")
    expected = torch.autograd.grad(z, list(exact.parameters()), dy.double())
    for name, a, b in zip(("y", *parameters), (y, *grads), (z, *expected)):
        assert torch.isfinite(a).all(), name
        assert (a.double() - b).norm() <= 0.25 * b.norm(), name
    if masked:
        assert not y[~mask].any()
    assert not grads[0][0].any()   # the padding row


@pytest.mark.gpu
def test_run_is_its_steps(native) -> None:
    """One backward through the run equals the operators' own gradients, step by
    step, bit for bit."""

    stack = _stack(2, "cuda")
    tokens, mask, dy = _batch("cuda")
    dy = dy.bfloat16()
    steps = []
    y = stack(tokens, mask, 17, dtype=torch.bfloat16, implementation="hip", keep=steps)
    grads = dict(zip(dict(stack.named_parameters()), torch.autograd.grad(y, list(stack.parameters()), dy)))
    flow = dy
    for layer in reversed(range(2)):
        for part, (name, module) in reversed(list(enumerate((("mixers", stack.mixers), ("blocks", stack.blocks))))):
            x, _ = steps[2 * layer + part]
            x = x.detach().requires_grad_()
            out = module[layer](x, mask, implementation="hip")
            branch = native.dropout_add(flow, None, PROBABILITY, 17, 2 * layer + part)
            parameters = dict(module[layer].named_parameters())
            d, *found = torch.autograd.grad(out, [x, *parameters.values()], branch)
            for key, value in zip(parameters, found):
                assert torch.equal(value, grads[f"{name}.{layer}.{key}"]), (name, layer, key)
            flow = flow + d
    table = stack.embed.weight.detach().requires_grad_()
    x = native.embedding(tokens, table, scale=stack.embed.scale, row_mask=mask, padding_index=0,
                         output_dtype=torch.bfloat16)
    assert torch.equal(torch.autograd.grad(x, table, flow)[0], grads["embed.weight"])


@pytest.mark.gpu
def test_captured_training_run(native) -> None:
    stack = _stack(2, "cuda")
    tokens, mask, dy = _batch("cuda")
    dy = dy.bfloat16()
    state = torch.tensor([17, 0], dtype=torch.int64, device="cuda")
    parameters = list(stack.parameters())

    def step():
        y = stack(tokens, mask, state, dtype=torch.bfloat16, implementation="hip")
        return (y.detach(), *torch.autograd.grad(y, parameters, dy))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    before = None
    for replay in range(3):
        tokens.copy_(torch.randint(0, VOCABULARY, tokens.shape, device="cuda"))
        mask[0, 60 - replay:] = False
        state[1] += 4   # four joins a step
        graph.replay()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)
        assert before is None or not torch.equal(before, captured[0])
        before = captured[0].clone()


@pytest.mark.gpu
@pytest.mark.parametrize("length", (1, 31, 33))
def test_evaluation_of_one_sequence(native, length) -> None:
    """A request: a single sequence, down to one token, without dropout; the
    bound of the training run, one direction."""

    stack = _stack(2, "cuda").eval()
    tokens = torch.randint(1, VOCABULARY, (1, length), device="cuda")
    with torch.no_grad():
        y = stack(tokens, None, 0, dtype=torch.bfloat16, implementation="hip")
        z = _stack(2, "cuda").double().eval()(tokens, None, 0, dtype=torch.float64, implementation="reference")
    assert (y.double() - z).norm() <= 0.125 * z.norm()
