"""Linear attention with a decay for each head: the definition token by token in
FP64 against the reference path on the CPU and the native kernels on the device:
values, states, gradients, masks, layouts, decays, segments, single tokens,
captured replays and refusals."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from lsso_amd.ball import causal, hip
from lsso_amd.ball import reference as canonical

HALVES = (torch.float16, torch.bfloat16)


def _recurrence(q, k, v, log_decay, scale, mask=None, state=None):
    """The definition, one token after another, in FP64."""

    batch, length, heads, features = q.shape
    shared = heads // k.shape[2]
    q, k, v = (x.double() for x in (q, k, v))
    k, v = (x.repeat_interleave(shared, dim=2) for x in (k, v))
    decay = log_decay.double().exp()[:, None, None]
    s = torch.zeros(batch, heads, features, v.shape[-1], dtype=torch.float64, device=q.device)
    s = s if state is None else state.double()
    outputs = []
    for t in range(length):
        kept = torch.ones(batch, dtype=torch.bool, device=q.device) if mask is None else mask[:, t]
        new = decay * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        s = torch.where(kept[:, None, None, None], new, s)
        y = scale * (q[:, t, :, None, :] @ s)[..., 0, :]
        outputs.append(torch.where(kept[:, None, None], y, torch.zeros_like(y)))
    y = torch.stack(outputs, dim=1) if outputs else q.new_zeros(batch, 0, heads, v.shape[-1])
    return y, s


def _decays(heads):
    return torch.log1p(-(2.0 ** -torch.linspace(2.0, 8.0, heads))).float()


def _mask(kind, batch, length, generator):
    if kind is None:
        return None
    if kind == "suffix":   # the last sample of several is empty
        counts = torch.randint(0, length + 1, (batch,), generator=generator)
        counts[0] = length
        if batch > 1:
            counts[-1] = 0
        return torch.arange(length)[None, :] < counts[:, None]
    if kind == "prefix":   # left padding
        counts = torch.randint(0, length + 1, (batch,), generator=generator)
        return torch.arange(length)[None, :] >= counts[:, None]
    return torch.rand(batch, length, generator=generator) < 0.6


def _inputs(batch, length, heads, kv_heads, features, out, dtype, seed=0):
    generator = torch.Generator().manual_seed(seed)
    q = torch.randn(batch, length, heads, features, generator=generator).to(dtype)
    k = torch.randn(batch, length, kv_heads, features, generator=generator).to(dtype)
    v = torch.randn(batch, length, kv_heads, out, generator=generator).to(dtype)
    return q, k, v, _decays(heads), generator


# ------------------------------------------------------------------- reference
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 1), (2, 5, 2, 1, 3, 4), (2, 64, 4, 2, 8, 8), (3, 131, 2, 2, 6, 5),
                                   (2, 0, 2, 1, 3, 4)])
@pytest.mark.parametrize("kind", (None, "suffix", "prefix", "holes"))
def test_reference_is_the_definition(shape, kind) -> None:
    q, k, v, log_decay, generator = _inputs(*shape, torch.float64)
    mask = _mask(kind, shape[0], shape[1], generator)
    state = torch.randn(shape[0], shape[2], shape[4], shape[5], generator=generator, dtype=torch.float64)
    y, last = canonical.linear_attention(q, k, v, log_decay, row_mask=mask, initial_state=state, return_state=True)
    expected, expected_last = _recurrence(q, k, v, log_decay, shape[4] ** -0.5, mask, state)
    # Sums of up to 131 terms in another order, in FP64.
    torch.testing.assert_close(y, expected, rtol=1e-11, atol=1e-11)
    torch.testing.assert_close(last, expected_last, rtol=1e-11, atol=1e-11)


def test_reference_gradients_match_differences() -> None:
    q, k, v, log_decay, generator = _inputs(2, 5, 2, 1, 3, 2, torch.float64)
    mask = torch.tensor([[True, False, True, True, False], [False] * 5])
    state = torch.randn(2, 2, 3, 2, generator=generator, dtype=torch.float64)
    leaves = [x.requires_grad_() for x in (q, k, v, state)]
    assert torch.autograd.gradcheck(
        lambda q, k, v, s: canonical.linear_attention(
            q, k, v, log_decay, row_mask=mask, initial_state=s, return_state=True), leaves)


def test_reference_steps_go_on_from_a_prompt() -> None:
    q, k, v, log_decay, _ = _inputs(2, 9, 4, 2, 6, 5, torch.float64)
    whole, last = canonical.linear_attention(q, k, v, log_decay, return_state=True)
    y, state = canonical.linear_attention(q[:, :6], k[:, :6], v[:, :6], log_decay, return_state=True)
    for t in range(6, 9):
        step = canonical.linear_attention_step(q[:, t], k[:, t], v[:, t], log_decay, state)
        torch.testing.assert_close(step, whole[:, t], rtol=1e-11, atol=1e-11)
    torch.testing.assert_close(state, last, rtol=1e-11, atol=1e-11)


def test_forgets_at_once() -> None:
    q, k, v, _, _ = _inputs(1, 70, 1, 1, 4, 4, torch.float64)
    y = canonical.linear_attention(q, k, v, torch.tensor([-math.inf]), scale=1.0)
    torch.testing.assert_close(y, (q * k).sum(-1, keepdim=True) * v)


# ------------------------------------------------------------------ C refusals
def _shape(**changes):
    fields = {"batch": 2, "length": 3, "heads": 4, "kv_heads": 2, "features": 8, "value_features": 8, "dtype": 2,
              "scale": 1.0}
    fields.update(changes)
    strides = [causal.HeadStrides(96, 32, 8) for _ in range(3)]
    if fields.pop("stride", 0):
        strides[1] = causal.HeadStrides(96, -32, 8)
    return causal.LinearAttentionShape(*fields.values(), *strides)


def test_refusals_on_the_cpu() -> None:
    library = hip.open_library()
    kept, forward_size, backward_size = (ctypes.c_size_t() for _ in range(3))
    pointers = [ctypes.byref(size) for size in (kept, forward_size, backward_size)]

    def sizes(out=pointers[0], **changes):
        return library.lsso_hip_linear_attention_sizes(ctypes.byref(_shape(**changes)), out, *pointers[1:])

    def forward(q=16, k=16, v=16, log_decay=16, state=None, y=16, last=None, workspace=None, count=0, **changes):
        return library.lsso_hip_linear_attention(
            ctypes.byref(_shape(**changes)), q, k, v, log_decay, None, state, None, y, last, workspace, count, None)

    def backward(grad=16, strides=causal.HeadStrides(96, 32, 8), last=None, q=16, log_decay=16, grad_q=16, grad_s=None,
                 workspace=None, count=0, **changes):
        return library.lsso_hip_linear_attention_backward(
            ctypes.byref(_shape(**changes)), grad, None if strides is None else ctypes.byref(strides), last, q, 16, 16,
            log_decay, None, None, None, grad_q, None, None, grad_s, workspace, count, None)

    def step(q=16, state=16, stride=256, y=16, log_decay=16, **changes):
        return library.lsso_hip_linear_attention_step(
            ctypes.byref(_shape(**{"length": 1, **changes})), q, 16, 16, log_decay, None, state, stride, y, None)

    # Shared heads: FP32 gradients of each, and past two chunks the segments' states.
    assert sizes() == 0 and kept.value == 0 and forward_size.value == 0 and backward_size.value == 2 * 3 * 4 * 8 * 4
    assert sizes(length=1000, kv_heads=4) == 0 and kept.value >= 2 * 2 * 4 * 64
    assert forward_size.value >= 4 * kept.value and backward_size.value >= 4 * kept.value
    for wrong in ({"batch": -1}, {"length": -1}, {"heads": 0}, {"kv_heads": 3}, {"features": 0}, {"features": 129},
                  {"value_features": 129}, {"dtype": 3}, {"scale": math.inf}, {"scale": math.nan}, {"stride": 1},
                  {"batch": 2**22}, {"batch": 2**23, "heads": 1, "kv_heads": 1}, {"heads": 8192, "kv_heads": 1}, {"length": 2**31}):
        assert sizes(**wrong) < 0, wrong
        assert forward(**wrong) < 0 and step(**{**wrong, "length": wrong.get("length", 1)}) < 0, wrong
        assert library.lsso_hip_last_error()
    assert sizes(out=None) < 0
    assert library.lsso_hip_linear_attention_sizes(None, *pointers) < 0
    assert forward(batch=0) == 0 and forward(length=0) == 0 and backward(batch=0) == 0 and step(batch=0) == 0
    for wrong in ({"q": None}, {"k": 17}, {"v": None}, {"y": None}, {"log_decay": None}, {"log_decay": 18},
                  {"state": 18}, {"last": 18}, {"length": 1000}, {"length": 1000, "workspace": 255, "count": 1 << 30},
                  {"length": 1000, "workspace": 256, "count": 64}):
        assert forward(**wrong) < 0, wrong
    for wrong in ({"grad": None}, {"strides": None}, {"strides": causal.HeadStrides(1, -1, 1)}, {"q": None},
                  {"log_decay": None}, {"last": 18}, {"grad_q": 17}, {"grad_s": 18}, {}):   # {}: no workspace
        assert backward(**wrong) < 0, wrong
    for wrong in ({"q": None}, {"state": None}, {"state": 18}, {"stride": 255}, {"y": 17}, {"length": 2},
                  {"log_decay": None}):
        assert step(**wrong) < 0, wrong


# ---------------------------------------------------------------------- device
def _bound(expected, magnitude, dtype, small):
    """One rounding to the type, and what FP32 sums of terms of this magnitude are off:
    scores and states over up to 128 terms (2^-17), two 16-bit parts (2^-18), carried
    states and exponentials (2^-18).  FP16 parts below its normal range are off by half
    of 2^-24 each, of 64 tokens at a time: `small`."""

    half = torch.finfo(dtype).eps / 2
    tiny = 2.0**-24 if dtype == torch.float16 else 0.0
    return half * (1 + 2.0**-10) * expected.abs() + 2.0**-15 * magnitude + tiny * (1 + 64 * small) + 1e-30


def _check(q, k, v, log_decay, mask, state, grads, device="cuda", view=lambda x: x.cuda()):
    """Native values and gradients of one call against the recurrence in FP64."""

    dtype, scale = q.dtype, q.shape[-1] ** -0.5
    leaves = [view(x).detach().requires_grad_() for x in (q, k, v)]
    first = None if state is None else state.to(device).requires_grad_()
    result = hip.linear_attention(*leaves, log_decay.to(device), row_mask=None if mask is None else mask.to(device),
                                  initial_state=first, return_state=state is not None)
    outputs = result if state is not None else (result,)
    inputs = leaves + ([] if state is None else [first])
    dy, ds = grads
    given = [dy.to(device)] + ([] if state is None else [ds.to(device)])
    found = torch.autograd.grad(outputs, inputs, given)

    def oracle(f):
        ends = [f(x.double()).requires_grad_() for x in (q, k, v)] + ([] if state is None else [f(state.double()).requires_grad_()])
        y, last = _recurrence(*ends[:3], log_decay, scale, mask, None if state is None else ends[3])
        if state is None:
            return [y], torch.autograd.grad([y], ends, [f(dy.double())])
        return [y, last], torch.autograd.grad([y, last], ends, [f(dy.double()), f(ds.double())])

    values, gradients = oracle(lambda x: x.clone())
    sizes, gradient_sizes = oracle(lambda x: x.abs())
    # FP16 factors here are normal: q, k, v, dy of size one, so products reach scale * D.
    small = 8.0 + scale * q.shape[-1]
    for name, a, e, m in zip(("y", "state"), outputs, values, sizes):
        assert a.dtype == (dtype if name == "y" else torch.float32) and a.is_contiguous()
        off = (a.detach().cpu().double() - e.detach()).abs()
        assert (off <= _bound(e.detach(), m.detach(), a.dtype, small if name == "y" else 0)
                + (2.0**-24 * 64 * 8 if dtype == torch.float16 and name == "state" else 0)).all(), name
    for name, a, e, m in zip(("dq", "dk", "dv", "ds"), found, gradients, gradient_sizes):
        off = (a.cpu().double() - e).abs()
        assert (off <= _bound(e, m, a.dtype, small)
                + (2.0**-24 * 64 * 8 if dtype == torch.float16 and name == "ds" else 0)).all(), (name, off.max())


def _case(batch, length, heads, kv_heads, features, out, dtype, kind, with_state, seed=0, view=lambda x: x.cuda()):
    q, k, v, log_decay, generator = _inputs(batch, length, heads, kv_heads, features, out, dtype, seed)
    mask = _mask(kind, batch, length, generator)
    state = torch.randn(batch, heads, features, out, generator=generator) if with_state else None
    dy = torch.randn(batch, length, heads, out, generator=generator).to(dtype)
    ds = torch.randn(batch, heads, features, out, generator=generator)
    _check(q, k, v, log_decay, mask, state, (dy, ds), view=view)


SIZES = [(1, 1, 1, 1, 1, 1), (2, 3, 2, 1, 5, 7), (1, 15, 2, 2, 16, 32), (2, 64, 4, 2, 64, 64), (1, 65, 3, 1, 33, 40),
         (2, 130, 2, 2, 128, 96), (1, 257, 6, 2, 80, 24), (3, 66, 2, 1, 100, 128), (1, 128, 2, 2, 8, 72),
         (2, 63, 1, 1, 3, 128), (1, 127, 2, 1, 128, 6), (2, 17, 4, 4, 40, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("kind,with_state", [(None, False), (None, True), ("suffix", True), ("holes", False)])
def test_values_and_gradients(native, dtype, size, kind, with_state) -> None:
    _case(*size, dtype, kind, with_state)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kind", (None, "suffix", "prefix", "holes"))
def test_segments(native, dtype, kind) -> None:
    """Few heads: 11 chunks are walked in three segments, each from its own state."""

    _case(2, 700, 2, 1, 32, 48, dtype, kind, True, seed=3)
    _case(1, 1030, 1, 1, 17, 9, dtype, kind, True, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
def test_padding_longer_than_a_segment(native, dtype) -> None:
    """A state, and the gradient of one, that pass whole segments without a token."""

    q, k, v, log_decay, generator = _inputs(2, 1200, 1, 1, 16, 16, dtype)
    mask = torch.zeros(2, 1200, dtype=torch.bool)
    mask[0, 700:710] = True
    state, ds = (torch.randn(2, 1, 16, 16, generator=generator) for _ in range(2))
    dy = torch.randn(2, 1200, 1, 16, generator=generator).to(dtype)
    _check(q, k, v, log_decay, mask, state, (dy, ds))


@pytest.mark.gpu
def test_what_the_mask_excludes_reaches_nothing(native) -> None:
    for dtype in HALVES:
        q, k, v, log_decay, generator = _inputs(2, 100, 2, 1, 24, 24, dtype)
        mask = _mask("holes", 2, 100, generator)
        wild = [torch.where(mask[..., None, None], x, bad) for x, bad in zip((q, k, v), (math.nan, math.inf, -math.inf))]
        dy = torch.randn(2, 100, 2, 24, generator=generator).to(dtype)
        wild_dy = torch.where(mask[..., None, None], dy, math.nan)
        results = []
        for inputs, grad in (((q, k, v), dy), (wild, wild_dy)):
            leaves = [x.cuda().requires_grad_() for x in inputs]
            y, last = native.linear_attention(*leaves, log_decay.cuda(), row_mask=mask.cuda(), return_state=True)
            results.append([y, last, *torch.autograd.grad(y, leaves, grad.cuda())])
        for a, b in zip(*results):
            assert torch.equal(a, b)
        assert not results[0][0][~mask.cuda()].any() and not results[0][2][~mask.cuda()].any()


@pytest.mark.gpu
def test_layouts(native) -> None:
    """Slices of a packed projection, heads before tokens, odd bases and strides, and
    broadcast inputs whose gradient is summed."""

    for dtype in HALVES:
        q, k, v, log_decay, generator = _inputs(2, 70, 4, 4, 24, 24, dtype)
        log_decay = log_decay.cuda()
        plain = native.linear_attention(q.cuda(), k.cuda(), v.cuda(), log_decay)
        packed = torch.cat((q, k, v), dim=2).cuda()
        assert torch.equal(native.linear_attention(*packed.split(4, dim=2), log_decay), plain)
        assert torch.equal(native.linear_attention(*(x.transpose(1, 2).cuda().contiguous().transpose(1, 2)
                                                     for x in (q, k, v)), log_decay), plain)
        room = [torch.zeros(x.numel() * 2 + 1, dtype=dtype, device="cuda") for x in (q, k, v)]
        odd = []
        for r, x in zip(room, (q, k, v)):   # one element past an aligned base, 25 elements from head to head
            to = r[1:1 + 2 * 70 * 4 * 25].view(2, 70, 4, 25)[..., :24]
            to.copy_(x)
            odd.append(to)
        assert torch.equal(native.linear_attention(*odd, log_decay), plain)
        columns = [x.cuda().mT.contiguous().mT for x in (q, k, v)]   # no unit feature stride
        assert torch.equal(native.linear_attention(*columns, log_decay), plain)
        one = k[:1].cuda().requires_grad_()
        y = native.linear_attention(q.cuda(), one.expand(2, -1, -1, -1), v.cuda(), log_decay)
        whole = k[:1].expand(2, -1, -1, -1).contiguous().cuda().requires_grad_()
        z = native.linear_attention(q.cuda(), whole, v.cuda(), log_decay)
        assert torch.equal(y, z)
        dy = torch.randn(y.shape, generator=generator).to(dtype).cuda()
        (a,), (b,) = torch.autograd.grad(y, one, dy), torch.autograd.grad(z, whole, dy)
        assert torch.equal(a, b.sum(0, keepdim=True))
        # The gradient of a sum is one value, broadcast.
        leaf = q.cuda().requires_grad_()
        (a,) = torch.autograd.grad(native.linear_attention(leaf, k.cuda(), v.cuda(), log_decay).sum(), leaf)
        (b,) = torch.autograd.grad(native.linear_attention(leaf, k.cuda(), v.cuda(), log_decay), leaf, torch.ones_like(y))
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rate", (0.0, -1e-4, -3.0, -200.0, -math.inf))
def test_decays(native, dtype, rate) -> None:
    q, k, v, _, generator = _inputs(1, 300, 1, 1, 16, 16, dtype)
    state, ds = (torch.randn(1, 1, 16, 16, generator=generator) for _ in range(2))
    dy = torch.randn(1, 300, 1, 16, generator=generator).to(dtype)
    _check(q, k, v, torch.tensor([rate]), None, state, (dy, ds))


@pytest.mark.gpu
def test_states_past_half_precision(native) -> None:
    """A state of 70,000 in float16, read by a query that brings it back."""

    length = 70 * 64
    q = torch.full((1, length, 1, 16), 2.0**-8, dtype=torch.float16, device="cuda")
    k = torch.ones_like(q)
    v = torch.full_like(q, 16.0)
    y, last = native.linear_attention(q, k, v, torch.zeros(1, device="cuda"), scale=1.0, return_state=True)
    assert torch.equal(last, torch.full_like(last, 16.0 * length))
    # 16 (t + 1) summed over 16 features of 2^-8: t + 1, exact up to 2,048 and rounded past it.
    expected = torch.arange(1.0, length + 1, device="cuda").half().view(1, -1, 1, 1).expand_as(y)
    assert torch.equal(y, expected)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
def test_an_infinite_product_is_infinite(native, dtype) -> None:
    big = 60000.0 if dtype == torch.float16 else 3e38
    q = torch.full((1, 1, 1, 8), 1.0, dtype=dtype, device="cuda")
    k = torch.full_like(q, big)
    y = native.linear_attention(q, k, torch.full_like(q, 2.0), torch.zeros(1, device="cuda"), scale=1.0)
    assert torch.isposinf(y).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1), (3, 4, 2, 64, 64), (2, 6, 2, 33, 40), (5, 2, 1, 128, 128), (2, 3, 3, 7, 5),
                                  (2, 2, 2, 128, 30)])
@pytest.mark.parametrize("masked", (False, True))
def test_step(native, dtype, size, masked) -> None:
    batch, heads, kv_heads, features, out = size
    q, k, v, log_decay, generator = _inputs(batch, 1, heads, kv_heads, features, out, dtype)
    state = torch.randn(batch, heads, features, out, generator=generator)
    mask = torch.arange(batch) % 2 == 0 if masked else None
    expected, last = _recurrence(q, k, v, log_decay, features**-0.5, None if mask is None else mask[:, None], state)
    sizes, _ = _recurrence(q.abs(), k.abs(), v.abs(), log_decay, features**-0.5, None, state.abs())
    for room in (0, 1, 4):   # states of a batch that lie apart, 16-byte aligned or not
        pool = torch.zeros(batch, heads * features * out + room, device="cuda")
        slots = pool[:, :heads * features * out].view(batch, heads, features, out)
        slots.copy_(state)
        y = native.linear_attention_step(q[:, 0].cuda(), k[:, 0].cuda(), v[:, 0].cuda(), log_decay.cuda(), slots,
                                         row_mask=None if mask is None else mask.cuda())
        # FP32 sums of up to 128 terms, one rounding.
        bound = torch.finfo(dtype).eps / 2 * expected.abs() * (1 + 2.0**-10) + 2.0**-16 * sizes + 2.0**-25
        assert ((y.cpu().double() - expected[:, 0]).abs() <= bound[:, 0]).all()
        # exp, product and sum: four roundings.
        assert ((slots.cpu().double() - last).abs() <= 2.0**-21 * (state.double().abs() + (last - state).abs() + 1)).all()
        if mask is not None:
            assert torch.equal(slots.cpu()[~mask], state[~mask])
        assert not pool[:, heads * features * out:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
def test_steps_go_on_from_a_prompt(native, dtype) -> None:
    """A padded batch of prompts, then tokens one at a time, as one long sequence."""

    lengths = (37, 5, 64)
    q, k, v, log_decay, _ = _inputs(3, 70, 4, 2, 32, 32, dtype)
    prompt = torch.arange(64)[None, :] < torch.tensor(lengths)[:, None]
    device = [x.cuda() for x in (q, k, v)]
    y, state = native.linear_attention(*(x[:, :64] for x in device), log_decay.cuda(), row_mask=prompt.cuda(),
                                       return_state=True)
    for t in range(64, 70):
        step = native.linear_attention_step(*(x[:, t] for x in device), log_decay.cuda(), state)
        for b, n in enumerate(lengths):
            rows = [*range(n), *range(64, t + 1)]
            chosen = [x[b:b + 1, rows] for x in (q, k, v)]
            expected, _ = _recurrence(*chosen, log_decay, 32**-0.5)
            sizes, _ = _recurrence(*(x.abs() for x in chosen), log_decay, 32**-0.5)
            off = (step[b].cpu().double() - expected[0, -1]).abs()
            assert (off <= _bound(expected[0, -1], sizes[0, -1], dtype, 12.0)).all()


@pytest.mark.gpu
def test_long_sequences(native) -> None:
    """20,000 tokens of one head: 78 segments, against the reference path in FP64."""

    q, k, v, log_decay, generator = _inputs(1, 20000, 1, 1, 64, 64, torch.bfloat16)
    mask = _mask("holes", 1, 20000, generator).cuda()
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    log_decay = torch.tensor([-1.0 / 4096], device="cuda")
    y, last = native.linear_attention(*leaves, log_decay, row_mask=mask, return_state=True)
    dy, ds = torch.randn_like(y), torch.randn_like(last)
    found = [y, last, *torch.autograd.grad((y, last), leaves, (dy, ds))]

    def reference(f):
        ends = [f(x.detach().double()).requires_grad_() for x in leaves]
        ys = canonical.linear_attention(*ends, log_decay.double(), row_mask=mask, return_state=True)
        return [*ys, *torch.autograd.grad(ys, ends, (f(dy.double()), f(ds.double())))]

    for a, e, m in zip(found, reference(lambda x: x), reference(torch.abs)):
        assert ((a.detach().double() - e.detach()).abs() <= _bound(e.detach(), m.detach(), a.dtype, 0.0)).all()


@pytest.mark.gpu
def test_offsets_past_32_bits(native) -> None:
    """66 tokens 2^26 elements apart: the last ones past 2^32 elements."""

    stride, length = 1 << 26, 66
    room = torch.empty(stride * (length - 1) + 3 * 64, dtype=torch.bfloat16, device="cuda")
    views = [room.as_strided((1, length, 2, 32), (stride, stride, 32, 1), 64 * i) for i in range(3)]
    q, k, v, log_decay, _ = _inputs(1, length, 2, 2, 32, 32, torch.bfloat16)
    for to, x in zip(views, (q, k, v)):
        to.copy_(x)
    far = [x.detach().requires_grad_() for x in views]
    near = [x.cuda().requires_grad_() for x in (q, k, v)]
    y, z = (native.linear_attention(*x, log_decay.cuda()) for x in (far, near))
    assert torch.equal(y, z)
    dy = torch.randn_like(y)
    for a, b in zip(torch.autograd.grad(y, far, dy), torch.autograd.grad(z, near, dy)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_empty(native) -> None:
    decay = _decays(2).cuda()
    q = torch.empty(2, 0, 2, 8, dtype=torch.float16, device="cuda", requires_grad=True)
    state = torch.randn(2, 2, 8, 8, device="cuda", requires_grad=True)
    y, last = native.linear_attention(q, q, q, decay, initial_state=state, return_state=True)
    assert y.shape == (2, 0, 2, 8) and torch.equal(last, state)
    ds = torch.randn_like(last)
    assert torch.equal(torch.autograd.grad(last, state, ds)[0], ds)
    none = torch.empty(0, 5, 2, 8, dtype=torch.float16, device="cuda")
    assert native.linear_attention(none, none, none, decay, return_state=True)[1].shape == (0, 2, 8, 8)
    assert native.linear_attention_step(none[:, 0], none[:, 0], none[:, 0], decay,
                                        torch.empty(0, 2, 8, 8, device="cuda")).shape == (0, 2, 8)
    # The gradient of the state alone, and of y alone where the state is returned.
    q, k, v = (torch.randn(1, 70, 2, 8, device="cuda").half().requires_grad_() for _ in range(3))
    y, last = native.linear_attention(q, k, v, decay, return_state=True)
    dq, dk, dv = torch.autograd.grad(last, (q, k, v), torch.ones_like(last), retain_graph=True)
    assert not dq.any() and dk.any() and dv.any()
    first = torch.zeros(1, 2, 8, 8, device="cuda", requires_grad=True)
    y = native.linear_attention(q, k, v, decay, initial_state=first)
    assert torch.autograd.grad(y.float().sum(), first)[0].any()


@pytest.mark.gpu
def test_other_streams_and_repeats(native) -> None:
    q, k, v, log_decay, _ = _inputs(2, 600, 2, 1, 64, 64, torch.bfloat16)
    q, k, v, log_decay = (x.cuda() for x in (q, k, v, log_decay))
    expected = native.linear_attention(q, k, v, log_decay)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        results = [native.linear_attention(q, k, v, log_decay) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(stream)
    for y in results:
        assert torch.equal(y, expected)


@pytest.mark.gpu
def test_captured_replays(native) -> None:
    """Training and serving steps in two graphs, replayed in turn with eager work between."""

    q, k, v, log_decay, _ = _inputs(2, 600, 2, 1, 32, 32, torch.bfloat16)
    log_decay = log_decay.cuda()
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    dy = torch.randn(2, 600, 2, 32, device="cuda").bfloat16()
    state = torch.zeros(2, 2, 32, 32, device="cuda")
    tokens = [torch.randn(2, h, 32, device="cuda").bfloat16() for h in (2, 1, 1)]

    def train():
        y = native.linear_attention(*leaves, log_decay)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    def serve():
        return native.linear_attention_step(*tokens, log_decay, state)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        train()
        serve()
    torch.cuda.current_stream().wait_stream(stream)
    training, serving = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(training):
        trained = train()
    with torch.cuda.graph(serving):
        served = serve()
    state.zero_()
    for seed in range(4):
        torch.manual_seed(seed)
        with torch.no_grad():
            for leaf in leaves:
                leaf.copy_(torch.randn_like(leaf))
        before = state.clone()
        training.replay()
        serving.replay()
        after, got = state.clone(), served.clone()
        torch.cuda.synchronize()
        for a, b in zip(trained, train()):
            assert torch.equal(a, b)
        state.copy_(before)
        assert torch.equal(serve(), got) and torch.equal(state, after)


@pytest.mark.gpu
def test_saved_tensors_are_checked(native) -> None:
    q, k, v, log_decay, _ = _inputs(1, 8, 2, 2, 8, 8, torch.float16)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x[..., :4] if x.dim() == 4 else x):
        y = native.linear_attention(*leaves, log_decay.cuda())
        with pytest.raises(RuntimeError, match="the saved query"):
            y.sum().backward()
    y = native.linear_attention(*leaves, log_decay.cuda())
    with torch.no_grad():
        leaves[1].zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    # A step changes its state in place, and says so.
    state = torch.zeros(1, 2, 8, 8, device="cuda")
    version = state._version
    native.linear_attention_step(*(x.detach()[:, 0] for x in leaves), log_decay.cuda(), state)
    assert state._version > version


@pytest.mark.gpu
def test_refusals(native) -> None:
    q, k, v, log_decay, _ = _inputs(2, 4, 4, 2, 8, 6, torch.float16)
    q, k, v, log_decay = (x.cuda() for x in (q, k, v, log_decay))
    state = torch.zeros(2, 4, 8, 6, device="cuda")
    for arguments, keywords, error in (
        ((q.cpu(), k, v, log_decay), {}, RuntimeError), ((q, k.cpu(), v, log_decay), {}, RuntimeError),
        ((q.float(), k.float(), v.float(), log_decay), {}, TypeError), ((q, k.bfloat16(), v, log_decay), {}, TypeError),
        ((q[0], k[0], v[0], log_decay), {}, ValueError), ((q, k[:, :3], v, log_decay), {}, ValueError),
        ((q, k, v[:, :, :1], log_decay), {}, ValueError), ((q[:, :, :3], k, v, log_decay[:3]), {}, ValueError),
        ((q, k[..., :4], v, log_decay), {}, ValueError), ((q, k, v, log_decay[:2]), {}, ValueError),
        ((q, k, v, log_decay.double()), {}, ValueError), ((q, k, v, log_decay.cpu()), {}, RuntimeError),
        ((q, k, v, log_decay.clone().requires_grad_()), {}, ValueError),
        ((q, k, v, log_decay), {"scale": math.inf}, ValueError),
        ((q, k, v, log_decay), {"row_mask": torch.ones(2, 4, device="cuda")}, ValueError),
        ((q, k, v, log_decay), {"row_mask": torch.ones(2, 3, dtype=torch.bool, device="cuda")}, ValueError),
        ((q, k, v, log_decay), {"row_mask": torch.ones(2, 4, dtype=torch.bool)}, RuntimeError),
        ((q, k, v, log_decay), {"initial_state": state.half()}, ValueError),
        ((q, k, v, log_decay), {"initial_state": state[:1]}, ValueError),
        ((q, k, v, log_decay), {"initial_state": state.cpu()}, RuntimeError),
    ):
        with pytest.raises(error):
            native.linear_attention(*arguments, **keywords)
    wide = torch.zeros(1, 2, 1, 129, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        native.linear_attention(wide, wide, wide, log_decay[:1])
    one = (q[:, 0], k[:, 0], v[:, 0], log_decay)
    for arguments, error in (
        ((*one, state.transpose(0, 1)), ValueError), ((*one, state.mT.contiguous().mT), ValueError),
        ((*one, state[:1].expand(2, -1, -1, -1)), ValueError), ((*one, state.half()), ValueError),
        ((*one, state.cpu()), RuntimeError), ((q, k, v, log_decay, state), ValueError),
        ((q[:, 0].clone().requires_grad_(), *one[1:], state), RuntimeError),
        ((*one, state.clone().requires_grad_()), RuntimeError),
    ):
        with pytest.raises(error):
            native.linear_attention_step(*arguments)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError):
            native.linear_attention(dual, k, v, log_decay)
        with pytest.raises(NotImplementedError):
            native.linear_attention_step(dual[:, 0], *one[1:], state)
