"""Residual dropout: the generator against its published known answers and an
independent numpy form, the native kernel against the mask in FP64, gradients,
captured replays and refusals."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from lsso_amd.ball import ResidualDropout, block, hip
from lsso_amd.ball import reference as canonical

TYPES = (torch.float16, torch.bfloat16, torch.float32)


def _philox(counter, key):
    """One Philox-4x32-10 block in Python integers."""

    c, k = list(counter), list(key)
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k[1], p & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def _keep(count, threshold, seed, offset):
    seed, offset = seed % 2**64, offset % 2**64
    values = []
    for group in range((count + 7) // 8):
        words = _philox((group & 0xFFFFFFFF, group >> 32, offset & 0xFFFFFFFF, offset >> 32),
                        (seed & 0xFFFFFFFF, seed >> 32))
        values += [half for word in words for half in (word & 0xFFFF, word >> 16)]
    return torch.from_numpy(np.array(values[:count]) >= threshold)


def test_generator_matches_its_known_answers() -> None:
    # Known answers that its authors publish with the generator.
    assert _philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert _philox((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("seed,offset", [(0, 0), (2**63 + 5, 2**40 + 1), (-1, -1), (12345678901234, 7)])
def test_reference_mask_is_the_generator(seed, offset) -> None:
    mask = canonical.dropout_keep(torch.Size((7, 11)), 6554, seed % 2**64, offset % 2**64, torch.device("cpu"))
    assert torch.equal(mask.reshape(-1), _keep(77, 6554, seed, offset))


def test_threshold() -> None:
    assert [block.dropout_threshold(p) for p in (0.0, 0.1, 0.5, 1 - 2**-20)] == [0, 6554, 32768, 65535]
    for p in (-0.1, 1.0, math.nan):
        with pytest.raises(ValueError):
            block.dropout_threshold(p)


def test_module_on_the_cpu() -> None:
    layer = ResidualDropout(0.25)
    x, r = torch.randn(3, 5, requires_grad=True), torch.randn(3, 5)
    keep = _keep(15, 16384, 9, 2).view(3, 5)
    y = layer(x, r, seed=9, offset=2)
    assert torch.allclose(y, r + keep * x / 0.75)
    assert torch.equal(layer(x, r, seed=torch.tensor([9, 2]), offset=0), y)
    (grad,) = torch.autograd.grad(y.sum(), x)
    assert torch.allclose(grad, keep / 0.75)
    assert torch.equal(layer.eval()(x, r, seed=9), r + x)
    with pytest.raises(ValueError):
        layer(x, r, seed=9, implementation="other")


def test_native_evaluation_calls_the_kernel(monkeypatch) -> None:
    """With probability 0, so that it refuses what training refuses."""

    monkeypatch.setattr(hip, "dropout_add", lambda *arguments: arguments)
    x, r = torch.randn(2, 3), torch.randn(2, 3)
    layer = ResidualDropout(0.25)
    for implementation in ("hip", "cuda"):
        assert layer.train()(x, r, seed=9, offset=2, implementation=implementation) == (x, r, 0.25, 9, 2)
        assert layer.eval()(x, r, seed=9, offset=2, implementation=implementation) == (x, r, 0.0, 9, 2)


def test_refusals_on_the_cpu() -> None:
    library = hip.open_library()

    def call(x=16, residual=None, dtype=2, count=8, threshold=5, state=None, y=16):
        return library.lsso_hip_dropout_add(x, residual, dtype, count, threshold, 1, 2, state, y, None)

    assert call(count=0, x=None, y=None) == 0
    for wrong in ({"count": -1}, {"count": 2**34 + 1}, {"dtype": 4}, {"threshold": 65536}, {"x": None}, {"y": None},
                  {"x": 17}, {"residual": 18, "dtype": 3}, {"y": 18, "dtype": 3}, {"state": 12}):
        assert call(**wrong) < 0, wrong
        assert library.lsso_hip_last_error()


def _expected(x, r, keep, scale):
    kept = torch.where(keep, x.double() * scale, 0.0)
    return kept if r is None else r.double() + kept


def _bound(expected, x, scale, dtype):
    # Three FP32 roundings (scale, product, sum) of terms no larger than
    # |x| scale + |y|, then one to the type; FP16 below its normal range rounds
    # by half of 2^-24.
    half = torch.finfo(dtype).eps / 2
    terms = x.double().abs() * scale + expected.abs()
    return 3 * 2.0**-24 * terms + half * expected.abs() * (1 + 2.0**-10) + 2.0**-25


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 301), (2, 5, 192), (2049, 17)])
@pytest.mark.parametrize("residual", (True, False))
def test_values_and_gradients(native, dtype, shape, residual) -> None:
    generator = torch.Generator().manual_seed(1)
    x, r, dy = (torch.randn(shape, generator=generator).to(dtype) for _ in range(3))
    seed, offset, p = 0x123456789ABCDEF, 2**33 + 1, 0.3
    keep = canonical.dropout_keep(x.shape, block.dropout_threshold(p), seed, offset, torch.device("cpu"))
    scale = 65536 / (65536 - block.dropout_threshold(p))
    xd = x.cuda().requires_grad_()
    rd = r.cuda().requires_grad_() if residual else None
    y = native.dropout_add(xd, rd, p, seed, offset)
    assert y.is_contiguous() and y.dtype == dtype
    expected = _expected(x, r if residual else None, keep, scale)
    assert ((y.detach().cpu().double() - expected).abs() <= _bound(expected, x, scale, dtype)).all()
    grads = torch.autograd.grad(y, (xd, rd) if residual else (xd,), dy.cuda())
    expected = _expected(dy, None, keep, scale)
    assert ((grads[0].cpu().double() - expected).abs() <= _bound(expected, dy, scale, dtype)).all()
    if residual:
        assert torch.equal(grads[1].cpu(), dy)


@pytest.mark.gpu
def test_first_elements_are_the_integers_generator(native) -> None:
    x = torch.ones(50, device="cuda")
    for seed, offset in ((0, 0), (-1, -1), (2**63 + 5, 2**40 + 1)):
        y = native.dropout_add(x, None, 0.5, seed, offset)
        assert torch.equal(y.cpu() != 0, _keep(50, 32768, seed, offset))


@pytest.mark.gpu
def test_elements_past_32_bits(native) -> None:
    count = (1 << 31) + 29
    y = native.dropout_add(torch.ones(count, dtype=torch.float16, device="cuda"), None, 0.5, 9, 4)
    first = (1 << 31) - 24   # the first element of a block of 8
    values = []
    for group in range(first // 8, (count + 7) // 8):
        words = _philox((group & 0xFFFFFFFF, group >> 32, 4, 0), (9, 0))
        values += [half >= 32768 for word in words for half in (word & 0xFFFF, word >> 16)]
    assert torch.equal(y[first:].cpu(), 2.0 * torch.tensor(values[:count - first]).half())


@pytest.mark.gpu
def test_layouts_do_not_change_the_mask(native) -> None:
    base = torch.randn(40, 24, device="cuda")
    plain = native.dropout_add(base, None, 0.4, 5)
    assert torch.equal(native.dropout_add(base.t().contiguous().t(), None, 0.4, 5), plain)
    room = torch.zeros(40 * 24 + 1, device="cuda")
    room[1:] = base.reshape(-1)   # a base that is aligned to one element only
    assert torch.equal(native.dropout_add(room[1:].view(40, 24), None, 0.4, 5), plain)
    broadcast = torch.randn(1, 24, device="cuda", requires_grad=True)
    y = native.dropout_add(broadcast.expand(40, 24), None, 0.4, 5)
    (grad,) = torch.autograd.grad(y, broadcast, torch.ones_like(y))
    keep = canonical.dropout_keep(torch.Size((40, 24)), block.dropout_threshold(0.4), 5, 0, torch.device("cpu"))
    torch.testing.assert_close(grad.cpu()[0], keep.sum(0).float() * 65536 / (65536 - 26214), rtol=1e-5, atol=0)


@pytest.mark.gpu
def test_dropped_elements_and_probability_zero(native) -> None:
    x = torch.full((64,), math.inf, device="cuda")
    r = torch.arange(64.0, device="cuda")
    y = native.dropout_add(x, r, 0.5, 3)
    keep = _keep(64, 32768, 3, 0)
    assert torch.equal(y.cpu(), torch.where(keep, x.cpu(), r.cpu()))
    assert torch.equal(native.dropout_add(r, r, 0.0, 3), 2 * r)
    empty = torch.empty(0, 8, device="cuda", requires_grad=True)
    assert native.dropout_add(empty, None, 0.5, 3).shape == (0, 8)


@pytest.mark.gpu
def test_replays_read_the_state(native) -> None:
    x = torch.randn(65, 33, device="cuda", dtype=torch.bfloat16)
    r = torch.randn_like(x)
    state = torch.tensor([77, 0], device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        native.dropout_add(x, r, 0.2, state, 4)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = native.dropout_add(x, r, 0.2, state, 4)
        state[1] += 1
    seen = []
    for step in range(4):
        graph.replay()
        assert torch.equal(y, native.dropout_add(x, r, 0.2, 77, 4 + step))
        seen.append(y.clone())
    assert not torch.equal(seen[0], seen[1])


@pytest.mark.gpu
def test_state_changed_before_the_backward_is_refused(native) -> None:
    x = torch.randn(8, device="cuda", requires_grad=True)
    state = torch.tensor([1, 2], device="cuda")
    y = native.dropout_add(x, None, 0.2, state)
    state += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
def test_refusals(native) -> None:
    x = torch.randn(4, 8, device="cuda")
    for arguments, error in (
        ((x.cpu(), None, 0.1, 1), RuntimeError), ((x.double(), None, 0.1, 1), TypeError),
        ((x, x.half(), 0.1, 1), ValueError), ((x, x[:2], 0.1, 1), ValueError), ((x, x.cpu(), 0.1, 1), RuntimeError),
        ((x, None, 1.0, 1), ValueError), ((x, None, 0.1, torch.zeros(3, dtype=torch.int64, device="cuda")), ValueError),
        ((x, None, 0.1, torch.zeros(2, dtype=torch.int32, device="cuda")), ValueError),
        ((x, None, 0.1, torch.zeros(2, dtype=torch.int64)), RuntimeError),
    ):
        with pytest.raises(error):
            native.dropout_add(*arguments)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_native_evaluation(native, dtype) -> None:
    layer = ResidualDropout(0.25).eval()
    x, r = (torch.randn(5, 37, device="cuda").to(dtype) for _ in range(2))
    assert torch.equal(layer(x, r, seed=1, implementation="hip"), r + x)
    assert torch.equal(layer(x, seed=1, implementation="hip"), x)
    other = torch.float16 if dtype == torch.float32 else torch.float32
    for arguments, error in (((x.cpu(), r.cpu()), RuntimeError), ((x, r.cpu()), RuntimeError), ((x, r[:1]), ValueError),
                             ((x, r.to(other)), ValueError), ((x.double(), r.double()), TypeError)):
        for mode in (True, False):
            with pytest.raises(error):
                layer.train(mode)(*arguments, seed=1, implementation="hip")
