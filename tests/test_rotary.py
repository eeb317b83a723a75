"""Rotary positions: frequencies, the reference path and the native kernel against
complex numbers in FP64; layouts, positions, strides, gradients and refusals."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from lsso_amd.ball import causal, hip, rotary_amplitude, rotary_frequencies
from lsso_amd.ball import reference as canonical

TYPES = (torch.float16, torch.bfloat16, torch.float32)


def _turned(x, position_ids, frequencies, layout, amplitude=1.0, sign=1.0):
    """x's pairs as complex numbers times amplitude e^(i angle), FP64."""

    position_ids = torch.arange(x.shape[1]) if position_ids is None else position_ids.cpu()
    angle = sign * position_ids.double()[..., None, None] * frequencies.cpu()
    wheel = torch.polar(torch.full_like(angle, amplitude), angle)
    count = 2 * frequencies.shape[0]
    x = x.detach().cpu().double()
    pairs = x[..., :count].unflatten(-1, (2, -1)).mT if layout == "half" else x[..., :count].unflatten(-1, (-1, 2))
    pairs = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * wheel)
    return torch.cat(((pairs.mT if layout == "half" else pairs).flatten(-2), x[..., count:]), dim=-1)


def test_frequencies() -> None:
    f = rotary_frequencies(8)
    assert f.dtype == torch.float64
    torch.testing.assert_close(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14, atol=0)
    assert torch.equal(rotary_frequencies(8, scaling="linear", factor=4.0), f / 4)
    base = rotary_frequencies(8, scaling="base", factor=16.0)
    torch.testing.assert_close(base[[0, -1]], torch.stack((f[0], f[-1] / 16)), rtol=1e-13, atol=0)
    # Over 2 pi 1,000 positions the pairs make 1,000, 100, 10 and 1 turns.
    turns = rotary_frequencies(8, scaling="turns", factor=4.0, original_length=6283, few_turns=4.0, many_turns=50.0)
    kept = (f[2] * 6283 / (2 * math.pi) - 4) / 46
    expected = torch.stack((f[0], f[1], f[2] * (kept + (1 - kept) / 4), f[3] / 4))
    torch.testing.assert_close(turns, expected, rtol=1e-13, atol=0)
    assert rotary_amplitude(1.0) == 1.0 and rotary_amplitude(math.e) == pytest.approx(1.1)
    for wrong, error in (({"rotary_features": 7}, ValueError), ({"rotary_features": 0}, ValueError),
                         ({"rotary_features": 8.0}, TypeError), ({"rotary_features": 8, "base": 0.0}, ValueError),
                         ({"rotary_features": 8, "factor": 0.0}, ValueError),
                         ({"rotary_features": 8, "scaling": "other"}, ValueError),
                         ({"rotary_features": 2, "scaling": "base"}, ValueError),
                         ({"rotary_features": 8, "scaling": "turns"}, ValueError)):
        with pytest.raises(error):
            rotary_frequencies(**wrong)


@pytest.mark.parametrize("layout", ("interleaved", "half"))
def test_reference(layout) -> None:
    generator = torch.Generator().manual_seed(0)
    q, k = (torch.randn(2, 5, h, 10, generator=generator, dtype=torch.float64) for h in (3, 1))
    f = rotary_frequencies(6)
    ids = torch.randint(0, 10**6, (2, 5), generator=generator)
    for positions in (None, ids[0], ids):
        a, b = canonical.rotary(q, k, positions, f, layout=layout, amplitude=1.25)
        torch.testing.assert_close(a, _turned(q, positions, f, layout, 1.25), rtol=1e-12, atol=1e-12)
        torch.testing.assert_close(b, _turned(k, positions, f, layout, 1.25), rtol=1e-12, atol=1e-12)
    assert canonical.rotary(q, None, ids, f, layout=layout)[1] is None
    assert torch.autograd.gradcheck(
        lambda x: canonical.rotary(x, None, ids, f, layout=layout)[0], q.requires_grad_())
    with pytest.raises(ValueError):
        canonical.rotary(q, k, ids, f, layout="other")


def test_refusals_on_the_cpu() -> None:
    library = hip.open_library()

    def call(x=16, y=16, heads=2, stride=8, count=1, dtype=2, batch=1, length=3, features=8, rotary=8, layout=1,
             frequencies=16, ids=None, kind=0, tensors=True):
        array = (causal.RotaryTensor * 2)()
        for i in range(2):
            array[i] = causal.RotaryTensor(x, y, heads, 48, 16, stride)
        return library.lsso_hip_rotary(array if tensors else None, count, dtype, batch, length, features, rotary, layout,
                                       frequencies, 1.0, 0, ids, kind, 0, 1, None)

    assert call(batch=0) == 0 and call(length=0, x=None, y=None) == 0
    for wrong in ({"tensors": False}, {"count": 0}, {"count": 3}, {"x": None}, {"y": None}, {"x": 17}, {"y": 18, "dtype": 3},
                  {"heads": 0}, {"heads": 5000}, {"stride": -1}, {"dtype": 4}, {"batch": -1}, {"length": -1},
                  {"features": 0}, {"features": 4098, "rotary": 4098}, {"rotary": 7}, {"rotary": 10}, {"rotary": 0},
                  {"layout": 3}, {"frequencies": None}, {"frequencies": 20}, {"kind": 5}, {"kind": 2},
                  {"kind": 2, "ids": 20}, {"kind": -1}, {"batch": 2**21, "length": 2**21}):
        assert call(**wrong) < 0, wrong
        assert library.lsso_hip_last_error()


def _bound(expected, x, frequencies, layout, amplitude, dtype):
    """cos and sin: the angle's turns rounded to FP32 (2^-25 of a turn: 2^-22.3), 2 ulp
    of the function and one of the amplitude (2^-22); two products and a sum of FP32
    (2^-22 of the terms); one rounding to the type, FP16 below its normal range to
    half of 2^-24."""

    count = 2 * frequencies.shape[0]
    x = x.detach().cpu().double().abs()
    pairs = x[..., :count].unflatten(-1, (2, -1)).mT if layout == "half" else x[..., :count].unflatten(-1, (-1, 2))
    sums = pairs.sum(-1, keepdim=True).expand(pairs.shape)
    terms = torch.cat(((sums.mT if layout == "half" else sums).flatten(-2), torch.zeros_like(x[..., count:])), dim=-1)
    return 2.0**-20 * amplitude * terms + torch.finfo(dtype).eps / 2 * expected.abs() * (1 + 2.0**-10) + 2.0**-25


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ("interleaved", "half"))
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 2, 2), (2, 3, 3, 1, 64, 64), (1, 17, 2, 4, 40, 20), (3, 5, 1, 1, 33, 30),
                                  (1, 200, 4, 2, 128, 64), (2, 7, 5, 5, 13, 12), (1, 3, 2, 1, 300, 258), (1, 2, 1, 1, 4096, 4096)])
def test_values_and_gradients(native, dtype, layout, size) -> None:
    batch, length, heads, kv_heads, features, turned = size
    generator = torch.Generator().manual_seed(1)
    q, k, dq, dk = (torch.randn(batch, length, h, features, generator=generator).to(dtype)
                    for h in (heads, kv_heads, heads, kv_heads))
    f = rotary_frequencies(turned).cuda()
    ids = torch.randint(0, 10**6, (batch, length), generator=generator)
    a, b = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    for positions in (None, ids[0], ids, ids.int(), ids.float() + 0.25, ids.double() + 0.125):
        where = None if positions is None else positions.cuda()
        turned_pair = native.rotary(a, b, where, f, layout=layout, amplitude=1.25)
        grads = torch.autograd.grad(turned_pair, (a, b), (dq.cuda(), dk.cuda()))
        for x, y, sign in ((q, turned_pair[0], 1), (k, turned_pair[1], 1), (dq, grads[0], -1), (dk, grads[1], -1)):
            expected = _turned(x, positions, f, layout, 1.25, sign)
            assert y.dtype == dtype and y.is_contiguous()
            off = (y.detach().cpu().double() - expected).abs()
            assert (off <= _bound(expected, x, f, layout, 1.25, dtype)).all()
            # What is not turned is copied.
            assert torch.equal(y.detach().cpu()[..., 2 * f.shape[0]:], x[..., 2 * f.shape[0]:])


@pytest.mark.gpu
def test_far_positions_keep_their_phases(native) -> None:
    """2^31 and more positions on: the angle's turns have 20 bits left of 52."""

    x = torch.ones(1, 4, 1, 8, device="cuda")
    f = rotary_frequencies(8).cuda()
    ids = torch.tensor([2**31 - 1, 2**31, 2**32 + 3, 2**33 + 7], device="cuda")
    y, _ = native.rotary(x, None, ids, f)
    assert ((y.cpu().double() - _turned(x, ids, f, "interleaved")).abs() < 4e-5).all()
    # A distance is what the product of two turned vectors shows.
    near, _ = native.rotary(x, None, ids - 2**31, f)
    torch.testing.assert_close((y[0, 0, 0] * y[0, 1, 0]).sum(), (near[0, 0, 0] * near[0, 1, 0]).sum(), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ("interleaved", "half"))
def test_layouts(native, dtype, layout) -> None:
    generator = torch.Generator().manual_seed(2)
    q, k = (torch.randn(2, 9, h, 24, generator=generator).to(dtype).cuda() for h in (4, 2))
    f = rotary_frequencies(24).cuda()
    ids = torch.randint(0, 1000, (2, 9), generator=generator).cuda()
    plain = native.rotary(q, k, ids, f, layout=layout)
    packed = torch.cat((q, k), dim=2)
    for a, b in (packed.split((4, 2), dim=2), (q.transpose(1, 2).contiguous().transpose(1, 2), k),
                 (q.mT.contiguous().mT, k.mT.contiguous().mT)):
        for x, y in zip(native.rotary(a, b, ids, f, layout=layout), plain):
            assert torch.equal(x, y)
    room = torch.zeros(2 * 9 * 4 * 25 + 1, dtype=dtype, device="cuda")
    odd = room[1:].view(2, 9, 4, 25)[..., :24]
    odd.copy_(q)
    assert torch.equal(native.rotary(odd, None, ids, f, layout=layout)[0], plain[0])
    # Positions read at their strides, and broadcast.
    wide = torch.zeros(2, 9, 3, dtype=torch.int64, device="cuda")
    wide[..., 1] = ids
    assert torch.equal(native.rotary(q, None, wide[..., 1], f, layout=layout)[0], plain[0])
    assert torch.equal(native.rotary(q, None, ids[:1].expand(2, -1), f, layout=layout)[0],
                       native.rotary(q, None, ids[0], f, layout=layout)[0])
    one = q[:1, :, :1].detach().requires_grad_()
    y, _ = native.rotary(one.expand(2, -1, 4, -1), None, ids, f, layout=layout)
    assert torch.equal(y, native.rotary(one.detach().expand(2, -1, 4, -1).contiguous(), None, ids, f, layout=layout)[0])
    (grad,) = torch.autograd.grad(y.float().sum(), one)   # dy is one value, broadcast
    back = _turned(torch.ones_like(y), ids, f, layout, sign=-1)
    half = torch.finfo(dtype).eps / 2
    bound = 9 * half * (back.abs().sum((0, 2)) + 1)       # eight values of one rounding each, and their sum's
    assert ((grad.cpu().double()[0, :, 0] - back.sum((0, 2))).abs() <= bound).all()


@pytest.mark.gpu
def test_only_what_is_asked_for(native) -> None:
    q, k = (torch.randn(1, 6, h, 16, device="cuda").half() for h in (2, 1))
    f = rotary_frequencies(16).cuda()
    k.requires_grad_()
    a, b = native.rotary(q, k, None, f)
    (grad,) = torch.autograd.grad(b, k, torch.ones_like(b))
    expected, _ = native.rotary(torch.ones_like(k.detach()), None, -torch.arange(6, device="cuda"), f)
    assert torch.equal(grad, expected)   # turned back: as at the opposite position
    y, none = native.rotary(k, None, None, f)
    assert none is None and torch.equal(y, b)
    empty = torch.empty(0, 5, 2, 16, device="cuda", requires_grad=True)
    assert native.rotary(empty, None, None, f)[0].shape == (0, 5, 2, 16)


@pytest.mark.gpu
def test_elements_past_32_bits(native) -> None:
    count = (1 << 31) // 1024 + 3
    x = torch.ones(1, count, 4, 256, dtype=torch.float16, device="cuda")
    f = rotary_frequencies(256).cuda()
    y, _ = native.rotary(x, None, None, f, layout="half")
    last = slice(count - 2, count)
    expected = _turned(x[:, last], torch.arange(count - 2, count), f, "half")
    assert ((y[:, last].cpu().double() - expected).abs() <= _bound(expected, x[:, last], f, "half", 1.0, torch.float16)).all()


@pytest.mark.gpu
def test_captured_replays(native) -> None:
    q, k = (torch.randn(2, 33, h, 64, device="cuda").bfloat16().requires_grad_() for h in (4, 2))
    ids = torch.zeros(2, 33, dtype=torch.int64, device="cuda")
    f = rotary_frequencies(64).cuda()

    def run():
        turned = native.rotary(q, k, ids, f, layout="half")
        return [*turned, *torch.autograd.grad(turned, (q, k), turned)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for step in range(3):
        ids.copy_(torch.arange(33, device="cuda") + 100 * step)
        graph.replay()
        for a, b in zip(captured, run()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals(native) -> None:
    q, k = (torch.randn(2, 5, h, 16, device="cuda") for h in (4, 2))
    f = rotary_frequencies(16).cuda()
    ids = torch.arange(5, device="cuda")
    for arguments, keywords, error in (
        ((q.cpu(), None, None, f), {}, RuntimeError), ((q.double(), None, None, f), {}, TypeError),
        ((q[0], None, None, f), {}, ValueError), ((q, k.cpu(), None, f), {}, RuntimeError),
        ((q, k.half(), None, f), {}, TypeError), ((q, k[:, :3], None, f), {}, ValueError),
        ((q, k[..., :8], None, f), {}, ValueError), ((q, k, None, f.float()), {}, TypeError),
        ((q, k, None, f.cpu()), {}, RuntimeError), ((q, k, None, f[:0]), {}, ValueError),
        ((q, k, None, torch.cat((f, f))), {}, ValueError), ((q, k, None, f.clone().requires_grad_()), {}, ValueError),
        ((q, k, ids[:4], f), {}, ValueError), ((q, k, ids.expand(3, -1), f), {}, ValueError),
        ((q, k, ids.half(), f), {}, TypeError), ((q, k, ids.cpu(), f), {}, RuntimeError),
        ((q, k, ids.float().requires_grad_(), f), {}, ValueError), ((q, k, ids, f), {"layout": "other"}, ValueError),
    ):
        with pytest.raises(error):
            native.rotary(*arguments, **keywords)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError):
            native.rotary(dual, None, None, f)
