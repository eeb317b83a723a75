"""Group norm with an activation, channels last: the reference path and the native
kernels against the formula in FP64; both forms, masks, layouts, gradients, captured
replays and refusals."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from lsso_amd.ball import GroupNorm, causal, hip
from lsso_amd.ball import reference as canonical

TYPES = (torch.float16, torch.bfloat16, torch.float32)
ACTIVATIONS = (None, "silu", "gelu")


def _act(z, name):
    return z if name is None else z * (torch.sigmoid(z) if name == "silu" else torch.special.ndtr(z))


def _formula(x, groups, weight, bias, eps, activation, mask):
    """FP64, sample by sample and group by group, over the kept tokens alone."""

    samples, channels = x.shape[0], x.shape[-1]
    rows = x.reshape(samples, -1, channels)
    results = []
    for s in range(samples):
        kept = torch.ones(rows.shape[1], dtype=torch.bool) if mask is None else mask.reshape(samples, -1)[s]
        some = rows[s][kept].double()
        y = torch.zeros(rows.shape[1], channels, dtype=torch.float64)
        if some.numel():
            parts = some.unflatten(-1, (groups, -1))
            mean = parts.mean((0, 2), keepdim=True)
            variance = (parts - mean).square().mean((0, 2), keepdim=True)
            z = ((parts - mean) / torch.sqrt(variance + eps)).flatten(-2) * weight + bias
            y = y.index_put((kept.nonzero()[:, 0],), _act(z, activation))
        results.append(y)
    return torch.stack(results).reshape(x.shape) if results else torch.zeros(x.shape, dtype=torch.float64)


def _inputs(shape, dtype, seed=0, mean=0.5):
    generator = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=generator) + mean).to(dtype)
    weight = 1.0 + 0.3 * torch.randn(shape[-1], generator=generator)
    bias = 0.3 * torch.randn(shape[-1], generator=generator)
    dy = torch.randn(shape, generator=generator).to(dtype)
    return x, weight, bias, dy, generator


# ------------------------------------------------------------------- reference
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("masked", (False, True))
def test_reference(activation, masked) -> None:
    x, weight, bias, _, generator = _inputs((3, 4, 2, 6), torch.float64)
    mask = torch.rand(3, 4, 2, generator=generator) < 0.6 if masked else None
    if masked:
        mask[2] = False
    arguments = [t.double().requires_grad_() for t in (x, weight, bias)]
    y = canonical.group_norm(arguments[0], 3, *arguments[1:], activation=activation, row_mask=mask)
    torch.testing.assert_close(y, _formula(x, 3, weight.double(), bias.double(), 1e-5, activation, mask), rtol=1e-11,
                               atol=1e-11)
    assert torch.autograd.gradcheck(
        lambda x, w, b: canonical.group_norm(x, 3, w, b, activation=activation, row_mask=mask), arguments)


def test_module_on_the_cpu() -> None:
    layer = GroupNorm(4, 12, activation="silu")
    x = torch.randn(2, 5, 12)
    mask = torch.rand(2, 5) < 0.5
    expected = canonical.group_norm(x, 4, layer.weight, layer.bias, activation="silu", row_mask=mask)
    assert torch.equal(layer(x, mask), expected)
    torch.testing.assert_close(
        GroupNorm(3, 12)(x), torch.nn.functional.group_norm(x.mT, 3).mT, rtol=1e-5, atol=1e-5)
    for wrong, error in (((5, 12), ValueError), ((0, 12), ValueError), ((2.0, 12), TypeError)):
        with pytest.raises(error):
            GroupNorm(*wrong)
    with pytest.raises(ValueError):
        GroupNorm(2, 12, activation="relu")
    with pytest.raises(ValueError):
        layer(x, implementation="other")


def test_refusals_on_the_cpu() -> None:
    library = hip.open_library()
    sizes = [ctypes.c_size_t() for _ in range(3)]

    def shape(samples=2, length=3, channels=8, groups=2, dtype=2, parameter=3, activation=0, eps=1e-5):
        return ctypes.byref(causal.GroupNormShape(samples, length, channels, groups, dtype, parameter, activation, eps))

    def forward(x=16, weight=None, bias=None, statistics=None, y=16, workspace=256, count=1 << 20, **changes):
        return library.lsso_hip_group_norm(shape(**changes), x, weight, bias, None, statistics, y, workspace, count, None)

    def backward(grad=16, x=16, weight=None, statistics=16, grad_x=16, grad_weight=None, workspace=256, count=1 << 20,
                 **changes):
        return library.lsso_hip_group_norm_backward(shape(**changes), grad, x, weight, None, None, statistics, grad_x,
                                                    grad_weight, None, workspace, count, None)

    pointers = [ctypes.byref(size) for size in sizes]
    assert library.lsso_hip_group_norm_sizes(shape(), *pointers) == 0
    assert sizes[0].value == 2 * 2 * 2 and sizes[1].value > 0 and sizes[2].value > 0
    assert library.lsso_hip_group_norm_sizes(shape(length=1), *pointers) == 0
    assert sizes[0].value == 0 and sizes[1].value == 0 and sizes[2].value > 0   # each token by itself: nothing is kept
    for wrong in ({"samples": -1}, {"length": -1}, {"channels": 0}, {"groups": 0}, {"groups": 3}, {"dtype": 4},
                  {"parameter": 1}, {"activation": 3}, {"eps": -1.0}, {"eps": math.nan}, {"eps": math.inf},
                  {"channels": 1 << 21}, {"samples": 1 << 31}, {"samples": 1 << 30, "length": 1 << 30}):
        assert library.lsso_hip_group_norm_sizes(shape(**wrong), *pointers) < 0, wrong
        assert forward(**wrong) < 0 and backward(**wrong) < 0, wrong
        assert library.lsso_hip_last_error()
    assert library.lsso_hip_group_norm_sizes(None, *pointers) < 0
    assert library.lsso_hip_group_norm_sizes(shape(), None, *pointers[1:]) < 0
    assert forward(samples=0, x=None, y=None) == 0
    for wrong in ({"x": None}, {"y": None}, {"x": 17}, {"y": 17}, {"weight": 18}, {"bias": 18}, {"statistics": 18},
                  {"workspace": None}, {"workspace": 128}, {"count": 8}):
        assert forward(**wrong) < 0, wrong
    for wrong in ({"x": None}, {"grad": None}, {"grad": 17}, {"grad_x": 17}, {"weight": 18}, {"grad_weight": 18},
                  {"statistics": None}, {"workspace": None}, {"count": 8}):
        assert backward(**wrong) < 0, wrong


# ---------------------------------------------------------------------- device
# Sums of FP32: up to 256 parts of a workgroup one after another, 64 rows of a thread
# in blocks and 64 splits, each with about three roundings: 2^-24 * 1,024.
DEPTH = 2.0**-14


def _check(native, x, groups, weight, bias, dy, activation, mask, eps=1e-5, parameter=torch.float32):
    dtype = x.dtype
    weight, bias = weight.to(parameter), bias.to(parameter)
    leaves = [t.cuda().requires_grad_() for t in (x, weight, bias)]
    device_mask = None if mask is None else mask.cuda()
    y = native.group_norm(leaves[0], groups, *leaves[1:], eps=eps, activation=activation, row_mask=device_mask)
    found = torch.autograd.grad(y, leaves, dy.cuda())
    ends = [t.double().requires_grad_() for t in (x, weight, bias)]
    expected = _formula(ends[0], groups, *ends[1:], eps, activation, mask)
    grads = torch.autograd.grad(expected, ends, dy.double())
    expected = expected.detach()

    # xhat is off by DEPTH of (|x| + |mean|) rstd, the activation passes 1.13 of that
    # on, and the fast forms of 16-bit outputs are off by 1e-5 of their own value.
    rows = x.double().reshape(x.shape[0], -1, x.shape[-1])
    kept = torch.ones(rows.shape[:2], dtype=torch.bool) if mask is None else mask.reshape(rows.shape[:2])
    safe = torch.where(kept[..., None], rows, 0.0)
    parts = safe.unflatten(-1, (groups, -1))
    count = kept.sum(1).clamp_min(1).view(-1, 1, 1, 1) * parts.shape[-1]
    mean = parts.sum((1, 3), keepdim=True) / count
    centred = torch.where(kept[..., None, None], parts - mean, 0.0)
    rstd = 1.0 / torch.sqrt(centred.square().sum((1, 3), keepdim=True) / count + eps)
    size = (parts.abs().amax((1, 3), keepdim=True) * rstd).expand(parts.shape).flatten(-2)
    normal = (centred * rstd).flatten(-2).abs()
    rstd = rstd.expand(parts.shape).flatten(-2)
    half, fast = torch.finfo(dtype).eps / 2, 0.0 if dtype == torch.float32 else 1e-5
    off = DEPTH * (1 + 2 * size) * weight.double().abs() * 1.13 + fast * expected.reshape(rows.shape).abs() + DEPTH * 0.5
    bound = off + half * (1 + 2.0**-10) * expected.reshape(rows.shape).abs() + 2.0**-25
    assert y.dtype == dtype and y.is_contiguous()
    assert ((y.detach().cpu().double() - expected).abs().reshape(rows.shape) <= bound).all()
    # Gradients: sums of |dy| act' w, act' up to 1.13 and act'' up to 1.13 times z's error.
    dz = torch.where(kept[..., None], dy.double().reshape(rows.shape).abs(), 0.0) * 1.13
    dn = dz * weight.double().abs()

    def group_mean(t):
        return (t.unflatten(-1, (groups, -1)).sum((1, 3), keepdim=True) / count).expand(parts.shape).flatten(-2)

    relative = (DEPTH + fast) * 4 * (1 + 2 * size)
    terms = rstd * (dn + group_mean(dn) + (normal + 1) * group_mean(dn * (normal + 1)))
    bound = relative * terms + half * (1 + 2.0**-10) * grads[0].reshape(rows.shape).abs() + 2.0**-25
    assert ((found[0].cpu().double() - grads[0]).abs().reshape(rows.shape) <= bound).all()
    half = torch.finfo(parameter).eps / 2
    for a, e, m in ((found[1], grads[1], dz * (normal + 1)), (found[2], grads[2], dz)):
        assert a.dtype == parameter
        bound = (relative * m).sum((0, 1)) + half * (1 + 2.0**-10) * e.abs() + 2.0**-25
        assert ((a.cpu().double() - e).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("shape,groups", [((1, 2), 1), ((5, 8), 2), ((70, 256), 4), ((3, 24), 1), ((9, 96), 3), ((4, 100), 4),
                                          ((33, 768), 1), ((2, 2048), 1), ((2, 4104), 1), ((7, 30), 30), ((600, 320), 40),
                                          ((3, 530), 2)])
def test_each_token(native, dtype, activation, shape, groups) -> None:
    x, weight, bias, dy, _ = _inputs(shape, dtype)
    _check(native, x, groups, weight, bias, dy, activation, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("shape,groups", [((1, 2, 1), 1), ((2, 3, 8), 2), ((3, 65, 24), 3), ((2, 14, 14, 64), 32),
                                          ((1, 2000, 20), 4), ((2, 100, 300), 12), ((2, 7, 2080), 4), ((1, 33, 515), 5),
                                          ((40, 2, 16), 2)])
@pytest.mark.parametrize("masked", (False, True))
def test_samples(native, dtype, activation, shape, groups, masked) -> None:
    x, weight, bias, dy, generator = _inputs(shape, dtype, seed=1)
    mask = torch.rand(shape[:-1], generator=generator) < 0.6 if masked else None
    if masked and shape[0] > 1:
        mask[-1] = False   # a sample without a token
    _check(native, x, groups, weight, bias, dy, activation, mask)


@pytest.mark.gpu
def test_masked_tokens_by_themselves(native) -> None:
    x, weight, bias, dy, generator = _inputs((50, 64), torch.bfloat16)
    _check(native, x, 4, weight, bias, dy, "gelu", torch.rand(50, generator=generator) < 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 48), (3, 50, 48)])
def test_parameter_types(native, shape) -> None:
    for dtype in (torch.float16, torch.bfloat16):
        x, weight, bias, dy, _ = _inputs(shape, dtype)
        _check(native, x, 4, weight, bias, dy, "silu", None, parameter=dtype)
        x = x.cuda()
        plain = native.group_norm(x, 4)
        assert torch.equal(plain, native.group_norm(x, 4, torch.ones(48, device="cuda"), torch.zeros(48, device="cuda")))
        w = weight.cuda().requires_grad_()
        y = native.group_norm(x, 4, w)
        assert torch.equal(y, native.group_norm(x, 4, w, torch.zeros(48, device="cuda")))
        assert torch.autograd.grad(y.float().sum(), w)[0].shape == (48,)
        b = bias.cuda().requires_grad_()
        (grad,) = torch.autograd.grad(native.group_norm(x, 4, None, b), b, dy.cuda())
        assert ((grad.cpu().double() - dy.double().reshape(-1, 48).sum(0)).abs() <= DEPTH * dy.double().abs().reshape(-1, 48).sum(0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(64, 256), (2, 3000, 32)])
def test_a_mean_far_from_zero(native, shape) -> None:
    """A spread of 1 around 4,096, and one outlier as the first value."""

    for outlier in (False, True):
        x = torch.randn(shape, generator=torch.Generator().manual_seed(5)) + 4096.0
        if outlier:
            x = x - 4096.0
            x.view(-1)[0] = 10000.0
        y = native.group_norm(x.cuda(), 4)
        expected = _formula(x, 4, torch.ones(shape[-1]).double(), torch.zeros(shape[-1]).double(), 1e-5, None, None)
        # x itself is right to 2^-24; the mean of the group to a few times that of 4,096
        # (or of the outlier): 2^-24 * 4,096 * 16 = 4e-3.
        assert ((y.cpu().double() - expected).abs() <= 4e-3 * (1 + expected.abs())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(20, 64), (2, 90, 64)])
def test_what_the_mask_excludes_reaches_nothing(native, shape) -> None:
    for dtype in TYPES:
        x, weight, bias, dy, generator = _inputs(shape, dtype)
        mask = torch.rand(shape[:-1], generator=generator) < 0.5
        wild, wild_dy = torch.where(mask[..., None], x, math.nan), torch.where(mask[..., None], dy, math.inf)
        results = []
        for values, grads in ((x, dy), (wild, wild_dy)):
            leaves = [t.cuda().requires_grad_() for t in (values, weight, bias)]
            y = native.group_norm(leaves[0], 4, *leaves[1:], activation="gelu", row_mask=mask.cuda())
            results.append([y, *torch.autograd.grad(y, leaves, grads.cuda())])
        for a, b in zip(*results):
            assert torch.equal(a, b)
        assert not results[0][0][~mask.cuda()].any() and not results[0][1][~mask.cuda()].any()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(20, 64), (2, 90, 64)])
def test_layouts_and_repeats(native, shape) -> None:
    x, weight, bias, dy, _ = _inputs(shape, torch.float16)
    x, weight, bias, dy = (t.cuda() for t in (x, weight, bias, dy))
    plain = native.group_norm(x, 4, weight, bias)
    room = torch.zeros(x.numel() + 1, dtype=torch.float16, device="cuda")
    room[1:] = x.reshape(-1)
    assert torch.equal(native.group_norm(room[1:].view(shape), 4, weight, bias), plain)
    assert torch.equal(native.group_norm(x.transpose(0, 1).contiguous().transpose(0, 1), 4, weight, bias), plain)
    leaf = x.clone().requires_grad_()
    first = torch.autograd.grad(native.group_norm(leaf, 4, weight, bias), leaf, dy)[0]
    strided = torch.zeros((*shape[:-1], 2 * shape[-1]), dtype=torch.float16, device="cuda")[..., ::2]
    strided.copy_(dy)
    for _ in range(3):
        assert torch.equal(torch.autograd.grad(native.group_norm(leaf, 4, weight, bias), leaf, strided)[0], first)
    one = x[:1].clone().requires_grad_()
    y = native.group_norm(one.expand(shape), 4, weight, bias)
    (grad,) = torch.autograd.grad(y.float().sum(), one)   # dy is one value, broadcast
    assert grad.shape == one.shape
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = native.group_norm(x, 4, weight, bias)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(y, plain)


@pytest.mark.gpu
def test_empty(native) -> None:
    for shape in ((0, 8), (0, 3, 8), (2, 0, 8)):
        leaves = [torch.empty(shape, device="cuda"), torch.ones(8, device="cuda"), torch.ones(8, device="cuda")]
        leaves = [t.requires_grad_() for t in leaves]
        y = native.group_norm(leaves[0], 2, *leaves[1:])
        assert y.shape == shape
        grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
        assert grads[0].shape == shape and not grads[1].any() and not grads[2].any()


@pytest.mark.gpu
def test_elements_past_32_bits(native) -> None:
    count = (1 << 31) // 512 + 5
    x = torch.zeros(count, 512, dtype=torch.float16, device="cuda")
    x[-3:] = torch.randn(3, 512, device="cuda").half()
    y = native.group_norm(x, 8)
    assert torch.equal(y[-3:], native.group_norm(x[-3:].clone(), 8)) and not y[:8].any()
    del y
    one = native.group_norm(x.view(1, count, 512), 8)
    tail = x[-3:].float().view(3, 8, 64)
    variance = tail.square().sum((0, 2)) / (count * 64)
    expected = tail / torch.sqrt(variance + 1e-5)[None, :, None]
    torch.testing.assert_close(one[0, -3:].float().view(3, 8, 64), expected, rtol=2e-3, atol=2e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(70, 64), (2, 90, 64)])
def test_captured_replays(native, shape) -> None:
    x, weight, bias, dy, _ = _inputs(shape, torch.bfloat16)
    leaves = [t.cuda().requires_grad_() for t in (x, weight, bias)]
    dy = dy.cuda()

    def run():
        y = native.group_norm(leaves[0], 4, *leaves[1:], activation="silu")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for seed in range(3):
        torch.manual_seed(seed)
        with torch.no_grad():
            leaves[0].copy_(torch.randn(shape))
        graph.replay()
        for a, b in zip(captured, run()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals(native) -> None:
    x = torch.randn(3, 5, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for arguments, keywords, error in (
        ((x.cpu(), 2), {}, RuntimeError), ((x.double(), 2), {}, TypeError), ((x[0, 0], 2), {}, ValueError),
        ((x, 3), {}, ValueError), ((x, 0), {}, ValueError), ((x, True), {}, ValueError), ((x, 2.0), {}, ValueError),
        ((x, 2, w.cpu()), {}, RuntimeError), ((x, 2, w.half()), {}, TypeError), ((x, 2, w[:4]), {}, ValueError),
        ((x.half(), 2, w, w.half()), {}, TypeError), ((x, 2, None, w[None]), {}, ValueError),
        ((x, 2), {"activation": "relu"}, ValueError), ((x, 2), {"eps": -1.0}, ValueError),
        ((x, 2), {"eps": math.nan}, ValueError), ((x, 2), {"row_mask": torch.ones(3, 5, device="cuda")}, ValueError),
        ((x, 2), {"row_mask": torch.ones(3, dtype=torch.bool, device="cuda")}, ValueError),
        ((x, 2), {"row_mask": torch.ones(3, 5, dtype=torch.bool)}, RuntimeError),
    ):
        with pytest.raises(error):
            native.group_norm(*arguments, **keywords)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            native.group_norm(dual, 2)
