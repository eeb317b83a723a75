"""Workspaces of linear attention: the sizes that are asked for hold what the kernels
of the same shape write, and heads of more than 64 features in several pieces a
segment are what the definition says."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lsso_amd.ball import causal, hip
from lsso_amd.ball import reference as canonical
from test_linear_attention import HALVES, _bound, _inputs, _mask


def _up(n, d):
    return -(-n // d)


def _round256(size):
    return -(-size // 256) * 256


def _plan(batch, length, heads, features, out):
    """(segments, pieces) of a walk: as many segments of two and more chunks as the
    device holds workgroups, three to each of 256 compute units or, of more than 64
    features, two; pieces of all but the last until there are 1,024."""

    chunks = _up(length, 64)
    wide = features > 64 or out > 64
    blocks = batch * heads * (2 if features > 64 and out > 64 else 1)

    def parts(held, whole):
        return max(1, min(held // blocks, (whole + 1) // 2))

    segment = _up(chunks, parts(512 if wide else 768, chunks))
    segments = _up(chunks, segment)
    each = parts(1024 // (segments - 1), segment) if segments > 1 else 1
    return segments, (segments - 1) * _up(segment, _up(segment, each))


SHAPES = [(1, 4864, 8, 128, 128), (11, 791, 12, 80, 40), (11, 3188, 3, 128, 16), (1, 6242, 12, 80, 48),
          (2, 3884, 32, 128, 128), (2, 4096, 6, 128, 128), (64, 2048, 4, 64, 64), (1, 32768, 8, 64, 64), (3, 1, 2, 8, 8),
          (1, 129, 1, 65, 1), (1, 129, 1, 1, 65), (7, 1000, 5, 66, 3), (1, 1 << 20, 1, 128, 128)]


@pytest.mark.parametrize("shape", SHAPES)
def test_sizes_hold_what_is_launched(shape) -> None:
    library = hip.open_library()
    batch, length, heads, features, out = shape
    for size in ((features, out), (out, features)):
        native = causal.LinearAttentionShape(
            batch, length, heads, heads, *size, 1, 1.0, *(causal.HeadStrides(length * heads * f, heads * f, f)
                                                          for f in (size[0], size[0], size[1])))
        kept, forward, backward = (ctypes.c_size_t() for _ in range(3))
        assert library.lsso_hip_linear_attention_sizes(
            ctypes.byref(native), *(ctypes.byref(s) for s in (kept, forward, backward))) == 0
        segments, pieces = _plan(*shape)
        if segments == 1:
            assert kept.value == 0 and forward.value == 0 and backward.value == 0
            continue
        state = batch * heads * features * out
        assert kept.value == state * segments
        needed = _round256(4 * state * pieces) + _round256(4 * batch * pieces) + _round256(4 * state * segments)
        assert forward.value == needed and backward.value == needed


def _leaves(size, dtype, kind, seed):
    q, k, v, log_decay, generator = _inputs(*size, dtype, seed)
    mask = _mask(kind, size[0], size[1], generator)
    state, ds = (torch.randn(size[0], size[2], size[4], size[5], generator=generator).cuda() for _ in range(2))
    dy = torch.randn(size[0], size[1], size[2], size[5], generator=generator).to(dtype).cuda()
    return [x.cuda() for x in (q, k, v, state)], log_decay.cuda(), None if mask is None else mask.cuda(), dy, ds


def _exact(inputs, log_decay, mask, dy, ds, scale, f):
    """Values and gradients of the reference path in FP64 (itself tested against the
    definition), of f of the inputs."""

    ends = [f(x.detach().double()).requires_grad_() for x in inputs]
    ys = canonical.linear_attention(*ends[:3], log_decay.double(), scale=scale, row_mask=mask, initial_state=ends[3],
                                    return_state=True)
    return [*ys, *torch.autograd.grad(ys, ends, (f(dy.double()), f(ds.double())))]


WIDE = [(1, 4864, 8, 8, 128, 128), (11, 791, 12, 4, 80, 40), (2, 1500, 3, 1, 128, 16), (1, 1800, 2, 2, 24, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("size", WIDE)
@pytest.mark.parametrize("kind", (None, "suffix", "holes"))
def test_wide_segments(native, dtype, size, kind) -> None:
    """Several pieces to a segment of more than 64 features: values, states and
    gradients, from the forward's states (dq) and those of dv, transposed (dk)."""

    inputs, log_decay, mask, dy, ds = _leaves(size, dtype, kind, 7)
    leaves = [x.requires_grad_() for x in inputs]
    ys = native.linear_attention(*leaves[:3], log_decay, row_mask=mask, initial_state=leaves[3], return_state=True)
    found = [*ys, *torch.autograd.grad(ys, leaves, (dy, ds))]
    scale = size[4] ** -0.5
    values = _exact(inputs, log_decay, mask, dy, ds, scale, lambda x: x)
    sizes = _exact(inputs, log_decay, mask, dy, ds, scale, torch.abs)
    small = 8.0 + scale * size[4]
    for a, e, m in zip(found, values, sizes):
        assert ((a.detach().double() - e.detach()).abs() <= _bound(e.detach(), m.detach(), dtype, small)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
def test_wide_segments_alone(native, dtype) -> None:
    """Without gradients, and each gradient by itself: as in one call of all.  dk by
    itself makes states of its own, where it reads those of dv, transposed: then both
    are within their bound of the same value."""

    size = (3, 900, 6, 6, 96, 80)
    inputs, log_decay, mask, dy, _ = _leaves(size, dtype, "suffix", 8)
    leaves = [x.clone().requires_grad_() for x in inputs]

    def run(q, k, v, state):
        return native.linear_attention(q, k, v, log_decay, row_mask=mask, initial_state=state, return_state=True)

    y, last = run(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    alone, state = run(*inputs)
    assert torch.equal(alone, y) and torch.equal(state, last)
    sizes = [x.abs().requires_grad_() for x in inputs]
    (most,) = torch.autograd.grad(run(*sizes)[0], sizes[1], dy.abs())
    for i in range(4):
        one = [x.clone().requires_grad_(j == i) for j, x in enumerate(inputs)]
        (grad,) = torch.autograd.grad(run(*one)[0], one[i], dy)
        if i != 1:
            assert torch.equal(grad, grads[i])
        else:
            bound = 2 * _bound(grads[1].double(), most.double(), dtype, 8.0 + 96**0.5)
            assert ((grad.double() - grads[1].double()).abs() <= bound).all()
