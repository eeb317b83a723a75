"""What the factors of linear attention's products are held to: outputs of BF16 as
those of FP32 factors, small and large values of FP16, and values that are not finite."""

from __future__ import annotations

import math

import pytest
import torch

from lsso_amd.ball import reference as canonical
from test_linear_attention import _inputs


def _exact(inputs, log_decay, scale, dy, ds):
    """(y, S, dq, dk, dv, dS_0) of the reference path in FP64 (itself tested against
    the definition)."""

    ends = [x.detach().double().requires_grad_() for x in inputs]
    ys = canonical.linear_attention(*ends[:3], log_decay.double(), scale=scale, initial_state=ends[3], return_state=True)
    return [x.detach() for x in (*ys, *torch.autograd.grad(ys, ends, (dy.double(), ds.double())))]


def _native(native, inputs, log_decay, scale, dy, ds):
    leaves = [x.detach().requires_grad_() for x in inputs]
    ys = native.linear_attention(*leaves[:3], log_decay, scale=scale, initial_state=leaves[3], return_state=True)
    return [x.detach() for x in (*ys, *torch.autograd.grad(ys, leaves, (dy, ds)))]


def _tensors(size, dtype, seed=0):
    q, k, v, log_decay, generator = _inputs(*size, dtype, seed)
    state, ds = (torch.randn(size[0], size[2], size[4], size[5], generator=generator) for _ in range(2))
    dy = torch.randn(size[0], size[1], size[2], size[5], generator=generator).to(dtype)
    return [x.cuda() for x in (q, k, v, state)], log_decay.cuda(), dy.cuda(), ds.cuda()


def _apart(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(2, 700, 4, 2, 64, 64), (1, 300, 2, 2, 128, 96), (3, 64, 2, 2, 32, 16)])
def test_bfloat16_outputs_are_those_of_fp32_factors(native, size) -> None:
    """FP32 sums of about 200 terms are off by sqrt(200) 2^-24 = 8e-7 of the result's
    size.  That moves one in 6,000 values over a rounding border (8e-7 of steps of
    2^-8 to 2^-7), by such a step: sqrt(1.6e-4) 5.5e-3 = 7e-5 of the norm.  States and
    their gradients, which are FP32, are off by a few roundings in a row: 2^-21."""

    inputs, log_decay, dy, ds = _tensors(size, torch.bfloat16)
    scale = size[4] ** -0.5
    for i, (a, e) in enumerate(zip(_native(native, inputs, log_decay, scale, dy, ds),
                                   _exact(inputs, log_decay, scale, dy, ds))):
        bound = 2.0**-21 if i in (1, 5) else 8e-5
        assert _apart(a, e.to(a.dtype)) <= bound, i
    # What is returned beside it changes no value.
    assert torch.equal(native.linear_attention(*inputs[:3], log_decay),
                       native.linear_attention(*inputs[:3], log_decay, return_state=True)[0])


def _rounded_once(a, e, m) -> bool:
    """a is e but for one rounding to FP16 (half of 2^-24 below its normal range), the
    parts' 22 bits, FP32 sums of 200 terms and an exponential's last bits: 2^-16 of the
    terms' size m at worst."""

    bound = 2.0**-11 * (1 + 2.0**-10) * e.abs() + 2.0**-25 + 2.0**-16 * m
    return bool(((a.double() - e).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(2, 700, 4, 2, 64, 64), (1, 300, 2, 2, 128, 96), (2, 64, 2, 2, 32, 16), (1, 200, 2, 1, 33, 7)])
@pytest.mark.parametrize("small", (1e-2, 1e-3, 1e-4, 1e-5))
def test_small_float16_values_keep_their_bits_in_states(native, size, small) -> None:
    """S of small v and its gradient of small dy, which are FP32: 22 bits of each term
    and sqrt(200) roundings of the sums, 2^-20 of the norm.  dv and y of them: one
    rounding."""

    inputs, log_decay, dy, ds = _tensors(size, torch.float16)
    scale = size[4] ** -0.5
    inputs[2] = (inputs[2] * small).half()
    inputs[3], ds, dy = inputs[3] * small, ds * small, (dy * small).half()
    found = _native(native, inputs, log_decay, scale, dy, ds)
    exact = _exact(inputs, log_decay, scale, dy, ds)
    sizes = _exact([x.abs() for x in inputs], log_decay, scale, dy.abs(), ds.abs())
    for i in (1, 5):
        assert _apart(found[i], exact[i]) <= 2.0**-20
    for i in (0, 4):
        assert _rounded_once(found[i], exact[i], sizes[i])


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(2, 700, 4, 2, 64, 64), (1, 300, 2, 2, 128, 96), (2, 64, 2, 2, 32, 16), (1, 200, 2, 1, 33, 7)])
@pytest.mark.parametrize("small", (1e-2, 1e-4, 1e-5))
def test_small_float16_values_keep_their_bits_in_products(native, size, small) -> None:
    """dq and dk of small dy, whose products with v are small, and y and dv of small k:
    one rounding."""

    for which in ("dy", "k"):
        inputs, log_decay, dy, ds = _tensors(size, torch.float16)
        scale = size[4] ** -0.5
        if which == "dy":
            dy, ds = (dy * small).half(), ds * small
        else:
            inputs[1], inputs[3] = (inputs[1] * small).half(), inputs[3] * small
        found = _native(native, inputs, log_decay, scale, dy, ds)
        exact = _exact(inputs, log_decay, scale, dy, ds)
        sizes = _exact([x.abs() for x in inputs], log_decay, scale, dy.abs(), ds.abs())
        for i in (0, 2, 3, 4):
            assert _rounded_once(found[i], exact[i], sizes[i]), (which, i)


@pytest.mark.gpu
def test_rows_of_float16_of_different_sizes(native) -> None:
    """A chunk's queries, and their gradients, from 2^-10 to 2^10: each row has a power of
    its own."""

    size = (1, 130, 2, 1, 64, 64)
    inputs, log_decay, dy, ds = _tensors(size, torch.float16)
    rows = (2.0 ** torch.linspace(-10.0, 10.0, 65, device="cuda").round()).repeat(2).view(1, 130, 1, 1)
    inputs[0], dy = (inputs[0] * rows).half(), (dy / rows).half()
    found = _native(native, inputs, log_decay, 0.125, dy, ds)
    exact = _exact(inputs, log_decay, 0.125, dy, ds)
    sizes = _exact([x.abs() for x in inputs], log_decay, 0.125, dy.abs(), ds.abs())
    for i in (0, 2):   # rows of y and dq are each of one size; those of dk and dv are sums over all
        assert _rounded_once(found[i], exact[i], sizes[i])
    for i in (3, 4):
        assert _rounded_once(found[i], exact[i], sizes[i])


@pytest.mark.gpu
@pytest.mark.parametrize("scale", (1.0, 2.0**20, 2.0**-30))
def test_float16_products_past_65504(native, scale) -> None:
    """scale (q . k) of up to 10^12 and of 10^-9, brought back by v: FP32 values."""

    size = (1, 150, 2, 2, 64, 32)
    inputs, log_decay, dy, ds = _tensors(size, torch.float16)
    inputs[0], inputs[1] = (inputs[0] * 100).half(), (inputs[1] * 100).half()
    v = 1e-5 if scale == 1.0 else (2.0**-24 if scale > 1.0 else 100.0)
    inputs[2], inputs[3], dy = (inputs[2] * v).half(), inputs[3] * v, dy * 0
    found = _native(native, inputs, log_decay, scale, dy, ds)
    exact = _exact(inputs, log_decay, scale, dy, ds)
    sizes = _exact([x.abs() for x in inputs], log_decay, scale, dy.abs(), ds.abs())
    past = exact[0].abs() > 65000.0
    assert torch.isfinite(found[0][~past]).all()
    inside = torch.where(past, 0.0, found[0].double()), torch.where(past, 0.0, exact[0])
    assert _rounded_once(*inside, sizes[0])
    assert _apart(found[1], exact[1]) <= 2.0**-20


@pytest.mark.gpu
def test_float16_columns_of_different_sizes(native) -> None:
    """Value features from 2^-10 to 2^13, and states past 65,504 beside small ones: each
    column of S has a power of its own."""

    size = (2, 260, 2, 1, 64, 48)
    inputs, log_decay, dy, ds = _tensors(size, torch.float16)
    columns = 2.0 ** torch.linspace(-10.0, 13.0, 48, device="cuda").round()
    order = torch.randperm(48, generator=torch.Generator().manual_seed(0)).cuda()
    inputs[2], inputs[3] = (inputs[2] * columns[order]).half(), inputs[3] * columns[order] * 2.0**20
    inputs[0] = (inputs[0] * 2.0**-10).half()
    found = _native(native, inputs, log_decay, 0.125, dy, ds)
    exact = _exact(inputs, log_decay, 0.125, dy, ds)
    sizes = _exact([x.abs() for x in inputs], log_decay, 0.125, dy.abs(), ds.abs())
    past = exact[0].abs() > 65000.0
    inside = torch.where(past, 0.0, found[0].double()), torch.where(past, 0.0, exact[0])
    assert _rounded_once(*inside, sizes[0])
    for e in range(48):
        assert _apart(found[1][..., e], exact[1][..., e]) <= 2.0**-20


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_an_infinite_column_of_a_state_leaves_the_others(native, dtype) -> None:
    """States of 10^6, one value feature of them infinite."""

    inputs, log_decay, dy, ds = _tensors((1, 130, 2, 2, 32, 32), dtype)
    inputs[0], inputs[3] = (inputs[0] * 2.0**-8).to(dtype), inputs[3] * 1e6
    wild = [*inputs[:3], inputs[3].clone()]
    wild[3][..., 5] = math.inf
    y, last = native.linear_attention(*wild[:3], log_decay, scale=0.125, initial_state=wild[3], return_state=True)
    expected, after = native.linear_attention(*inputs[:3], log_decay, scale=0.125, initial_state=inputs[3], return_state=True)
    others = torch.arange(32, device="cuda") != 5
    assert torch.equal(y[..., others], expected[..., others]) and torch.equal(last[..., others], after[..., others])
    assert not torch.isfinite(y[..., 5]).any() and torch.isposinf(last[..., 5]).all()
    exact = _exact(inputs, log_decay, 0.125, dy, ds)
    sizes = _exact([x.abs() for x in inputs], log_decay, 0.125, dy.abs(), ds.abs())
    if dtype == torch.float16:
        assert _rounded_once(expected, exact[0], sizes[0])


def _agree(a, b) -> bool:
    """The same values: a chunk's power of two is that of its largest finite exponents,
    which a zero in place of an infinity leaves."""

    return torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("size", [(1, 200, 2, 1, 64, 64), (1, 700, 2, 2, 24, 40), (2, 130, 4, 4, 13, 9), (1, 150, 1, 1, 128, 128)])
@pytest.mark.parametrize("wild", (math.inf, -math.inf, math.nan))
@pytest.mark.parametrize("token", (70, 95, 127))
def test_what_is_not_finite_reaches_no_earlier_token(native, dtype, size, wild, token) -> None:
    """One value of v, q, k or dy: y of the tokens before it, gradients of those behind
    it, and value features beside it, as with a zero in its place."""

    inputs, log_decay, dy, ds = _tensors(size, dtype)
    scale, feature = size[4] ** -0.5, 5
    others = torch.arange(max(size[4:]), device="cuda") != feature
    before, behind = slice(0, token), slice(token + 1, size[1])

    def run(name, value):
        tensors = {"q": inputs[0], "k": inputs[1], "v": inputs[2], "dy": dy}
        tensors = {key: x.detach().clone() for key, x in tensors.items()}
        tensors[name][0, token, 0, feature] = value
        names = ("y", "s", "dq", "dk", "dv", "ds")
        return dict(zip(names, _native(native, [tensors["q"], tensors["k"], tensors["v"], inputs[3]], log_decay, scale,
                                       tensors["dy"], ds)))

    found, plain = run("v", wild), run("v", 0.0)
    assert torch.equal(found["y"][:, before], plain["y"][:, before])
    assert torch.equal(found["y"][..., others[:size[5]]], plain["y"][..., others[:size[5]]])
    assert not torch.isfinite(found["y"][0, token, 0, feature]) and not torch.isfinite(found["s"][0, 0, :, feature]).any()
    assert _agree(found["dq"][:, before], plain["dq"][:, before])
    assert torch.equal(found["dk"][:, behind], plain["dk"][:, behind])
    found, plain = run("dy", wild), run("dy", 0.0)
    assert torch.equal(found["y"], plain["y"]) and torch.equal(found["s"], plain["s"])
    assert torch.equal(found["dv"][:, behind], plain["dv"][:, behind])
    assert torch.equal(found["dv"][..., others[:size[5]]], plain["dv"][..., others[:size[5]]])
    assert not torch.isfinite(found["dv"][0, token, 0, feature])
    assert _agree(found["dk"][:, behind], plain["dk"][:, behind])
    rows = torch.arange(size[1], device="cuda") != token
    assert torch.equal(found["dq"][:, rows], plain["dq"][:, rows])
    found, plain = run("k", wild), run("k", 0.0)
    assert _agree(found["y"][:, before], plain["y"][:, before])
    assert torch.equal(found["dq"][:, before], plain["dq"][:, before])
    assert torch.equal(found["dv"][:, rows], plain["dv"][:, rows])
    found, plain = run("q", wild), run("q", 0.0)
    assert torch.equal(found["y"][:, rows], plain["y"][:, rows])
    assert torch.equal(found["dk"][:, behind], plain["dk"][:, behind])
    assert _agree(found["dv"][:, behind], plain["dv"][:, behind])
