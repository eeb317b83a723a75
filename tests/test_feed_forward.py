"""Gated feed-forward block: value and gradients against FP64 with bounds that
follow each rounding, over tile edges, odd widths, masks and layouts; captured
replays and refusals."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from lsso_amd.ball import GatedFeedForward, block, hip
from lsso_amd.ball import reference as canonical

HALVES = (torch.float16, torch.bfloat16)


def _act(g, kind):
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = torch.special.ndtr(g)
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def _expected(x, weights, dy, kind, dtype, grad_dtype, mask=None):
    """{output: (value, bound)} in FP64.

    The bounds follow the operator's roundings, each at most half a step `e` of
    the type: of h = act(g) u, of the kept u act'(g) and act(g), of dg and du,
    and of the outputs; an FP32 sum of n products is off by at most n 2^-24 times the sum
    of their magnitudes.  Through act and act' an error of g grows by at most
    1.13 and 0.8 (the largest |act'| and |act''| of both activations); their own
    evaluation in FP32 is off by |g| 2^-22 and (1 + |g|) 2^-21: a relative error
    of |g| 2^-24 + 2^-23 in the exponential, which s (1 - s) <= 1 / 4 shrinks, and
    roundings of FP32.  `tiny`: half a step of FP16 below its normal range.  5%
    for the products of two errors."""

    e = torch.finfo(dtype).eps / 2
    out = torch.finfo(grad_dtype).eps / 2
    tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-134
    f = 2.0**-24
    x, dy = (v.double().reshape(-1, v.shape[-1]) for v in (x, dy))
    gate, up, down = (w.to(dtype).double() for w in weights)
    if mask is not None:
        x = torch.where(mask.reshape(-1, 1), x, 0.0)
        dy = torch.where(mask.reshape(-1, 1), dy, 0.0)
    k, hidden, n, rows = x.shape[1], gate.shape[0], down.shape[0], x.shape[0]
    g, u = x @ gate.T, x @ up.T
    eg, eu = k * f * (x.abs() @ gate.abs().T), k * f * (x.abs() @ up.abs().T)
    act, slope = _act(g, kind)
    ea = 1.13 * eg + g.abs() * 2.0**-22
    h = act * u
    eh = ea * u.abs() + act.abs() * eu + e * h.abs() + tiny
    y = h @ down.T
    found = {"y": (y, eh @ down.abs().T + hidden * f * (h.abs() @ down.abs().T) + e * y.abs() + tiny)}
    dh = dy @ down
    edh = n * f * (dy.abs() @ down.abs())
    es = 0.8 * eg + (1 + g.abs()) * 2.0**-21
    factor = u * slope
    ef = eu * slope.abs() + u.abs() * es + e * factor.abs() + tiny
    eb = ea + e * act.abs() + tiny
    dg, du = dh * factor, dh * act
    edg = edh * factor.abs() + dh.abs() * ef + e * dg.abs() + tiny
    edu = edh * act.abs() + dh.abs() * eb + e * du.abs() + tiny
    dx = dg @ gate + du @ up
    found["x"] = (dx, edg @ gate.abs() + edu @ up.abs() + 2 * hidden * f * (dg.abs() @ gate.abs() + du.abs() @ up.abs())
                  + e * dx.abs() + tiny)
    for name, p, ep, q, eq in (("gate", dg, edg, x, None), ("up", du, edu, x, None), ("down", dy, None, h, eh)):
        value = p.T @ q
        bound = rows * f * (p.abs().T @ q.abs()) + out * value.abs() + tiny
        bound = bound + (p.abs().T @ eq if ep is None else ep.T @ q.abs())
        found[name] = (value, bound)
    return {name: (value, 1.05 * bound) for name, (value, bound) in found.items()}


def _inputs(rows, k, hidden, n, dtype, weight_dtype, seed=0):
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, to=dtype):
        return (torch.randn(shape, generator=generator, device="cuda") * std).to(to)

    shape = rows if isinstance(rows, tuple) else (rows,)
    x, dy = normal(*shape, k), normal(*shape, n)
    weights = [normal(hidden, k, std=2 * k**-0.5, to=weight_dtype), normal(hidden, k, std=k**-0.5, to=weight_dtype),
               normal(n, hidden, std=hidden**-0.5, to=weight_dtype)]
    return x, weights, dy


def _verify(got, expected, shape=None):
    for name, value in got.items():
        reference, bound = expected[name]
        error = (value.double().reshape(reference.shape) - reference).abs()
        assert torch.isfinite(value).all(), name
        assert (error <= bound).all(), (name, float((error / bound).max()))


def _run(native, x, weights, dy, kind, mask=None):
    leaves = [v.detach().requires_grad_() for v in (x, *weights)]
    y = native.gated_feed_forward(*leaves, activation=kind, row_mask=mask)
    grads = torch.autograd.grad(y, leaves, dy)
    assert y.is_contiguous() and y.dtype == x.dtype
    for grad, leaf in zip(grads, leaves):
        assert grad.shape == leaf.shape and grad.dtype == leaf.dtype
    return dict(zip(("y", "x", "gate", "up", "down"), (y.detach(), *grads)))


def _check(native, rows, k, hidden, n, dtype, kind="silu", weight_dtype=None, mask=None, seed=0):
    weight_dtype = dtype if weight_dtype is None else weight_dtype
    x, weights, dy = _inputs(rows, k, hidden, n, dtype, weight_dtype, seed)
    got = _run(native, x, weights, dy, kind, mask)
    _verify(got, _expected(x, weights, dy, kind, dtype, weight_dtype, mask))
    with torch.no_grad():
        assert torch.equal(native.gated_feed_forward(x, *weights, activation=kind, row_mask=mask), got["y"])
    again = _run(native, x, weights, dy, kind, mask)
    assert all(torch.equal(got[name], again[name]) for name in got)
    return got


def test_formula_against_differences() -> None:
    """The bound's own formulas: gradients by central differences in FP64."""

    torch.manual_seed(0)
    x, dy = torch.randn(3, 4).double(), torch.randn(3, 2).double()
    weights = [torch.randn(5, 4).double(), torch.randn(5, 4).double(), torch.randn(2, 5).double()]
    for kind in ("silu", "gelu"):
        value = lambda: _expected(x, weights, dy, kind, torch.float64, torch.float64)  # noqa: E731
        found = value()
        for name, leaf in zip(("x", "gate", "up", "down"), (x, *weights)):
            flat = leaf.reshape(-1)
            for i in range(flat.numel()):
                at, step = float(flat[i]), 1e-5
                ends = []
                for to in (at + step, at - step):
                    flat[i] = to
                    ends.append(float((value()["y"][0] * dy).sum()))
                flat[i] = at
                assert abs((ends[0] - ends[1]) / (2 * step) - float(found[name][0].reshape(-1)[i])) < 1e-7


def test_module_on_the_cpu() -> None:
    layer = GatedFeedForward(6, 10, activation="gelu").double()
    x = torch.randn(2, 3, 6, dtype=torch.float64, requires_grad=True)
    mask = torch.tensor([[True, False, True], [False, False, False]])
    y = layer(x, mask)
    y.sum().backward()
    expected = _expected(x.detach(), [layer.gate.weight.detach(), layer.up.weight.detach(), layer.down.weight.detach()],
                         torch.ones(2, 3, 6, dtype=torch.float64), "gelu", torch.float64, torch.float64, mask)
    for name, value in (("y", y), ("x", x.grad), ("gate", layer.gate.weight.grad), ("down", layer.down.weight.grad)):
        torch.testing.assert_close(value.detach().reshape(expected[name][0].shape), expected[name][0])
    assert not y[1].any() and not x.grad[1].any()
    for wrong in ({"hidden": 0}, {"activation": "relu"}):
        with pytest.raises(ValueError):
            GatedFeedForward(**{"dim": 4, "hidden": 4, **wrong})
    with pytest.raises(ValueError):
        layer(x, implementation="other")


@pytest.mark.parametrize("kind", ("silu", "gelu"))
def test_reference_masked_rows_may_hold_anything(kind) -> None:
    torch.manual_seed(1)
    leaves = [torch.randn(shape).double().requires_grad_() for shape in ((2, 3, 4), (5, 4), (5, 4), (6, 5))]
    mask = torch.tensor([[True, False, True], [False, False, True]])
    dy = torch.randn(2, 3, 6).double()

    def run():
        y = canonical.gated_feed_forward(*leaves, activation=kind, row_mask=mask)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    plain = run()
    with torch.no_grad():
        leaves[0][~mask], dy[~mask] = math.nan, math.inf
    for a, b in zip(run(), plain):
        assert torch.equal(a, b)
    assert not plain[0][~mask].any() and not plain[1][~mask].any()


def _shape(rows=4, k=16, hidden=24, n=16, stride=16, dtype=2, weight=2, activation=1):
    return block.FeedForwardShape(rows, k, hidden, n, stride, dtype, weight, activation)


def test_refusals_on_the_cpu() -> None:
    library = hip.open_library()
    size, other = ctypes.c_size_t(), ctypes.c_size_t()

    def forward(shape=_shape(), x=16, gate=16, up=16, down=16, gates=None, product=None, y=16, workspace=256,
                room=1 << 20):
        return library.lsso_hip_feed_forward(ctypes.byref(shape), x, gate, up, down, None, gates, product, y, workspace,
                                             room, None)

    def backward(shape=_shape(), dy=16, stride=16, x=16, down=16, gates=16, product=16, grad_gate=16, workspace=256,
                 room=1 << 20):
        return library.lsso_hip_feed_forward_backward(ctypes.byref(shape), dy, stride, x, 16, 16, down, None, gates,
                                                      product, None, grad_gate, None, None, workspace, room, None)

    wrong_shapes = [_shape(rows=-1), _shape(k=0, stride=0), _shape(hidden=0), _shape(n=0), _shape(stride=15),
                    _shape(dtype=3), _shape(weight=1), _shape(activation=0), _shape(activation=3),
                    _shape(rows=2**31), _shape(hidden=2**20 + 1)]
    for shape in wrong_shapes:
        assert library.lsso_hip_feed_forward_workspace_bytes(ctypes.byref(shape), 0, ctypes.byref(size)) < 0
        assert library.lsso_hip_feed_forward_kept(ctypes.byref(shape), ctypes.byref(size), ctypes.byref(other)) < 0
        assert forward(shape=shape) < 0 and backward(shape=shape) < 0
    assert forward(shape=_shape(rows=0), x=None, y=None, workspace=None, room=0) == 0
    for wrong in ({"x": None}, {"gate": None}, {"down": None}, {"y": None}, {"x": 24}, {"up": 24}, {"gates": 16},
                  {"product": 16}, {"gates": 24, "product": 16}, {"workspace": None}, {"workspace": 128}, {"room": 16}):
        assert forward(**wrong) < 0, wrong
    for wrong in ({"dy": None}, {"dy": 24}, {"stride": 15}, {"x": None}, {"down": 24}, {"gates": None},
                  {"product": None}, {"workspace": None}, {"workspace": 128}, {"room": 16}):
        assert backward(**wrong) < 0, wrong
    shape = _shape(hidden=25)
    assert library.lsso_hip_feed_forward_kept(ctypes.byref(shape), ctypes.byref(size), ctypes.byref(other)) == 0
    assert (size.value, other.value) == (2 * 4 * 32, 4 * 32)
    for mask in (-1, 8):
        assert library.lsso_hip_feed_forward_backward_workspace_bytes(ctypes.byref(shape), 16, mask,
                                                                      ctypes.byref(size)) < 0
    assert library.lsso_hip_feed_forward_backward_workspace_bytes(ctypes.byref(shape), 15, 7, ctypes.byref(size)) < 0


def test_workspaces_hold_every_size() -> None:
    library = hip.open_library()
    size = ctypes.c_size_t()
    for rows in (0, 1, 63, 64, 513, 4104, 131072, 2**31 - 1):
        for k, hidden, n in ((1, 1, 1), (8, 8, 8), (300, 801, 300), (768, 2048, 768), (4096, 16384, 4096)):
            for weight in (2, 3):
                shape = _shape(rows, k, hidden, n, k, weight=weight)
                for training in (0, 1):
                    assert library.lsso_hip_feed_forward_workspace_bytes(
                        ctypes.byref(shape), training, ctypes.byref(size)) == 0
                    copies = (k % 8 != 0) * 2 * rows * ((k + 7) // 8 * 8)
                    assert size.value >= copies + (0 if training else 2 * rows * hidden)
                assert library.lsso_hip_feed_forward_backward_workspace_bytes(
                    ctypes.byref(shape), n, 7, ctypes.byref(size)) == 0
                assert size.value >= 4 * rows * hidden


def test_kept_factors_on_the_cpu() -> None:
    library = hip.open_library()
    gates, product = ctypes.c_size_t(), ctypes.c_size_t()
    for rows, hidden, pitch, wide in ((4, 25, 32, 32), (3, 32, 32, 32), (7, 33, 40, 64), (1, 801, 808, 832)):
        for code, dtype in ((1, torch.float16), (2, torch.bfloat16)):
            for fine in (0, 1):
                shape = block.FeedForwardShape(rows, 16, hidden, 16, 16, code, code, 1, fine)
                assert library.lsso_hip_feed_forward_kept(
                    ctypes.byref(shape), ctypes.byref(gates), ctypes.byref(product)) == 0
                # 16-bit values: two factors, and a byte or two more of both per column, by 32 columns
                assert gates.value == rows * (2 * pitch + fine * wide // code)
                assert product.value == rows * pitch
                assert block._feed_forward_kept(rows, hidden, dtype, bool(fine)) == (gates.value, pitch)
    for fine in (-1, 2, 24):
        shape = block.FeedForwardShape(4, 16, 24, 16, 16, 2, 2, 1, fine)
        assert library.lsso_hip_feed_forward_kept(ctypes.byref(shape), ctypes.byref(gates), ctypes.byref(product)) < 0


def test_workspaces_hold_every_buffer() -> None:
    """The sum of all that a call keeps beside each other: copies of operands with
    odd rows or of float32, h (its second part of few rows), dg and du, both
    transposes, the weight gradients' partials, and at least two splits' partials
    of a small product with a long K."""

    library = hip.open_library()
    size = ctypes.c_size_t()

    def whole(n):
        return (n + 7) // 8 * 8

    def split(rows, columns, k):   # 64 x 64 tiles for half the 256 CUs or fewer, 8 stages of 64 k or more
        tiles = -(-rows // 64) * -(-columns // 64)
        return 4 * 2 * rows * whole(columns) if rows > 32 and tiles <= 128 and k >= 512 else 0

    for rows in (1, 32, 33, 64, 513, 4104, 131072):
        for k, hidden, n in ((1, 1, 1), (8, 8, 8), (300, 801, 300), (64, 4096, 72), (4096, 64, 4096), (768, 2048, 768)):
            for weight in (2, 3):
                shape = _shape(rows, k, hidden, n, k, weight=weight)
                x = 2 * rows * whole(k) * (k % 8 != 0)
                weights = 2 * (2 * hidden * whole(k) * (weight == 3 or k % 8 != 0)
                               + n * whole(hidden) * (weight == 3 or hidden % 8 != 0))
                h = 2 * rows * whole(hidden)
                for training in (0, 1):
                    assert library.lsso_hip_feed_forward_workspace_bytes(
                        ctypes.byref(shape), training, ctypes.byref(size)) == 0
                    assert size.value >= (x + weights + (0 if training else h) + (h if rows <= 32 else 0)
                                          + split(rows, n, hidden)), (rows, k, hidden, n, weight, training)
                partials = 4 * (2 * hidden * whole(k) + n * whole(hidden))
                transposes = 2 * (2 * k * whole(hidden) + hidden * whole(n))
                assert library.lsso_hip_feed_forward_backward_workspace_bytes(
                    ctypes.byref(shape), n, 7, ctypes.byref(size)) == 0
                assert size.value >= (x + 2 * rows * whole(n) * (n % 8 != 0) + 2 * h + partials + transposes
                                      + split(rows, k, 2 * hidden)), (rows, k, hidden, n, weight)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kind", ("silu", "gelu"))
@pytest.mark.parametrize("rows", (1, 2, 17, 33, 64, 65, 200))
def test_rows(native, dtype, kind, rows) -> None:
    _check(native, rows, 64, 136, 48, dtype, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("widths", [(8, 8, 8), (1, 1, 1), (7, 9, 3), (16, 24, 40), (33, 65, 31), (100, 266, 100),
                                    (300, 801, 300), (64, 70, 521), (521, 64, 72), (256, 688, 256), (40, 1000, 24)])
@pytest.mark.parametrize("dtype", HALVES)
def test_widths(native, widths, dtype) -> None:
    _check(native, 70, *widths, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("widths", [(64, 136, 48), (33, 65, 31)])
@pytest.mark.parametrize("dtype", HALVES)
def test_float32_weights(native, widths, dtype) -> None:
    _check(native, 150, *widths, dtype, weight_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,hidden,n", [(1576, 192, 512, 192), (4104, 300, 801, 300), (3000, 640, 256, 1040),
                                             (20000, 64, 2112, 64), (40000, 72, 520, 264), (66000, 32, 64, 264)])
def test_large_tiles_and_row_ranges(native, rows, k, hidden, n) -> None:
    _check(native, rows, k, hidden, n, torch.bfloat16, "gelu")


def _step(native, x, weights, dy, kind, fine, mask=None):
    leaves = [v.detach().requires_grad_() for v in (x, *weights)]
    y = native.gated_feed_forward(*leaves, activation=kind, row_mask=mask, fine_factors=fine)
    return dict(zip(("y", "x", "gate", "up", "down"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,k,hidden,n", [(1, 64, 136, 48), (17, 33, 65, 31), (32, 96, 1000, 24), (33, 64, 136, 48),
                                             (70, 7, 9, 3), (200, 300, 801, 300), (4104, 128, 264, 128),
                                             (8000, 72, 2048, 520), (12000, 64, 264, 64)])
def test_rounded_factors(native, rows, k, hidden, n, dtype) -> None:
    """The same value and, to the roundings of the factors, gradients."""

    x, weights, dy = _inputs(rows, k, hidden, n, dtype, dtype)
    mask = torch.rand(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) < 0.8
    got = _step(native, x, weights, dy, "gelu", False, mask)
    _verify(got, _expected(x, weights, dy, "gelu", dtype, dtype, mask))
    wide = _step(native, x, weights, dy, "gelu", True, mask)
    assert torch.equal(got["y"], wide["y"]) and torch.equal(got["down"], wide["down"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("kind", ("silu", "gelu"))
@pytest.mark.parametrize("rows,hidden", [(16, 40), (32, 33), (48, 136), (130, 801), (4100, 264), (9000, 520)])
def test_fine_factors(native, dtype, kind, rows, hidden) -> None:
    """dg and du of single products: x has at most one 1 in a row or a column, so
    that dWu is act(g) dh of that row.  Then the factor's rounding (half a step of 12
    bits, 2^-12, for bfloat16 and of 16, 2^-16, for float16), dg's or du's and the
    output's are all that there is, beside act's and act''s own |g| 2^-22 and (1 + |g|)
    2^-21.  The second rounding of a value of the type changes nothing."""

    size = min(rows, 520)
    generator = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.zeros(rows, size, device="cuda", dtype=dtype)
    chosen = torch.randperm(rows, device="cuda", generator=generator)[:size]
    x[chosen, torch.arange(size, device="cuda")] = 1
    gate, up = (torch.randn(hidden, size, device="cuda", generator=generator).to(dtype) for _ in range(2))
    down = torch.randn(1, hidden, device="cuda", generator=generator).to(dtype)
    dy = torch.ones(rows, 1, device="cuda", dtype=dtype)
    got = _step(native, x, (gate, up, down), dy, kind, True)
    g, u, dh = gate.double(), up.double(), down.double().t()
    act, slope = _act(g, kind)
    e, f = torch.finfo(dtype).eps / 2, 2.0**-16 if dtype == torch.float16 else 2.0**-12
    tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-134
    for name, value, error in (("up", act * dh, g.abs() * 2.0**-22 * dh.abs()),
                               ("gate", u * slope * dh, (1 + g.abs()) * 2.0**-21 * (u * dh).abs())):
        bound = (e + f) * value.abs() + error + tiny
        assert ((got[name].double() - value).abs() <= 1.02 * bound).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("rows", (16, 48))
def test_factors_past_the_range_of_float16(native, rows) -> None:
    """u act'(g) of 95,000 times 0.74: kept of 24 bits, with FP32's range."""

    x = torch.eye(16, device="cuda").half().repeat(rows // 16, 1) * 200
    gate, up = (torch.eye(16, device="cuda") * value for value in (0.0025, 475.0))
    down, dy = torch.eye(16, device="cuda"), torch.full((rows, 16), 2.0**-10, device="cuda").half()
    got = _step(native, x, [w.half() for w in (gate, up, down)], dy, "silu", True)
    g, u = 200 * gate.half().double(), 95000.0
    value = _act(g, "silu")[1] * u * 2.0**-10 * 200 * (rows // 16)
    found = torch.diagonal(got["gate"]).double()
    assert ((found - torch.diagonal(value)).abs() <= 2.0**-9 * torch.diagonal(value)).all()
    assert not torch.isfinite(_step(native, x, [w.half() for w in (gate, up, down)], dy, "silu", False)["gate"]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,k,hidden,n", [(8000, 72, 2048, 520), (8000, 520, 2041, 72), (22000, 512, 72, 520),
                                             (4200, 200, 1032, 776), (2100, 200, 1032, 776)])
def test_tiles_of_every_size(native, rows, k, hidden, n, dtype) -> None:
    """Products of each kernel whose tiles go round the device once and twice, in
    each of the three sizes, the last ones partly outside."""

    _check(native, rows, k, hidden, n, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,hidden,n", [((3, 70), 64, 136, 48), ((2, 33), 33, 65, 31), ((8, 513), 128, 256, 128),
                                             ((16, 2500), 64, 264, 136)])
def test_masked_rows_may_hold_anything(native, rows, k, hidden, n) -> None:
    dtype = torch.bfloat16
    mask = torch.rand(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.7
    mask[-1] = False
    x, weights, dy = _inputs(rows, k, hidden, n, dtype, dtype)
    expected = _expected(x, weights, dy, "silu", dtype, dtype, mask)
    x[~mask], dy[~mask] = math.nan, math.inf
    got = _run(native, x, weights, dy, "silu", mask)
    _verify(got, expected)
    assert not got["y"][~mask].any() and not got["x"][~mask].any()
    nothing = _run(native, x, weights, dy, "silu", torch.zeros_like(mask))
    assert not any(value.any() for value in nothing.values())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", (1, 15, 16, 18, 31, 32, 33))
@pytest.mark.parametrize("widths", [(64, 136, 48), (33, 65, 31), (768, 520, 1000)])
@pytest.mark.parametrize("weight_dtype", (torch.bfloat16, torch.float32))
def test_few_masked_rows(native, rows, widths, weight_dtype) -> None:
    mask = torch.ones(rows, dtype=torch.bool, device="cuda")
    mask[rows // 2::3] = False   # of a single row, that row
    _check(native, (rows,), *widths, torch.bfloat16, "gelu", weight_dtype=weight_dtype, mask=mask, seed=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows", (1, 17, 32))
def test_few_rows_are_rounded_once(native, dtype, rows) -> None:
    """Up to 32 rows carry h as two 16-bit values: half a step of what the first
    rounding left, e^2 of h (FP16: or half a step below the normal range), stands
    in the place of e."""

    x, weights, _ = _inputs(rows, 96, 264, 80, dtype, dtype)
    y = native.gated_feed_forward(x, *weights)
    e, f = torch.finfo(dtype).eps / 2, 2.0**-24
    tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-134
    xs, (gate, up, down) = x.double(), (w.double() for w in weights)
    g, u = xs @ gate.T, xs @ up.T
    h = _act(g, "silu")[0] * u
    eg, eu = 96 * f * (xs.abs() @ gate.abs().T), 96 * f * (xs.abs() @ up.abs().T)
    act = _act(g, "silu")[0].abs()
    eh = (1.13 * eg + g.abs() * 2.0**-22) * u.abs() + act * eu + (e * e + f) * h.abs() + tiny
    exact = h @ down.T
    # Twice the products: each part's are summed.
    bound = eh @ down.abs().T + 2 * 264 * f * (h.abs() @ down.abs().T) + e * exact.abs() + tiny
    assert ((y.double() - exact).abs() <= 1.05 * bound).all()


@pytest.mark.gpu
def test_offsets_past_32_bits(native) -> None:
    """The last rows of h and its factors lie past 2^31 elements: they meet the
    bounds of those rows alone."""

    rows, k, hidden, n, tail = (1 << 20) + 300, 16, 2048, 8, 300
    x, weights, dy = _inputs(rows, k, hidden, n, torch.bfloat16, torch.bfloat16)
    mask = torch.ones(rows, dtype=torch.bool, device="cuda")
    mask[:-tail] = False   # the weights' gradients come from the tail alone
    whole = _run(native, x, weights, dy, "silu", mask)
    expected = _expected(x[-tail:], weights, dy[-tail:], "silu", torch.bfloat16, torch.bfloat16)
    _verify({name: value[-tail:] if name in ("y", "x") else value for name, value in whole.items()}, expected)
    assert not whole["y"][:-tail].any() and not whole["x"][:-tail].any()


@pytest.mark.gpu
def test_rows_past_one_grid_of_copies(native) -> None:
    """2^30 rows of one feature, copied into whole pieces by more workgroups than
    fit a launch's x; all but the last rows are zeros."""

    rows, tail = (1 << 30) + 77, 300
    x, weights, dy = _inputs(tail, 1, 1, 1, torch.bfloat16, torch.bfloat16)
    long_x, long_dy = (torch.zeros(rows, 1, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    long_x[-tail:], long_dy[-tail:] = x, dy
    got = _run(native, long_x, weights, long_dy, "silu")
    _verify({name: value[-tail:] if name in ("y", "x") else value for name, value in got.items()},
            _expected(x, weights, dy, "silu", torch.bfloat16, torch.bfloat16))
    assert not got["y"][:-tail].any() and not got["x"][:-tail].any()


@pytest.mark.gpu
def test_masked_rows_equal_the_rows_alone(native) -> None:
    x, weights, _ = _inputs((4, 100), 96, 264, 96, torch.float16, torch.float16)
    mask = torch.zeros(4, 100, dtype=torch.bool, device="cuda")
    mask[:, :37] = True
    y = native.gated_feed_forward(x, *weights, row_mask=mask)
    assert torch.equal(y[mask], native.gated_feed_forward(x, *weights)[mask])


@pytest.mark.gpu
def test_layouts(native) -> None:
    x, weights, dy = _inputs((5, 30), 64, 72, 40, torch.bfloat16, torch.bfloat16)
    plain = _run(native, x, weights, dy, "silu")
    wide = torch.full((5, 30, 70), math.nan, device="cuda", dtype=torch.bfloat16)
    for first, stop in ((0, 64), (3, 67)):   # rows of 140 bytes; an odd base
        view = wide[..., first:stop]
        view.copy_(x)
        spread = torch.full((5, 30, 48), math.nan, device="cuda", dtype=torch.bfloat16)[..., 5:45]
        spread.copy_(dy)
        moved = [w.t().contiguous().t() for w in weights]
        got = _run(native, view, moved, spread, "silu")
        assert all(torch.equal(got[name], plain[name]) for name in plain)
    padded = torch.full((5, 30, 80), math.nan, device="cuda", dtype=torch.bfloat16)
    padded[..., :64] = x   # whole pieces, read in place; NaN behind each row
    got = _run(native, padded[..., :64], weights, dy, "silu")
    assert all(torch.equal(got[name], plain[name]) for name in plain)
    got = _run(native, x.transpose(0, 1).contiguous().transpose(0, 1), weights, dy, "silu")
    assert all(torch.equal(got[name], plain[name]) for name in plain)
    leaves = [v.detach().requires_grad_() for v in (x, *weights)]
    ones = torch.autograd.grad(native.gated_feed_forward(*leaves).sum(), leaves)   # stride-0 gradient
    expected = torch.autograd.grad(native.gated_feed_forward(*leaves), leaves, torch.ones_like(dy))
    assert all(torch.equal(a, b) for a, b in zip(ones, expected))


@pytest.mark.gpu
def test_gradients_asked_for_one_by_one(native) -> None:
    x, weights, dy = _inputs(130, 64, 136, 48, torch.bfloat16, torch.bfloat16)
    whole = _run(native, x, weights, dy, "gelu")
    for name, wanted in (("x", 0), ("gate", 1), ("up", 2), ("down", 3)):
        values = [v.detach() for v in (x, *weights)]
        values[wanted].requires_grad_()
        y = native.gated_feed_forward(*values, activation="gelu")
        (grad,) = torch.autograd.grad(y, values[wanted], dy)
        assert torch.equal(grad, whole[name]), name


@pytest.mark.gpu
def test_empty_batches_and_vectors(native) -> None:
    x, weights, dy = _inputs((0, 5), 16, 24, 8, torch.float16, torch.float16)
    got = _run(native, x, weights, dy, "silu")
    assert got["y"].shape == (0, 5, 8) and not any(got[name].any() for name in ("gate", "up", "down"))
    x, weights, dy = _inputs((), 16, 24, 8, torch.float16, torch.float16)
    _verify(_run(native, x, weights, dy, "silu"), _expected(x[None], weights, dy[None], "silu", torch.float16, torch.float16))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ("silu", "gelu"))
def test_saturated_gates(native, kind) -> None:
    """Gates of +-1 to +-3e4 in both types: no NaN from an exponential's range."""

    for dtype in HALVES:
        x = torch.eye(16, device="cuda", dtype=dtype)
        gates = torch.logspace(0, 4.4, 16, device="cuda")
        gate = torch.diag(torch.where(torch.arange(16, device="cuda") % 2 == 0, gates, -gates)).to(dtype)
        up = torch.eye(16, device="cuda", dtype=dtype)
        down = torch.eye(16, device="cuda", dtype=dtype)
        dy = torch.ones(16, 16, device="cuda", dtype=dtype)
        got = _run(native, x, [gate, up, down], dy, kind)
        value, slope = _act(torch.diagonal(gate).double(), kind)
        limit = torch.finfo(dtype).eps * value.abs() * 2 + gates.double() * 2.0**-22 + 2.0**-24
        assert ((torch.diagonal(got["y"]).double() - value).abs() <= limit).all()
        limit = torch.finfo(dtype).eps * slope.abs() * 2 + (1 + gates.double()) * 2.0**-21 + 2.0**-24
        assert ((torch.diagonal(got["gate"]).double() - slope).abs() <= limit).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ("silu", "gelu"))
@pytest.mark.parametrize("rows", (16, 32, 48))
def test_products_past_the_range_are_infinite(native, kind, rows) -> None:
    """h of 200 times +-400, past FP16's 65,504: an infinite y with h's sign, of a
    few rows as of many.  (Its row's other columns are infinity times 0: NaN.)"""

    x = torch.eye(16, device="cuda", dtype=torch.float16).repeat(rows // 16, 1)
    sign = torch.where(torch.arange(16, device="cuda") % 2 == 0, 1.0, -1.0)
    gate, up = torch.eye(16, device="cuda") * 200, torch.diag(400 * sign)
    y = native.gated_feed_forward(x, gate.half(), up.half(), torch.eye(16, device="cuda").half(), activation=kind)
    assert torch.equal(torch.diagonal(y[-16:]), (sign * math.inf).half())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ("silu", "gelu"))
@pytest.mark.parametrize("rows", (16, 48))
def test_infinite_gates(native, kind, rows) -> None:
    """Gates whose FP32 sums overflow: act(inf) u is infinite, and act(-inf) =
    -inf * 0 is NaN, as the formulas are in FP64."""

    x = torch.eye(16, device="cuda", dtype=torch.bfloat16).repeat(rows // 16, 1) * 1e38
    sign = torch.where(torch.arange(16, device="cuda") % 2 == 0, 1.0, -1.0)
    gate, up = torch.diag(16 * sign).bfloat16(), (torch.eye(16, device="cuda") * 1e-37).bfloat16()
    y = native.gated_feed_forward(x, gate, up, torch.eye(16, device="cuda").bfloat16(), activation=kind)
    found, expected = torch.diagonal(y[-16:]), _act(sign.double() * math.inf, kind)[0].bfloat16()
    assert torch.equal(found.isnan(), expected.isnan())
    assert torch.equal(found[::2], expected[::2]) and expected[0] == math.inf


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ("silu", "gelu"))
@pytest.mark.parametrize("rows", (32, 96))
@pytest.mark.parametrize("dtype,lowest,scale", [(torch.float16, -6.0, 6e4), (torch.bfloat16, -12.0, 1.0)])
def test_negative_gates_to_a_relative_error(native, kind, rows, dtype, lowest, scale) -> None:
    """y = act(g) u of single gates down to where a 16-bit h is still normal, to
    one rounding of the value itself: act's own FP32 steps are off by the rounded
    argument of the exponential (three roundings of at most 104 in powers of two:
    2^-15.9 of it), the fit (2^-19) and a few roundings of 2^-23: less than 2^-15.
    In bfloat16 the kept factors round once more, and the sum of equal rows once."""

    x = torch.eye(32, device="cuda", dtype=dtype).repeat(rows // 32, 1)
    g = torch.linspace(-3.0, lowest, 32, device="cuda").to(dtype)
    weights = [torch.diag(g), torch.eye(32, device="cuda", dtype=dtype) * scale, torch.eye(32, device="cuda", dtype=dtype)]
    got = _run(native, x, weights, torch.ones_like(x), kind)
    act, slope = _act(g.double(), kind)
    if kind == "gelu":   # ndtr takes the tail from 1 - erf, which is 0 from -8.3 on
        cdf = torch.special.erfc(-g.double() * math.sqrt(0.5)) / 2
        act, slope = g.double() * cdf, cdf + g.double() * torch.exp(-0.5 * g.double() ** 2) / math.sqrt(2 * math.pi)
    e, fine = torch.finfo(dtype).eps / 2, 2.0**-15
    u = torch.diagonal(weights[1]).double()
    found = torch.diagonal(got["y"][-32:]).double()
    # h, and of more than a few rows nothing else: the second product is by 1.
    assert ((found - act * u).abs() <= (e + fine) * 1.01 * (act * u).abs()).all()
    if dtype == torch.bfloat16:
        for name, value in (("up", act), ("gate", slope)):
            found = torch.diagonal(got[name]).double() / (rows // 32)
            assert ((found - value).abs() <= (2 * e + 2 * fine) * 1.01 * value.abs()).all(), name


@pytest.mark.gpu
def test_captured_training_step(native) -> None:
    x, weights, dy = _inputs((4, 65), 64, 136, 64, torch.bfloat16, torch.bfloat16)
    x.requires_grad_()
    for w in weights:
        w.requires_grad_()
    mask = torch.ones(4, 65, dtype=torch.bool, device="cuda")
    mask[1, 40:] = False

    def step():
        y = native.gated_feed_forward(x, *weights, row_mask=mask)
        return (y.detach(), *torch.autograd.grad(y, (x, *weights), dy))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        with torch.no_grad():
            x.normal_()
            dy.normal_()
            mask[2, torch.randint(0, 65, (20,), device="cuda")] = False
        graph.replay()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_streams_at_once(native) -> None:
    cases = [_inputs(300, 64, 520, 64, torch.bfloat16, torch.bfloat16, seed) for seed in (1, 2)]
    expected = [_run(native, *case, "silu") for case in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    found = [None, None]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                found[i] = _run(native, *cases[i], "silu")
    torch.cuda.synchronize()
    for a, b in zip(found, expected):
        assert all(torch.equal(a[name], b[name]) for name in b)


@pytest.mark.gpu
def test_refusals(native) -> None:
    x, weights, _ = _inputs(4, 16, 24, 8, torch.float16, torch.float16)
    gate, up, down = weights
    for arguments, options, error in (
        ((x.cpu(), gate, up, down), {}, RuntimeError), ((x, gate.cpu(), up, down), {}, RuntimeError),
        ((x.float(), gate, up, down), {}, TypeError), ((x, gate.float(), up, down), {}, TypeError),
        ((x, gate.bfloat16(), up.bfloat16(), down.bfloat16()), {}, TypeError),
        ((x, gate, up[:8], down), {}, ValueError), ((x, gate, up, down[:, :8]), {}, ValueError),
        ((x[:, :8], gate, up, down), {}, ValueError), ((x, gate[0], up, down), {}, ValueError),
        ((x, gate, up, down), {"activation": "relu"}, ValueError),
        ((x, gate, up, down), {"row_mask": torch.ones(3, dtype=torch.bool, device="cuda")}, ValueError),
        ((x, gate, up, down), {"row_mask": torch.ones(4, dtype=torch.bool)}, RuntimeError),
        ((x, gate, up, down[:0]), {}, ValueError),
    ):
        with pytest.raises(error):
            native.gated_feed_forward(*arguments, **options)
