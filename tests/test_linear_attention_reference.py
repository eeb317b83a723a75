"""The reference path of linear attention where values are not finite."""

from __future__ import annotations

import math

import pytest
import torch

from lsso_amd.ball import reference as canonical
from test_linear_attention import _inputs


@pytest.mark.parametrize("wild", (math.inf, -math.inf, math.nan))
@pytest.mark.parametrize("length,token", ((9, 4), (70, 65), (200, 70), (200, 127)))
def test_what_is_not_finite_reaches_no_earlier_token(wild, length, token) -> None:
    """One value of v, q, k or dy: y of the tokens before it and gradients of those
    behind it, as with a zero in its place."""

    q, k, v, log_decay, generator = _inputs(2, length, 2, 1, 6, 5, torch.float64)
    tensors = {"q": q, "k": k, "v": v, "dy": torch.randn(2, length, 2, 5, generator=generator, dtype=torch.float64)}
    before, behind = slice(0, token), slice(token + 1, length)

    def run(name, value):
        given = {key: x.clone() for key, x in tensors.items()}
        given[name][0, token, 0, 3] = value
        leaves = [given[key].requires_grad_() for key in ("q", "k", "v")]
        y = canonical.linear_attention(*leaves, log_decay)
        return dict(zip(("y", "dq", "dk", "dv"), (y.detach(), *torch.autograd.grad(y, leaves, given["dy"]))))

    for name, front, back in (("v", ("y", "dq"), ("dk", "dv")), ("dy", ("y", "dq"), ("dk", "dv")),
                              ("k", ("y", "dq"), ("dk", "dv")), ("q", ("y", "dq"), ("dk", "dv"))):
        found, plain = run(name, wild), run(name, 0.0)
        for key in front:
            assert torch.equal(found[key][:, before], plain[key][:, before]), (name, key)
        for key in back:
            assert torch.equal(found[key][:, behind], plain[key][:, behind]), (name, key)
        assert torch.equal(found["y"][1], plain["y"][1])
    assert not torch.isfinite(run("v", wild)["y"][0, token, 0, 3])
