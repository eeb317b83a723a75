"""Operators of a causal token mixer, each with its gradients or its form for
single tokens: rotary positions, linear attention with a decay for each head,
and group norm with an activation, channels last.

A case is a dict of plain values.  ``op`` names the operator:

rotary  the first ``rotary`` of ``dim`` features of each head of a query and a
        key turned by position times frequency, in pairs of neighbours
        ("interleaved") or of a feature and the one half the rotated part
        further ("half"); with ``train`` the gradients of both for given ones
        of the outputs.  ``factor`` > 1 scales the frequencies for contexts
        longer than ``original``.
attend  y_t = scale * q_t S_t with S_t = exp(log_decay_h) S_{t-1} + k_t (x) v_t.
        Tokens that ``mask`` excludes leave S as it is; their y is zero.
        ``shared`` query heads read one key and value head.  ``state``: S_0 is
        given and the last S returned; with ``train`` the gradients of q, k, v
        and of S_0.
step    one token of ``attend`` for each sequence, its state updated in place.
norm    y = act((x - mean) / sqrt(var + eps) * weight + bias) over the tokens
        and the channels of each group of a sample; ``tokens`` makes each token
        a sample of its own; ``mask`` leaves tokens out.  With ``train`` the
        gradients of x, weight and bias.
"""

from __future__ import annotations

import functools
import math

import torch

own = False

_CHUNK = 64
_EPS = 1e-5
_BASE = 10000.0
# Turns over the original context between which a feature goes from fully
# scaled to unscaled.
_FEW_TURNS, _MANY_TURNS = 1.0, 32.0


def _rotary(name, batch, length, heads, kv_heads, dim, rotary, layout, dtype, train, positions, start, factor=1.0):
    return {"name": name, "op": "rotary", "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rotary": rotary, "layout": layout, "dtype": dtype, "train": train, "positions": positions,
            "start": start, "factor": factor, "original": 4096}


def _attend(name, batch, length, heads, shared, dim, value_dim, dtype, train, mask=False, state=False):
    return {"name": name, "op": "attend", "batch": batch, "length": length, "heads": heads, "shared": shared,
            "dim": dim, "value_dim": value_dim, "dtype": dtype, "train": train, "mask": mask, "state": state}


def _step(name, batch, heads, shared, dim, value_dim, dtype, mask=False):
    return {"name": name, "op": "step", "batch": batch, "length": 1, "heads": heads, "shared": shared, "dim": dim,
            "value_dim": value_dim, "dtype": dtype, "train": False, "mask": mask, "state": True}


def _norm(name, batch, length, channels, groups, dtype, train, activation, tokens=False, mask=False):
    return {"name": name, "op": "norm", "batch": batch, "length": length, "channels": channels, "groups": groups,
            "dtype": dtype, "train": train, "activation": activation, "tokens": tokens, "mask": mask}


def listed():
    return [
        # One new token of each of 32 sequences, far into its context.
        _rotary("rotary_step", 32, 1, 12, 4, 64, 64, "half", "bfloat16", False, "int64", 100000),
        # A long prompt whose context was extended eightfold, half of each head turned.
        _rotary("rotary_long_half", 1, 32768, 12, 4, 128, 64, "half", "float16", False, "int64", 0, factor=8.0),
        # Queries and keys of the published shell's batch in training.
        _rotary("rotary_train_l4096", 64, 4096, 4, 4, 64, 64, "interleaved", "bfloat16", True, "none", 0),
        # A single request's next token: the latency of a step.
        _step("step_one", 1, 4, 1, 64, 64, "bfloat16"),
        # A serving batch's next tokens: every sequence's state is read and written.
        _step("step_batch", 128, 12, 1, 128, 128, "float16", mask=True),
        # Padded prompts of different lengths, three query heads to a key head; the states go on to the steps.
        _attend("attend_prompts_ragged", 8, 1537, 12, 3, 64, 64, "float16", False, mask=True, state=True),
        # One long prompt: few heads, so that the length has to fill the device.
        _attend("attend_long", 1, 32768, 8, 1, 64, 64, "bfloat16", False, state=True),
        # Training at the published forward + backward shell's features.
        _attend("attend_train_l2048", 64, 2048, 4, 1, 64, 64, "bfloat16", True),
        # A wide layer on pieces of two long sequences, their states carried on.
        _attend("attend_train_wide", 2, 4096, 6, 1, 128, 128, "float16", True, state=True),
        # Heads of each token normalised before the output projection of a training batch.
        _norm("norm_train_heads", 64, 4096, 256, 4, "bfloat16", True, "none", tokens=True),
        # Image features of 56 x 56 positions, 32 groups of channels, in training.
        _norm("norm_train_image", 32, 3136, 256, 32, "float16", True, "silu"),
        # Padded samples, channels of a group that no 16-byte access divides.
        _norm("norm_ragged", 8, 1001, 300, 12, "float32", False, "gelu", mask=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rotary", "attend", "attend", "step", "norm"))
    batch, length = _spread(rng, 1, 64), _spread(rng, 1, 4096)
    half = rng.choice(("float16", "bfloat16"))
    train = rng.random() < 0.5
    dims = (16, 24, 32, 40, 48, 64, 80, 96, 112, 128)
    shared = rng.choice((1, 1, 2, 3))
    heads = shared * rng.randint(1, 4)
    if rng.random() < 0.15:
        batch, length = 1, _spread(rng, 4096, 32768)
    if op == "rotary":
        dim = rng.choice(dims)
        case = _rotary("", batch, length, heads, heads // shared, dim, rng.choice((dim, dim, 2 * (dim // 4))),
                       rng.choice(("interleaved", "half")), rng.choice((half, "float32")), train,
                       rng.choice(("none", "int64", "float32")), rng.choice((0, _spread(rng, 1, 1000000))),
                       factor=rng.choice((1.0, 4.0, 16.0)))
    elif op == "attend":
        case = _attend("", batch, length, heads, shared, rng.choice(dims), rng.choice(dims), half, train,
                       mask=rng.random() < 0.5, state=rng.random() < 0.4)
    elif op == "step":
        case = _step("", _spread(rng, 1, 256), heads, shared, rng.choice(dims), rng.choice(dims), half,
                     mask=rng.random() < 0.4)
    else:
        groups = rng.choice((1, 2, 4, 6, 8, 16, 32))
        case = _norm("", batch, length, groups * rng.choice((4, 5, 8, 12, 16, 25, 32, 64)), groups,
                     rng.choice((half, "float32")), train, rng.choice(("none", "silu", "gelu")),
                     tokens=rng.random() < 0.3, mask=False)
        case["mask"] = not case["tokens"] and rng.random() < 0.4
    del case["name"]
    most = [work(c) for c in listed() if c["op"] == op and c["train"] >= case["train"]]
    while case["batch"] > 1 or case["length"] > 1:
        needed = work(case)
        if any(needed["flops"] <= w["flops"] and needed["bytes"] <= w["bytes"] for w in most):
            break
        if case["batch"] > 1:
            case["batch"] -= 1
        else:
            case["length"] = (case["length"] + 1) // 2
    return case


def work(case):
    s = 4 if case["dtype"] == "float32" else 2
    tokens = case["batch"] * case["length"]
    if case["op"] == "rotary":
        values = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        turned = tokens * (case["heads"] + case["kv_heads"]) * case["rotary"]
        passes = 2 if case["train"] else 1
        ids = {"none": 0, "int64": 8, "float32": 4}[case["positions"]] * tokens
        return {"bytes": passes * 2 * s * values + ids, "flops": passes * 3 * turned}
    if case["op"] in ("attend", "step"):
        heads, kv_heads, d, e = case["heads"], case["heads"] // case["shared"], case["dim"], case["value_dim"]
        inputs = tokens * (heads * d + kv_heads * (d + e))
        states = 4 * case["batch"] * heads * d * e if case["state"] else 0
        moved = s * (inputs + tokens * heads * e) + 2 * states + (tokens if case["mask"] else 0)
        if case["train"]:
            moved += s * (inputs + tokens * heads * e) + 2 * states
        # A product for the state and one for the answer; their gradients are four.
        return {"bytes": moved, "flops": (12 if case["train"] else 4) * tokens * heads * d * e}
    values = tokens * case["channels"]
    moved = s * values * (4 if case["train"] else 2) + 4 * case["channels"] * (4 if case["train"] else 2)
    moved += tokens if case["mask"] else 0
    return {"bytes": moved, "flops": (20 if case["train"] else 8) * values}


def _frequencies(case):
    """Radians a position of each pair, and what the turned features are multiplied by."""

    half = case["rotary"] // 2
    f = _BASE ** (-torch.arange(half, dtype=torch.float64) / half)
    if case["factor"] == 1.0:
        return f, 1.0
    turns = f * (case["original"] / (2.0 * math.pi))
    keep = ((turns - _FEW_TURNS) / (_MANY_TURNS - _FEW_TURNS)).clamp(0.0, 1.0)
    return f * (keep + (1.0 - keep) / case["factor"]), 1.0 + 0.1 * math.log(case["factor"])


def prepare(case, seed):
    device = torch.device("cuda")
    generator = torch.Generator(device=device).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    batch, length = case["batch"], case["length"]
    dtype = getattr(torch, case["dtype"])

    def normal(*shape, kind=dtype, std=1.0):
        return (torch.randn(shape, generator=generator, device=device) * std).to(kind)

    state = {"case": dict(case), "mask": None}
    if case["op"] == "rotary":
        frequencies, state["amplitude"] = _frequencies(case)
        state["frequencies"] = frequencies.to(device)
        state["positions"] = None
        if case["positions"] != "none":
            # Every sequence has come to a place of its own.
            first = case["start"] + torch.randint(0, 1000, (batch, 1), generator=host)
            ids = first + torch.arange(length)
            state["positions"] = ids.to(device=device, dtype=getattr(torch, case["positions"]))
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            shape = (batch, length, heads, case["dim"])
            state[name] = normal(*shape).requires_grad_(case["train"])
            state["d" + name] = normal(*shape) if case["train"] else None
        return state
    if case["op"] == "norm":
        channels = case["channels"]
        shape = (batch * length, channels) if case["tokens"] else (batch, length, channels)
        # Features with a mean of their own, as activations have.
        state["x"] = (normal(*shape, kind=torch.float32) + 0.5 * normal(channels, kind=torch.float32)).to(dtype)
        state["weight"] = 1.0 + normal(channels, kind=torch.float32, std=0.2)
        state["bias"] = normal(channels, kind=torch.float32, std=0.2)
        for name in ("x", "weight", "bias"):
            state[name].requires_grad_(case["train"])
        state["dy"] = normal(*shape) if case["train"] else None
    else:
        heads, kv_heads = case["heads"], case["heads"] // case["shared"]
        rows = (batch,) if case["op"] == "step" else (batch, length)
        for name, count, features in (("q", heads, case["dim"]), ("k", kv_heads, case["dim"]),
                                      ("v", kv_heads, case["value_dim"])):
            state[name] = normal(*rows, count, features).requires_grad_(case["train"])
        # Heads that forget over 8 to 256 tokens.
        spread = torch.arange(heads, dtype=torch.float64) / max(1, heads - 1)
        state["log_decay"] = torch.log1p(-(2.0 ** (-3.0 - 5.0 * spread))).float().to(device)
        state["s0"] = state["ds"] = None
        if case["state"]:
            shape = (batch, heads, case["dim"], case["value_dim"])
            state["s0"] = normal(*shape, kind=torch.float32).requires_grad_(case["train"])
            state["ds"] = normal(*shape, kind=torch.float32) if case["train"] else None
        state["dy"] = normal(*rows, heads, case["value_dim"]) if case["train"] else None
        if case["op"] == "step":
            if case["mask"]:   # sequences that have ended keep their place in the batch
                state["mask"] = (torch.rand(batch, generator=host) < 0.9).to(device)
            return state
    if case["mask"]:
        # Samples between a quarter of the length and all of it, the first one
        # whole and the last of several empty.
        lengths = torch.randint(max(1, length // 4), length + 1, (batch,), generator=host)
        lengths[-1] = 0
        lengths[0] = length
        state["mask"] = (torch.arange(length)[None, :] < lengths[:, None]).to(device)
    return state


@functools.lru_cache(maxsize=None)
def _native():
    from lsso_amd.ball import hip

    hip.load()
    return hip


# ---------------------------------------------------------------- plain forms
def _turned(x, cos, sin, rotary, layout):
    """The first `rotary` features of x turned, in 32 bits."""

    value, rest = x.float()[..., :rotary], x[..., rotary:]
    if layout == "half":
        first, second = value.chunk(2, dim=-1)
        turned = torch.cat((first * cos - second * sin, first * sin + second * cos), dim=-1)
    else:
        first, second = value[..., 0::2], value[..., 1::2]
        turned = torch.stack((first * cos - second * sin, first * sin + second * cos), dim=-1).flatten(-2)
    return torch.cat((turned.to(x.dtype), rest), dim=-1)


def _plain_rotary(state):
    case = state["case"]
    positions = state["positions"]
    if positions is None:
        positions = torch.arange(case["length"], device=state["q"].device).expand(case["batch"], -1)
    angles = positions.double()[..., None, None] * state["frequencies"]
    cos = (angles.cos() * state["amplitude"]).float()
    sin = (angles.sin() * state["amplitude"]).float()
    outputs = [_turned(state["q"], cos, sin, case["rotary"], case["layout"]),
               _turned(state["k"], cos, sin, case["rotary"], case["layout"])]
    if case["train"]:
        outputs += [_turned(state["dq"], cos, -sin, case["rotary"], case["layout"]),
                    _turned(state["dk"], cos, -sin, case["rotary"], case["layout"])]
    return outputs


def _decayed(a, b, c, log_decay, mask, first=None):
    """o_t = sum over s <= t of decay^(tokens between) (a_t . b_s) c_s, plus
    decay^(tokens so far) a_t first, and the state after the last token; by
    chunks.  a, b: [B, H, N, D]; c: [B, H, N, E]; mask: [B, N] of ones and zeros."""

    batch, heads, length, dim = a.shape
    count = (length + _CHUNK - 1) // _CHUNK
    room = count * _CHUNK - length
    a, b, c = (torch.nn.functional.pad(t, (0, 0, 0, room)).unflatten(2, (count, _CHUNK)) for t in (a, b, c))
    rank = torch.nn.functional.pad(mask, (0, room)).cumsum(1).float().view(batch, 1, count, _CHUNK)
    end = rank[..., -1]                                                 # [B, 1, count]
    start = torch.nn.functional.pad(end[..., :-1], (1, 0))
    rate = log_decay.view(1, heads, 1, 1)
    zero = torch.zeros((), device=a.device)
    lower = torch.ones(_CHUNK, _CHUNK, device=a.device, dtype=torch.bool).tril()
    weights = torch.where(lower, torch.exp(rate[..., None] * (rank[..., :, None] - rank[..., None, :]).clamp_min(0.0)), zero)
    within = (a @ b.mT * weights) @ c
    updates = (b * torch.exp(rate * (end[..., None] - rank))[..., None]).mT @ c      # [B, H, count, D, E]
    before = torch.ones(count, count, device=a.device, dtype=torch.bool).tril(-1)
    carry = torch.where(before, torch.exp(rate * (start[..., :, None] - end[..., None, :]).clamp_min(0.0)), zero)
    states = (carry @ updates.flatten(-2)).unflatten(-1, updates.shape[-2:])
    last = (torch.exp(rate * (end[..., -1:, None] - end[..., None, :])) @ updates.flatten(-2)).unflatten(
        -1, updates.shape[-2:])[:, :, 0]
    if first is not None:
        states = states + torch.exp(rate[..., 0] * start)[..., None, None] * first[:, :, None]
        last = last + torch.exp(rate * end[..., -1:, None]) * first
    across = (a * torch.exp(rate * (rank - start[..., None]))[..., None]) @ states
    return (within + across).flatten(2, 3)[:, :, :length], last


def _plain_attend(state):
    case, dtype = state["case"], state["q"].dtype
    shared, log_decay, s0 = case["shared"], state["log_decay"], state["s0"]
    scale = case["dim"] ** -0.5
    mask = state["mask"]
    kept = torch.ones(case["batch"], case["length"], device=log_decay.device) if mask is None else mask.float()

    def heads_first(x, repeat=1):
        x = torch.where(kept[..., None, None] > 0, x.float(), 0.0).transpose(1, 2)
        return x.repeat_interleave(repeat, dim=1)

    def tokens_first(x, repeat=1):
        x = torch.where(kept[:, None, :, None] > 0, x, 0.0)
        return x.unflatten(1, (-1, repeat)).sum(2).transpose(1, 2).to(dtype).contiguous()

    q, k, v = heads_first(state["q"]), heads_first(state["k"], shared), heads_first(state["v"], shared)
    y, last = _decayed(q, k, v, log_decay, kept, s0)
    outputs = [tokens_first(scale * y)] + ([last] if case["state"] else [])
    if not case["train"]:
        return outputs
    dy = scale * heads_first(state["dy"])
    dq, _ = _decayed(dy, v, k, log_decay, kept, None if s0 is None else s0.mT)
    back = kept.flip(1)
    q, k, v, dy = (t.flip(2) for t in (q, k, v, dy))
    dv, ds = _decayed(k, q, dy, log_decay, back)
    dk, _ = _decayed(v, dy, q, log_decay, back)
    if case["state"]:
        # What the last state owes to each token and to the first state.
        rate = log_decay.view(1, -1, 1, 1)
        since = (back.cumsum(1) - back)[:, None, :, None]
        dv = dv + torch.exp(rate * since) * (k @ state["ds"])
        dk = dk + torch.exp(rate * since) * (v @ state["ds"].mT)
        count = kept.sum(1).view(-1, 1, 1, 1)
        ds = torch.exp(rate) * ds + torch.exp(rate * count) * state["ds"]
    outputs += [tokens_first(dq), tokens_first(dk.flip(2), shared), tokens_first(dv.flip(2), shared)]
    return outputs + ([ds] if case["state"] else [])


def _plain_step(state):
    case, s, mask = state["case"], state["s0"], state["mask"]
    q = state["q"].float()
    k, v = (state[name].float().repeat_interleave(case["shared"], dim=1) for name in ("k", "v"))
    new = torch.exp(state["log_decay"])[:, None, None] * s + k[..., :, None] * v[..., None, :]
    y = case["dim"] ** -0.5 * (q[..., None, :] @ new)[..., 0, :]
    if mask is not None:
        new = torch.where(mask[:, None, None, None], new, s)
        y = torch.where(mask[:, None, None], y, 0.0)
    s.copy_(new)
    return [y.to(state["q"].dtype), s]


def _activation(z, name):
    """act(z) and act'(z)."""

    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    return z, torch.ones_like(z)


def _plain_norm(state):
    case, dtype, shape = state["case"], state["x"].dtype, state["x"].shape
    groups = case["groups"]
    grouped = (shape[0], -1, groups, case["channels"] // groups)
    weight, bias = (state[name].view(groups, -1) for name in ("weight", "bias"))
    x = state["x"].float().view(grouped)
    kept = None if state["mask"] is None else state["mask"][..., None, None]
    zero = torch.zeros((), device=x.device)

    def only(t):
        return t if kept is None else torch.where(kept, t, zero)

    tokens = x.shape[1] if kept is None else kept.sum(1, keepdim=True).clamp_min(1)
    size = tokens * x.shape[3]
    mean = only(x).sum((1, 3), keepdim=True) / size
    centred = only(x - mean)
    rstd = torch.rsqrt((centred * centred).sum((1, 3), keepdim=True) / size + _EPS)
    normal = centred * rstd
    y, slope = _activation(normal * weight + bias, case["activation"])
    outputs = [only(y).to(dtype).view(shape)]
    if not case["train"]:
        return outputs
    dz = only(state["dy"].float().view(grouped)) * slope
    dn = dz * weight
    dx = rstd * (dn - (dn.sum((1, 3), keepdim=True) + normal * (dn * normal).sum((1, 3), keepdim=True)) / size)
    grads = (dz * normal).sum((0, 1)).view(-1), dz.sum((0, 1)).view(-1)
    return [*outputs, only(dx).to(dtype).view(shape), *grads]


# ---------------------------------------------------------- framework's calls
def _own_rotary(state):
    case, q, k = state["case"], state["q"], state["k"]
    turned = _native().rotary(q, k, state["positions"], state["frequencies"], layout=case["layout"],
                              amplitude=state["amplitude"])
    if not case["train"]:
        return [*turned]
    return [turned[0].detach(), turned[1].detach(), *torch.autograd.grad(turned, (q, k), (state["dq"], state["dk"]))]


def _own_attend(state):
    case, inputs = state["case"], (state["q"], state["k"], state["v"])
    result = _native().linear_attention(
        *inputs, state["log_decay"], row_mask=state["mask"], initial_state=state["s0"], return_state=case["state"],
    )
    outputs = result if case["state"] else (result,)
    if not case["train"]:
        return [*outputs]
    if case["state"]:
        grads = torch.autograd.grad(outputs, (*inputs, state["s0"]), (state["dy"], state["ds"]))
    else:
        grads = torch.autograd.grad(outputs, inputs, (state["dy"],))
    return [*(value.detach() for value in outputs), *grads]


def _own_step(state):
    y = _native().linear_attention_step(
        state["q"], state["k"], state["v"], state["log_decay"], state["s0"], row_mask=state["mask"]
    )
    return [y, state["s0"]]


def _own_norm(state):
    case, leaves = state["case"], (state["x"], state["weight"], state["bias"])
    activation = None if case["activation"] == "none" else case["activation"]
    y = _native().group_norm(state["x"], case["groups"], state["weight"], state["bias"], eps=_EPS,
                             activation=activation, row_mask=state["mask"])
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "attend": _own_attend, "step": _own_step, "norm": _own_norm}[op](state)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "attend": _plain_attend, "step": _plain_step, "norm": _plain_norm}[op](state)


# --------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    batch, length, train = case["batch"], case["length"], case["train"]
    device = torch.device("cuda")

    def rotary():
        where = torch.arange(length, device=device).expand(batch, -1)
        where = where if state["positions"] is None else state["positions"]
        angle = where.double()[:, :, None, None] * state["frequencies"]
        wheel = torch.polar(torch.full_like(angle, state["amplitude"]), angle)

        def turn(x, by):
            x = x.detach().double()
            part = x[..., :case["rotary"]]
            pairs = part.unflatten(-1, (2, -1)).mT if case["layout"] == "half" else part.unflatten(-1, (-1, 2))
            turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
            turned = turned.mT if case["layout"] == "half" else turned
            return torch.cat((turned.flatten(-2), x[..., case["rotary"]:]), dim=-1)

        outputs = [turn(state["q"], wheel), turn(state["k"], wheel)]
        return outputs + ([turn(state["dq"], wheel.conj()), turn(state["dk"], wheel.conj())] if train else [])

    def attend():
        # Every pair of a query and a key, for one sample and a few heads at a time.
        heads, shared = case["heads"], case["shared"]
        rate = state["log_decay"].double()
        step = max(1, int(2.0e9 // (8 * length * length * shared))) * shared
        total = 4 if case["state"] else 3
        y = torch.zeros(batch, length, heads, case["value_dim"], dtype=torch.float64, device=device)
        last = torch.zeros(batch, heads, case["dim"], case["value_dim"], dtype=torch.float64, device=device)
        grads = [torch.zeros(state[n].shape, dtype=torch.float64, device=device) for n in ("q", "k", "v", "s0")[:total]]
        for b in range(batch):
            chosen = torch.arange(length, device=device) if state["mask"] is None else state["mask"][b].nonzero()[:, 0]
            n = chosen.numel()
            apart = torch.arange(n, device=device)
            apart = apart[:, None] - apart[None, :]
            for h in range(0, heads, step):
                end = min(heads, h + step)
                some, few = slice(h, end), slice(h // shared, end // shared)
                leaves = [state["q"][b, chosen, some], state["k"][b, chosen, few], state["v"][b, chosen, few]]
                leaves += [state["s0"][b, some]] if case["state"] else []
                leaves = [leaf.detach().double().requires_grad_(train) for leaf in leaves]
                q, k, v = (leaf.transpose(0, 1) for leaf in leaves[:3])
                k, v = (t.repeat_interleave(shared, dim=0) for t in (k, v))
                r = rate[some, None, None]
                scores = q @ k.mT
                scores = scores * torch.where(apart >= 0, torch.exp(r * apart.clamp_min(0)), 0.0)
                out = scores @ v
                del scores
                steps = torch.arange(1, n + 1, device=device)[:, None]
                final = (k * torch.exp(r * (n - steps))).mT @ v
                if case["state"]:
                    out = out + torch.exp(r * steps) * (q @ leaves[3])
                    final = final + torch.exp(r * n) * leaves[3]
                out = (case["dim"] ** -0.5 * out).transpose(0, 1)
                y[b, chosen, some], last[b, some] = out.detach(), final.detach()
                if train:
                    ends, given = [out], [state["dy"][b, chosen, some].double()]
                    if case["state"]:
                        ends, given = ends + [final], given + [state["ds"][b, some].double()]
                    found = torch.autograd.grad(ends, leaves, given)
                    grads[0][b, chosen, some], grads[1][b, chosen, few], grads[2][b, chosen, few] = found[:3]
                    if case["state"]:
                        grads[3][b, some] = found[3]
        return [y, *([last] if case["state"] else []), *(grads if train else [])]

    def step():
        keep = torch.ones(batch, dtype=torch.bool, device=device) if state["mask"] is None else state["mask"]
        new, y = state["s0"].double(), torch.zeros_like(state["q"][..., :1].double().expand(-1, -1, case["value_dim"]))
        decay = state["log_decay"].double().exp()
        for h in range(case["heads"]):
            q, k, v = state["q"][:, h].double(), state["k"][:, h // case["shared"]].double(), state["v"][:, h // case["shared"]].double()
            after = decay[h] * new[:, h] + torch.einsum("bd,be->bde", k, v)
            new[:, h] = torch.where(keep[:, None, None], after, new[:, h])
            y[:, h] = torch.where(keep[:, None], (q[:, :, None] * after).sum(1) / math.sqrt(case["dim"]), 0.0)
        return [y, new]

    def norm():
        # Samples one after another; the gradients of weight and bias add up.
        leaves = [state["x"].detach(), *(state[n].detach().double().requires_grad_(train) for n in ("weight", "bias"))]
        x = leaves[0].view(batch, 1 if not case["tokens"] else length, -1, case["channels"])
        y, dx = torch.zeros(x.shape, dtype=torch.float64, device=device), torch.zeros(x.shape, dtype=torch.float64, device=device)
        sums = [torch.zeros(case["channels"], dtype=torch.float64, device=device) for _ in range(2)]
        for b in range(batch):
            kept = slice(None) if state["mask"] is None else state["mask"][b].nonzero()[:, 0]
            rows = x[b][:, kept].double().requires_grad_(train)
            if rows.numel() == 0:
                continue
            parts = rows.unflatten(-1, (case["groups"], -1))
            variance, mean = torch.var_mean(parts, dim=(1, 3), correction=0, keepdim=True)
            z = ((parts - mean) / torch.sqrt(variance + _EPS)).flatten(-2) * leaves[1] + leaves[2]
            if case["activation"] != "none":
                z = z * (torch.sigmoid(z) if case["activation"] == "silu" else torch.special.ndtr(z))
            y[b][:, kept] = z.detach()
            if train:
                dy = state["dy"].view(x.shape)[b][:, kept].double()
                found = torch.autograd.grad(z, (rows, leaves[1], leaves[2]), dy)
                dx[b][:, kept] = found[0]
                sums = [total + part for total, part in zip(sums, found[1:])]
        shape = state["x"].shape
        return [y.view(shape), *([dx.view(shape), *sums] if train else [])]

    return {"rotary": rotary, "attend": attend, "step": step, "norm": norm}[case["op"]]()
