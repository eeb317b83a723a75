"""Native operators of a causal mixer: rotary positions, linear attention with a
decay for each head (over whole sequences and for single tokens) and group norm
with an activation, each with its first-order gradients.

They share the mixer's boundary (``lsso_amd.ball.hip``, which re-exports
them): the same library, loader, errors and stream, no fallback, and device
memory from PyTorch alone.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
import math

import torch

from .block import _ACTIVATIONS, _HALF_CODES, _VALUE_CODES, _hip, _mask_pointer, _on_device, _saved, _without_tangents

_ID_TYPES = {torch.int32: 1, torch.int64: 2, torch.float32: 3, torch.float64: 4}
_LAYOUTS = {"interleaved": 1, "half": 2}
_MOST_FEATURES = 128

SYMBOLS = (
    "lsso_hip_rotary",
    "lsso_hip_group_norm_sizes",
    "lsso_hip_group_norm",
    "lsso_hip_group_norm_backward",
    "lsso_hip_linear_attention_sizes",
    "lsso_hip_linear_attention",
    "lsso_hip_linear_attention_backward",
    "lsso_hip_linear_attention_step",
)


class RotaryTensor(ctypes.Structure):
    """``lsso_hip_rotary_tensor`` (include/lsso_hip.h)."""

    _fields_ = [
        ("x", ctypes.c_void_p),
        ("y", ctypes.c_void_p),
        ("heads", ctypes.c_int64),
        ("batch_stride", ctypes.c_int64),
        ("token_stride", ctypes.c_int64),
        ("head_stride", ctypes.c_int64),
    ]


class GroupNormShape(ctypes.Structure):
    """``lsso_hip_group_norm_shape`` (include/lsso_hip.h)."""

    _fields_ = [
        ("samples", ctypes.c_int64),
        ("length", ctypes.c_int64),
        ("channels", ctypes.c_int64),
        ("groups", ctypes.c_int64),
        ("dtype", ctypes.c_int),
        ("parameter_type", ctypes.c_int),
        ("activation", ctypes.c_int),
        ("eps", ctypes.c_float),
    ]


class HeadStrides(ctypes.Structure):
    """``lsso_hip_head_strides`` (include/lsso_hip.h)."""

    _fields_ = [("batch", ctypes.c_int64), ("token", ctypes.c_int64), ("head", ctypes.c_int64)]


class LinearAttentionShape(ctypes.Structure):
    """``lsso_hip_linear_attention_shape`` (include/lsso_hip.h)."""

    _fields_ = [
        ("batch", ctypes.c_int64),
        ("length", ctypes.c_int64),
        ("heads", ctypes.c_int64),
        ("kv_heads", ctypes.c_int64),
        ("features", ctypes.c_int64),
        ("value_features", ctypes.c_int64),
        ("dtype", ctypes.c_int),
        ("scale", ctypes.c_float),
        ("q", HeadStrides),
        ("k", HeadStrides),
        ("v", HeadStrides),
    ]


def declare(library: ctypes.CDLL) -> None:
    """Argument types of SYMBOLS."""

    vp, i64, i32, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
    size, size_p = ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)
    norm_p, attention_p = ctypes.POINTER(GroupNormShape), ctypes.POINTER(LinearAttentionShape)
    for name, arguments in (
        ("lsso_hip_rotary", [ctypes.POINTER(RotaryTensor), i32, i32, i64, i64, i64, i64, i32, vp, f32, i32, vp, i32,
                             i64, i64, vp]),
        # tensors, count, type, batch, length, features, rotary features, layout, frequencies, amplitude, inverse,
        # positions, type, batch stride, token stride, stream
        ("lsso_hip_group_norm_sizes", [norm_p, size_p, size_p, size_p]),
        ("lsso_hip_group_norm", [norm_p, vp, vp, vp, vp, vp, vp, vp, size, vp]),
        # shape, x, weight, bias, mask, statistics, y, workspace, bytes, stream
        ("lsso_hip_group_norm_backward", [norm_p, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, size, vp]),
        # shape, grad_y, x, weight, bias, mask, statistics, grads (x, weight, bias), workspace, bytes, stream
        ("lsso_hip_linear_attention_sizes", [attention_p, size_p, size_p, size_p]),
        ("lsso_hip_linear_attention", [attention_p, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, size, vp]),
        # shape, q, k, v, log_decay, mask, initial state, kept, y, final state, workspace, bytes, stream
        ("lsso_hip_linear_attention_backward", [attention_p, vp, ctypes.POINTER(HeadStrides), vp, vp, vp, vp, vp, vp,
                                                vp, vp, vp, vp, vp, vp, vp, size, vp]),
        # shape, grad_y, strides, grad of the final state, q, k, v, log_decay, mask, initial state, kept, grads (q, k,
        # v, initial state), workspace, bytes, stream
        ("lsso_hip_linear_attention_step", [attention_p, vp, vp, vp, vp, vp, vp, i64, vp, vp]),
        # shape, q, k, v, log_decay, mask, state, batch stride, y, stream
    ):
        entry = getattr(library, name)
        entry.restype = ctypes.c_int
        entry.argtypes = arguments


def _unit(value: torch.Tensor) -> torch.Tensor:
    """value with unit stride of its last dimension (any other strides)."""

    return value if value.stride(-1) == 1 or value.shape[-1] == 1 else value.contiguous()


# --------------------------------------------------------------------- rotary
def _rotary_launch(values, position_ids, frequencies, layout, amplitude, inverse):
    """The turned tensors of ``values`` (one or two of [B, N, H, D])."""

    hip = _hip()
    library = hip._library()
    values = [_unit(value) for value in values]
    batch, length, _heads, features = values[0].shape
    device = values[0].device
    turned = [torch.empty(value.shape, dtype=value.dtype, device=device) for value in values]
    tensors = (RotaryTensor * len(values))()
    for tensor, value, out in zip(tensors, values, turned):
        tensor.x, tensor.y, tensor.heads = value.data_ptr(), out.data_ptr(), value.shape[2]
        tensor.batch_stride, tensor.token_stride, tensor.head_stride = value.stride()[:3]
    if position_ids is None:
        pointer, kind, batch_stride, token_stride = None, 0, 0, 0
    else:
        pointer, kind = position_ids.data_ptr(), _ID_TYPES[position_ids.dtype]
        batch_stride, token_stride = position_ids.stride() if position_ids.dim() == 2 else (0, position_ids.stride(0))
    status = hip._launch(
        library.lsso_hip_rotary, device,
        tensors, len(values), _VALUE_CODES[values[0].dtype], batch, length, features, 2 * frequencies.shape[0], layout,
        frequencies.data_ptr(), amplitude, int(inverse), pointer, kind, batch_stride, token_stride,
    )
    hip._check(status, library)
    return turned


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, position_ids, frequencies, layout, amplitude):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(position_ids, frequencies)
        ctx.form = (layout, amplitude, frequencies.shape, None if position_ids is None else
                    (position_ids.dtype, tuple(position_ids.shape)))
        turned = _rotary_launch([query] if key is None else [query, key], position_ids, frequencies, layout, amplitude,
                                False)
        return turned[0] if key is None else tuple(turned)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        layout, amplitude, count, ids = ctx.form
        position_ids, frequencies = ctx.saved_tensors
        wanted = [i for i, grad in enumerate(grads) if grad is not None and ctx.needs_input_grad[i]]
        results = [None] * 6
        if wanted:
            device = grads[wanted[0]].device
            frequencies = _saved(frequencies, "frequencies", torch.float64, count, device)
            if ids is not None:
                position_ids = _saved(position_ids, "position_ids", ids[0], ids[1], device)
            turned = _rotary_launch([grads[i] for i in wanted], position_ids, frequencies, layout, amplitude, True)
            for i, value in zip(wanted, turned):
                results[i] = value
        return tuple(results)


def rotary(
    query: torch.Tensor,
    key: torch.Tensor | None,
    position_ids: torch.Tensor | None,
    frequencies: torch.Tensor,
    *,
    layout: str = "interleaved",
    amplitude: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotary positions of a query and a key (or of one tensor: key None).

    query, key: float16, bfloat16 or float32 [B, N, H, D], any number of heads
    each and any strides.  Their first R = 2 * len(frequencies) features are
    turned in pairs, (2j, 2j + 1) in the "interleaved" layout and (j, j + R / 2)
    in the "half" one, by the angle position * frequencies[j], and multiplied by
    ``amplitude``; the other features are copied.  position_ids: int32, int64,
    float32 or float64 [N] or [B, N] (0 .. N - 1 by default).  frequencies:
    float64 on the device (``rotary_frequencies``, also of extended contexts);
    angles are taken in 64 bits, so far positions keep their phases.

    Returns contiguous tensors of the inputs' type.  Differentiable (first order)
    in query and key."""

    _hip().require_available()
    _without_tangents(query, key)
    if not query.is_cuda:
        raise RuntimeError("query must be a CUDA (ROCm device) tensor")
    if query.dtype not in _VALUE_CODES:
        raise TypeError(f"rotary supports float16, bfloat16 and float32, got {query.dtype}")
    if query.dim() != 4 or query.shape[2] == 0:
        raise ValueError(f"query must have shape [B, N, H, D], got {list(query.shape)}")
    batch, length, _heads, features = query.shape
    device = query.device
    if key is not None:
        _on_device(key, "key", device)
        if key.dtype != query.dtype:
            raise TypeError(f"key must be {query.dtype}, got {key.dtype}")
        if key.dim() != 4 or key.shape[:2] != query.shape[:2] or key.shape[3] != features or key.shape[2] == 0:
            raise ValueError(f"key must have shape [{batch}, {length}, G, {features}], got {list(key.shape)}")
    _on_device(frequencies, "frequencies", device)
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1:
        raise TypeError("frequencies must be a float64 tensor of one dimension")
    if not 1 <= frequencies.shape[0] <= features // 2:
        raise ValueError(f"frequencies must be 1 to {features // 2} for {features} features, got {frequencies.shape[0]}")
    if frequencies.requires_grad or (position_ids is not None and position_ids.requires_grad):
        raise ValueError("rotary has no gradients for position_ids and frequencies")
    if position_ids is not None:
        _on_device(position_ids, "position_ids", device)
        if position_ids.dtype not in _ID_TYPES:
            raise TypeError(f"position_ids must be int32, int64, float32 or float64, got {position_ids.dtype}")
        if tuple(position_ids.shape) not in ((length,), (batch, length)):
            raise ValueError(
                f"position_ids must be None, [N] or [B, N] = {[batch, length]}, got {list(position_ids.shape)}"
            )
    kind = _LAYOUTS.get(layout)
    if kind is None:
        raise ValueError(f"layout must be one of {sorted(_LAYOUTS)}, got {layout!r}")
    frequencies = frequencies.contiguous()
    amplitude = float(amplitude)
    if torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad)):
        turned = _Rotary.apply(query, key, position_ids, frequencies, kind, amplitude)
        return (turned, None) if key is None else turned
    turned = _rotary_launch([query] if key is None else [query, key], position_ids, frequencies, kind, amplitude, False)
    return turned[0], turned[1] if key is not None else None


# ----------------------------------------------------------------- group norm
@lru_cache(maxsize=1024)
def _group_norm_plan(shape: tuple):
    """(the native shape, kept floats, forward and backward bytes): they depend
    on these numbers alone."""

    hip = _hip()
    library = hip._library()
    native = GroupNormShape(*shape)
    sizes = [ctypes.c_size_t() for _ in range(3)]
    hip._check(library.lsso_hip_group_norm_sizes(ctypes.byref(native), *map(ctypes.byref, sizes)), library)
    return ctypes.byref(native), *(size.value for size in sizes)


def _pointer(value: torch.Tensor | None):
    return None if value is None else value.data_ptr()


def _group_norm_launch(x, weight, bias, row_mask, shape, keep):
    """y, and with ``keep`` the statistics that the backward reads."""

    hip = _hip()
    library = hip._library()
    device = x.device
    mask, mask_ptr = _mask_pointer(row_mask, x.shape[:-1], device)
    x = x.contiguous()
    native, kept, size, _ = _group_norm_plan(shape)
    statistics = torch.empty(kept, dtype=torch.float32, device=device) if keep and kept else None
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    y = torch.empty(x.shape, dtype=x.dtype, device=device)
    status = hip._launch(
        library.lsso_hip_group_norm, device,
        native, x.data_ptr(), _pointer(weight), _pointer(bias), mask_ptr, _pointer(statistics), y.data_ptr(),
        _pointer(workspace), size,
    )
    hip._check(status, library)
    return y, statistics


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, row_mask, shape):
        y, statistics = _group_norm_launch(x, weight, bias, row_mask, shape, True)
        ctx.save_for_backward(x, weight, bias, row_mask, statistics)
        ctx.shape = shape
        ctx.like = [None if v is None else (v.dtype, tuple(v.shape)) for v in (x, weight, bias, row_mask, statistics)]
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        hip = _hip()
        library = hip._library()
        device = grad_y.device
        saved = [
            None if value is None else _saved(value, name, *like, device)
            for value, name, like in zip(ctx.saved_tensors, ("x", "weight", "bias", "row_mask", "statistics"), ctx.like)
        ]
        x = saved[0]
        needs = ctx.needs_input_grad[:3]
        grads = [
            torch.empty(like[1], dtype=like[0], device=device) if need else None
            for need, like in zip(needs, ctx.like)
        ]
        if not any(needs):
            return (None,) * 5
        native, _, _, size = _group_norm_plan(ctx.shape)
        workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        grad_y = grad_y.contiguous()
        status = hip._launch(
            library.lsso_hip_group_norm_backward, device,
            native, grad_y.data_ptr(), *(_pointer(value) for value in saved), *(_pointer(grad) for grad in grads),
            _pointer(workspace), size,
        )
        hip._check(status, library)
        return (*grads, None, None)


def group_norm(
    x: torch.Tensor,
    groups: int,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    *,
    eps: float = 1e-5,
    activation: str | None = None,
    row_mask: torch.Tensor | None = None,
) -> torch.Tensor:
    """Group norm with an activation, channels last:
    y = act((x - mean) / sqrt(var + eps) * weight + bias).

    x: float16, bfloat16 or float32 [B, ..., C]; the statistics of sample b and
    group g are over all its tokens and the g-th C / groups channels, so [B * N, C]
    normalises each token by itself.  weight, bias: [C] of x's type or float32, or
    None (ones, zeros).  activation: None, "silu" or "gelu" (exact).  row_mask
    (bool, x.shape[:-1]): the tokens it excludes count in no statistic, whatever
    they hold, give zeros and reach no gradient.  y: contiguous, of x's type.

    Statistics and sums are FP32, variances from deviations.  Differentiable (first
    order) in x, weight and bias, deterministically.  Tokens by themselves of groups of
    more than 8,192 channels go as samples of one row, with a workspace of two FP32
    values for each of x."""

    _hip().require_available()
    _without_tangents(x, weight, bias)
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA (ROCm device) tensor")
    if x.dtype not in _VALUE_CODES:
        raise TypeError(f"group norm supports float16, bfloat16 and float32, got {x.dtype}")
    if x.dim() < 2 or x.shape[-1] == 0:
        raise ValueError(f"x must have shape [B, ..., C], got {list(x.shape)}")
    channels = x.shape[-1]
    if not isinstance(groups, int) or isinstance(groups, bool) or groups <= 0 or channels % groups:
        raise ValueError(f"groups must be a positive divisor of {channels} channels, got {groups!r}")
    given = [value for value in (weight, bias) if value is not None]
    for name, value in (("weight", weight), ("bias", bias)):
        if value is not None:
            _on_device(value, name, x.device)
            if value.dtype not in (x.dtype, torch.float32) or value.dtype != given[0].dtype:
                raise TypeError(f"weight and bias must both be {x.dtype} or float32, got {value.dtype}")
            if tuple(value.shape) != (channels,):
                raise ValueError(f"{name} must have shape [{channels}], got {list(value.shape)}")
    if activation is not None and activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be None or one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if weight is not None:
        weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    shape = (
        x.shape[0], math.prod(x.shape[1:-1]), channels, groups, _VALUE_CODES[x.dtype],
        _VALUE_CODES[given[0].dtype if given else x.dtype], 0 if activation is None else _ACTIVATIONS[activation], eps,
    )
    if torch.is_grad_enabled() and (x.requires_grad or any(value.requires_grad for value in given)):
        return _GroupNorm.apply(x, weight, bias, row_mask, shape)
    return _group_norm_launch(x, weight, bias, row_mask, shape, False)[0]


# ----------------------------------------------------------- linear attention
@lru_cache(maxsize=1024)
def _attention_plan(fields: tuple, strides: tuple):
    """(the native shape, kept floats, forward and backward bytes): they depend on
    these numbers alone."""

    hip = _hip()
    library = hip._library()
    native = LinearAttentionShape(*fields, *(HeadStrides(*s) for s in strides))
    sizes = [ctypes.c_size_t() for _ in range(3)]
    hip._check(library.lsso_hip_linear_attention_sizes(ctypes.byref(native), *map(ctypes.byref, sizes)), library)
    return ctypes.byref(native), *(size.value for size in sizes)


def _attention_fields(query, key, value, scale):
    batch, length, heads, features = query.shape
    return batch, length, heads, key.shape[2], features, value.shape[3], _HALF_CODES[query.dtype], scale


def _attention_launch(query, key, value, log_decay, scale, row_mask, initial_state, return_state, keep):
    """(y, the last state or None, and with ``keep`` what the backward reads or None)."""

    hip = _hip()
    library = hip._library()
    device = query.device
    query, key, value = _unit(query), _unit(key), _unit(value)
    mask, mask_ptr = _mask_pointer(row_mask, query.shape[:2], device)
    native, kept, size, _ = _attention_plan(
        _attention_fields(query, key, value, scale), tuple(t.stride()[:3] for t in (query, key, value))
    )
    states = torch.empty(kept, dtype=torch.float32, device=device) if keep and kept else None
    state = initial_state if initial_state is None else initial_state.contiguous()
    batch, length, heads, features = query.shape
    y = torch.empty((batch, length, heads, value.shape[3]), dtype=query.dtype, device=device)
    last = None
    if return_state:
        last = torch.empty((batch, heads, features, value.shape[3]), dtype=torch.float32, device=device)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    status = hip._launch(
        library.lsso_hip_linear_attention, device,
        native, query.data_ptr(), key.data_ptr(), value.data_ptr(), log_decay.data_ptr(), mask_ptr, _pointer(state),
        _pointer(states), y.data_ptr(), _pointer(last), _pointer(workspace), size,
    )
    hip._check(status, library)
    return y, last, states


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, initial_state, log_decay, scale, row_mask, return_state):
        ctx.set_materialize_grads(False)
        y, last, states = _attention_launch(
            query, key, value, log_decay, scale, row_mask, initial_state, return_state, ctx.needs_input_grad[0]
        )
        saved = (query, key, value, initial_state, log_decay, row_mask, states)
        ctx.save_for_backward(*saved)
        ctx.scale = scale
        ctx.like = [None if v is None else (v.dtype, tuple(v.shape)) for v in saved]
        return (y, last) if return_state else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_last=None):
        hip = _hip()
        library = hip._library()
        needs = ctx.needs_input_grad[:4]
        if (grad_y is None and grad_last is None) or not any(needs):
            return (None,) * 8
        device = (grad_last if grad_y is None else grad_y).device
        names = ("query", "key", "value", "initial_state", "log_decay", "row_mask", "states")
        saved = list(ctx.saved_tensors)
        for i, (name, like) in enumerate(zip(names, ctx.like)):
            if saved[i] is None:
                continue
            if saved[i].device != device or saved[i].dtype != like[0] or tuple(saved[i].shape) != like[1]:
                _saved(saved[i], name, *like, device)
            saved[i] = _unit(saved[i]) if i < 3 else saved[i].contiguous()
        query, key, value, initial_state, log_decay, row_mask, states = saved
        batch, length, heads, _features = query.shape
        if grad_y is None:
            grad_y = torch.zeros((1, 1, 1, value.shape[3]), dtype=query.dtype, device=device)
            grad_y = grad_y.expand(batch, length, heads, -1)
        grad_y = _unit(grad_y)
        grad_last = None if grad_last is None else grad_last.contiguous()
        grads = [
            torch.empty(like[1], dtype=like[0], device=device) if need else None
            for need, like in zip(needs, ctx.like)
        ]
        native, _, _, size = _attention_plan(
            _attention_fields(query, key, value, ctx.scale), tuple(t.stride()[:3] for t in (query, key, value))
        )
        workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        status = hip._launch(
            library.lsso_hip_linear_attention_backward, device,
            native, grad_y.data_ptr(), ctypes.byref(HeadStrides(*grad_y.stride()[:3])), _pointer(grad_last),
            query.data_ptr(), key.data_ptr(), value.data_ptr(), log_decay.data_ptr(), _pointer(row_mask),
            _pointer(initial_state), _pointer(states), *(_pointer(grad) for grad in grads), _pointer(workspace), size,
        )
        hip._check(status, library)
        return (*grads, None, None, None, None)


def _check_attention(query, key, value, log_decay, state, dims: int) -> None:
    """What linear_attention and its step refuse alike; dims: of the tensors."""

    if not query.is_cuda:
        raise RuntimeError("query must be a CUDA (ROCm device) tensor")
    if query.dtype not in _HALF_CODES:
        raise TypeError(f"linear attention supports float16 and bfloat16, got {query.dtype}")
    device = query.device
    for name, tensor in (("key", key), ("value", value)):
        _on_device(tensor, name, device)
        if tensor.dtype != query.dtype:
            raise TypeError(f"{name} must be {query.dtype}, got {tensor.dtype}")
    rows = query.shape[:dims - 2]
    if (
        query.dim() != dims or key.dim() != dims or value.dim() != dims or key.shape[:-2] != rows
        or value.shape[:-1] != key.shape[:-1] or key.shape[-1] != query.shape[-1] or 0 in query.shape[-2:]
        or 0 in key.shape[-2:] or value.shape[-1] == 0 or query.shape[-2] % key.shape[-2]
    ):
        raise ValueError(
            f"query [{'B, N' if dims == 4 else 'B'}, H, D], key [..., G, D] and value [..., G, E] must agree and G divide "
            f"H, got {list(query.shape)}, {list(key.shape)} and {list(value.shape)}"
        )
    heads, features, out = query.shape[-2], query.shape[-1], value.shape[-1]
    if features > _MOST_FEATURES or out > _MOST_FEATURES:
        raise ValueError(f"linear attention takes up to {_MOST_FEATURES} features a head, got {features} and {out}")
    _on_device(log_decay, "log_decay", device)
    if log_decay.dtype != torch.float32 or tuple(log_decay.shape) != (heads,):
        raise ValueError(f"log_decay must be float32 [{heads}], got {log_decay.dtype} {list(log_decay.shape)}")
    if log_decay.requires_grad:
        raise ValueError("linear attention has no gradient for log_decay: the decays are fixed")
    if state is not None:
        _on_device(state, "state", device)
        if state.dtype != torch.float32 or tuple(state.shape) != (rows[0], heads, features, out):
            raise ValueError(
                f"the state must be float32 {[rows[0], heads, features, out]}, got {state.dtype} {list(state.shape)}"
            )


def linear_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    log_decay: torch.Tensor,
    *,
    scale: float | None = None,
    row_mask: torch.Tensor | None = None,
    initial_state: torch.Tensor | None = None,
    return_state: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Causal linear attention with a decay for each head:
    S_t = exp(log_decay_h) S_{t-1} + k_t (x) v_t,  y_t = scale q_t S_t.

    query: float16/bfloat16 [B, N, H, D]; key: [B, N, G, D]; value: [B, N, G, E]; G
    divides H, and head h reads key and value head h // (H / G); D and E up to 128,
    any strides.  log_decay: float32 [H], at most 0.  scale: D^-0.5 by default.
    row_mask (bool [B, N]): an excluded token leaves S as it is, as if it were not
    there, whatever it holds; its y is zero and it reaches no gradient.
    initial_state: float32 [B, H, D, E] (zeros by default).  Returns y, contiguous
    [B, N, H, E], and with ``return_state`` the float32 state after the last token,
    which a later call or ``linear_attention_step`` goes on from.

    S is FP32; products take 16-bit operands, FP32 ones as parts that hold them (24
    bits in BF16, 22 in FP16), and accumulate in FP32: y and the gradients are off by
    one rounding of their type.  An infinity or a NaN reaches no y before its token.
    Differentiable (first order) in query, key, value and initial_state,
    deterministically; log_decay is fixed."""

    _hip().require_available()
    _without_tangents(query, key, value, log_decay, initial_state)
    _check_attention(query, key, value, log_decay, initial_state, 4)
    scale = query.shape[-1] ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    log_decay = log_decay.contiguous()
    return_state = bool(return_state)
    if torch.is_grad_enabled() and (
        query.requires_grad or key.requires_grad or value.requires_grad
        or (initial_state is not None and initial_state.requires_grad)
    ):
        return _LinearAttention.apply(query, key, value, initial_state, log_decay, scale, row_mask, return_state)
    y, last, _ = _attention_launch(
        query, key, value, log_decay, scale, row_mask, initial_state, return_state, False
    )
    return (y, last) if return_state else y


def linear_attention_step(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    log_decay: torch.Tensor,
    state: torch.Tensor,
    *,
    scale: float | None = None,
    row_mask: torch.Tensor | None = None,
) -> torch.Tensor:
    """One token of ``linear_attention`` for each sequence: ``state`` becomes S of
    that token in place, and y [B, H, E] is returned.

    query: [B, H, D]; key: [B, G, D]; value: [B, G, E]; state: float32 [B, H, D, E],
    contiguous but for its batch stride.  row_mask (bool [B]): the sequences it
    excludes keep their state, and their y is zero.  FP32 throughout, y rounded
    once.  No gradients: a training step runs ``linear_attention``."""

    hip = _hip()
    hip.require_available()
    _without_tangents(query, key, value, log_decay, state)
    _check_attention(query, key, value, log_decay, state, 3)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (query, key, value, state)):
        raise RuntimeError("linear_attention_step has no gradients: call it under torch.no_grad()")
    scale = query.shape[-1] ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    batch, heads, features, out = state.shape
    one = state[0] if batch else state
    if not one.is_contiguous() or (batch > 1 and state.stride(0) < heads * features * out):
        raise ValueError("state must be contiguous but for its batch stride, since it is updated in place")
    library = hip._library()
    device = query.device
    query, key, value, log_decay = _unit(query), _unit(key), _unit(value), log_decay.contiguous()
    mask, mask_ptr = _mask_pointer(row_mask, (batch,), device)
    native, *_ = _attention_plan(
        (batch, 1, heads, key.shape[1], features, out, _HALF_CODES[query.dtype], scale),
        tuple((t.stride(0), 0, t.stride(1)) for t in (query, key, value)),
    )
    y = torch.empty((batch, heads, out), dtype=query.dtype, device=device)
    status = hip._launch(
        library.lsso_hip_linear_attention_step, device,
        native, query.data_ptr(), key.data_ptr(), value.data_ptr(), log_decay.data_ptr(), mask_ptr, state.data_ptr(),
        state.stride(0) if batch > 1 else heads * features * out, y.data_ptr(),
    )
    hip._check(status, library)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return y


__all__ = ["group_norm", "linear_attention", "linear_attention_step", "rotary"]
