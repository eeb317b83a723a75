"""Native operators around the mixer: token embedding, gated feed-forward block
and residual dropout, each with its first-order gradients.

They share the mixer's boundary (``lsso_amd.ball.hip``, which re-exports
them): the same library, loader, errors and stream, no fallback, and device
memory from PyTorch alone.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache

import torch
from torch.autograd import forward_ad

_F32 = 3
_VALUE_CODES = {torch.float16: 1, torch.bfloat16: 2, torch.float32: _F32}
_HALF_CODES = {torch.float16: 1, torch.bfloat16: 2}
_TOKEN_BYTES = {torch.int32: 4, torch.int64: 8}
_ACTIVATIONS = {"silu": 1, "gelu": 2}
_MOST_ELEMENTS = 1 << 34

SYMBOLS = (
    "lsso_hip_embedding",
    "lsso_hip_embedding_grad_workspace_bytes",
    "lsso_hip_embedding_grad",
    "lsso_hip_dropout_add",
    "lsso_hip_feed_forward_kept",
    "lsso_hip_feed_forward_workspace_bytes",
    "lsso_hip_feed_forward",
    "lsso_hip_feed_forward_backward_workspace_bytes",
    "lsso_hip_feed_forward_backward",
)


class FeedForwardShape(ctypes.Structure):
    """``lsso_hip_feed_forward_shape`` (include/lsso_hip.h)."""

    _fields_ = [
        ("rows", ctypes.c_int64),
        ("in_features", ctypes.c_int64),
        ("hidden", ctypes.c_int64),
        ("out_features", ctypes.c_int64),
        ("x_stride", ctypes.c_int64),
        ("dtype", ctypes.c_int),
        ("weight_type", ctypes.c_int),
        ("activation", ctypes.c_int),
        ("fine_factors", ctypes.c_int),
    ]


def declare(library: ctypes.CDLL) -> None:
    """Argument types of SYMBOLS."""

    vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
    size, size_p = ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)
    shape_p = ctypes.POINTER(FeedForwardShape)
    for name, arguments in (
        ("lsso_hip_embedding", [vp, i32, i64, vp, i32, i64, i64, i64, ctypes.c_float, vp, vp, i32, vp]),
        # tokens, token bytes, count, weight, type, vocabulary, dim, stride, scale, mask, y, type, stream
        ("lsso_hip_embedding_grad_workspace_bytes", [i64, i64, i64, size_p]),
        ("lsso_hip_embedding_grad", [vp, i32, i64, vp, i32, i64, i64, i64, ctypes.c_float, vp, i64, vp, i32, vp,
                                     size, vp]),
        # tokens, token bytes, count, grad_y, type, stride, vocabulary, dim, scale, mask, padding index,
        # grad_weight, type, workspace, bytes, stream
        ("lsso_hip_dropout_add", [vp, vp, i32, i64, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_uint64, vp, vp, vp]),
        # x, residual, type, count, threshold, seed, offset, state, y, stream
        ("lsso_hip_feed_forward_kept", [shape_p, size_p, size_p]),
        ("lsso_hip_feed_forward_workspace_bytes", [shape_p, i32, size_p]),
        ("lsso_hip_feed_forward", [shape_p, vp, vp, vp, vp, vp, vp, vp, vp, vp, size, vp]),
        # shape, x, gate, up, down, mask, gates, product, y, workspace, bytes, stream
        ("lsso_hip_feed_forward_backward_workspace_bytes", [shape_p, i64, i32, size_p]),
        ("lsso_hip_feed_forward_backward", [shape_p, vp, i64, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, size,
                                            vp]),
        # shape, grad_y, stride, x, gate, up, down, mask, gates, product, grads (x, gate, up, down),
        # workspace, bytes, stream
    ):
        entry = getattr(library, name)
        entry.restype = ctypes.c_int
        entry.argtypes = arguments


@lru_cache(maxsize=1)
def _hip():
    """The boundary module, which imports this one."""

    from . import hip

    return hip


def _on_device(value: torch.Tensor, name: str, device: torch.device) -> None:
    if not value.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA (ROCm device) tensor")
    if value.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {value.device}")


def _without_tangents(*values: torch.Tensor | None) -> None:
    """Refuse forward-mode derivatives: a launch outside autograd would drop
    them without a word."""

    if forward_ad._current_level < 0:   # no forward-mode level is open
        return
    for value in values:
        if value is not None and forward_ad.unpack_dual(value).tangent is not None:
            raise NotImplementedError("the native path has no forward-mode derivatives")


def _mask_pointer(row_mask: torch.Tensor | None, shape: tuple, device: torch.device):
    """(contiguous mask or None, its address or None)."""

    if row_mask is None:
        return None, None
    if row_mask.dtype != torch.bool or tuple(row_mask.shape) != tuple(shape):
        raise ValueError(f"row_mask must be a bool tensor of shape {tuple(shape)}")
    _on_device(row_mask, "row_mask", device)
    row_mask = row_mask.contiguous()
    return row_mask, row_mask.data_ptr()


def _saved(value: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device: torch.device) -> torch.Tensor:
    """A saved tensor whose extent is checked before its pointer is taken: a
    program's saved-tensor hooks may hand back another one."""

    if value.device != device or value.dtype != dtype or tuple(value.shape) != tuple(shape):
        raise RuntimeError(
            f"the saved {name} must be {dtype} {list(shape)} on {device}, "
            f"got {value.dtype} {list(value.shape)} on {value.device}"
        )
    return value if value.is_contiguous() else value.contiguous()


# ------------------------------------------------------------------ embedding
@lru_cache(maxsize=1024)
def _embedding_workspace(count: int, vocabulary: int, dim: int) -> int:
    hip = _hip()
    library = hip._library()
    size = ctypes.c_size_t()
    hip._check(library.lsso_hip_embedding_grad_workspace_bytes(count, vocabulary, dim, ctypes.byref(size)), library)
    return size.value


def _embedding_forward(tokens, weight, scale, row_mask, output_dtype):
    hip = _hip()
    library = hip._library()
    device = weight.device
    vocabulary, dim = weight.shape
    mask, mask_ptr = _mask_pointer(row_mask, tokens.shape, device)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    if weight.stride(1) != 1 or weight.stride(0) < dim:
        weight = weight.contiguous()
    y = torch.empty((*tokens.shape, dim), dtype=output_dtype, device=device)
    status = hip._launch(
        library.lsso_hip_embedding, device,
        tokens.data_ptr(), _TOKEN_BYTES[tokens.dtype], tokens.numel(), weight.data_ptr(),
        _VALUE_CODES[weight.dtype], vocabulary, dim, weight.stride(0) if vocabulary > 1 else dim, scale, mask_ptr,
        y.data_ptr(), _VALUE_CODES[output_dtype],
    )
    hip._check(status, library)
    return y


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, row_mask, padding_index, output_dtype):
        y = _embedding_forward(tokens, weight, scale, row_mask, output_dtype)
        ctx.save_for_backward(tokens, row_mask)
        ctx.table = (tuple(weight.shape), weight.dtype, tuple(tokens.shape), tokens.dtype)
        ctx.scale = scale
        ctx.padding_index = -1 if padding_index is None else padding_index
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        hip = _hip()
        library = hip._library()
        device = grad_y.device
        tokens, row_mask = ctx.saved_tensors
        (vocabulary, dim), weight_dtype, token_shape, token_dtype = ctx.table
        tokens = _saved(tokens, "tokens", token_dtype, token_shape, device)
        if row_mask is not None:
            row_mask = _saved(row_mask, "row_mask", torch.bool, token_shape, device)
        flat = hip._rows(grad_y, dim)
        count = tokens.numel()
        grad = torch.empty((vocabulary, dim), dtype=weight_dtype, device=device)
        size = _embedding_workspace(count, vocabulary, dim)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        status = hip._launch(
            library.lsso_hip_embedding_grad, device,
            tokens.data_ptr(), _TOKEN_BYTES[token_dtype], count, flat.data_ptr(), _VALUE_CODES[flat.dtype],
            flat.stride(0) if count > 1 else dim, vocabulary, dim, ctx.scale,
            None if row_mask is None else row_mask.data_ptr(), ctx.padding_index, grad.data_ptr(),
            _VALUE_CODES[weight_dtype], workspace.data_ptr(), size,
        )
        hip._check(status, library)
        return None, grad, None, None, None, None


def embedding(
    tokens: torch.Tensor,
    weight: torch.Tensor,
    *,
    scale: float = 1.0,
    row_mask: torch.Tensor | None = None,
    padding_index: int | None = None,
    output_dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """Token embedding y = cast(scale * weight[tokens]).

    tokens: int32 or int64 ids of any shape; weight: float16, bfloat16 or
    float32 [V, D]; y: contiguous [*tokens.shape, D] of ``output_dtype`` (the
    weight's by default).  ``row_mask`` (bool, tokens.shape): tokens it excludes
    give zeros and no gradient, whatever their id.  ``padding_index``: a row of
    the table that receives no gradient.  The row of an id outside [0, V) that
    is not masked is NaN, and it has no gradient.

    Differentiable (first order) in ``weight``: the dense [V, D] gradient is
    summed in FP32 per table row over the sorted tokens, deterministically."""

    _hip().require_available()
    _without_tangents(weight)
    if not weight.is_cuda:
        raise RuntimeError("weight must be a CUDA (ROCm device) tensor")
    if weight.dim() != 2 or weight.dtype not in _VALUE_CODES:
        raise TypeError("weight must be a float16, bfloat16 or float32 [V, D] tensor")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError("weight must have at least one row and one feature")
    if tokens.dtype not in _TOKEN_BYTES:
        raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
    _on_device(tokens, "tokens", weight.device)
    output_dtype = weight.dtype if output_dtype is None else output_dtype
    if output_dtype not in _VALUE_CODES:
        raise TypeError("output_dtype must be float16, bfloat16 or float32")
    scale = float(scale)
    if padding_index is not None and not 0 <= padding_index < weight.shape[0]:
        raise ValueError(f"padding_index must be a row of the table, got {padding_index}")
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(tokens, weight, scale, row_mask, padding_index, output_dtype)
    return _embedding_forward(tokens, weight, scale, row_mask, output_dtype)


# -------------------------------------------------------------------- dropout
def dropout_threshold(probability: float) -> int:
    """The drop probability in units of 2^-16, as the generator applies it."""

    if not 0.0 <= probability < 1.0:
        raise ValueError(f"probability must be in [0, 1), got {probability}")
    return min(65535, int(probability * 65536.0 + 0.5))


def _dropout_launch(x, residual, threshold, seed, offset, state):
    hip = _hip()
    library = hip._library()
    if not x.is_contiguous():
        x = x.contiguous()
    if residual is not None and not residual.is_contiguous():
        residual = residual.contiguous()
    y = torch.empty_like(x)
    status = hip._launch(
        library.lsso_hip_dropout_add, x.device,
        x.data_ptr(), None if residual is None else residual.data_ptr(), _VALUE_CODES[x.dtype], x.numel(), threshold,
        seed, offset, None if state is None else state.data_ptr(), y.data_ptr(),
    )
    hip._check(status, library)
    return y


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, seed, offset, state):
        if state is not None:
            ctx.save_for_backward(state)
        ctx.draw = (threshold, seed, offset, state is not None)
        ctx.device = x.device
        return _dropout_launch(x, residual, threshold, seed, offset, state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        threshold, seed, offset, by_state = ctx.draw
        state = _saved(ctx.saved_tensors[0], "seed", torch.int64, (2,), ctx.device) if by_state else None
        needs_x, needs_residual = ctx.needs_input_grad[:2]
        grad_x = _dropout_launch(grad_y, None, threshold, seed, offset, state) if needs_x else None
        return grad_x, grad_y if needs_residual else None, None, None, None, None


def dropout_add(
    x: torch.Tensor,
    residual: torch.Tensor | None,
    probability: float,
    seed: int | torch.Tensor,
    offset: int = 0,
) -> torch.Tensor:
    """Residual dropout y = residual + keep * x * s (without a residual, the
    second term alone), with a mask that is never stored.

    x, residual: float16, bfloat16 or float32 of one shape; y is contiguous.
    Element i (in row-major order of the shape) is kept when the 16-bit value i
    % 8 of the Philox-4x32-10 block of counter (i // 8, offset) under the key
    ``seed`` is at least t = round(65536 * probability); s = 65536 / (65536 - t).
    A dropped element is left out, whatever it holds.

    ``seed``: an integer, or a device int64 tensor [2] of a seed and a number
    that is added to ``offset``, which a captured graph reads at each replay.
    The tensor must not change between the forward and its backward.  Calls
    that must not share a mask take different seeds or offsets.

    Differentiable (first order) in x and residual; the backward draws the mask
    again."""

    _hip().require_available()
    _without_tangents(x, residual)
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA (ROCm device) tensor")
    if x.dtype not in _VALUE_CODES:
        raise TypeError(f"dropout supports float16, bfloat16 and float32, got {x.dtype}")
    if x.numel() > _MOST_ELEMENTS:
        raise ValueError(f"dropout takes up to {_MOST_ELEMENTS} elements, got {x.numel()}")
    if residual is not None:
        _on_device(residual, "residual", x.device)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(
                f"residual must be {x.dtype} {list(x.shape)}, got {residual.dtype} {list(residual.shape)}"
            )
    threshold = dropout_threshold(probability)
    state = None
    if isinstance(seed, torch.Tensor):
        _on_device(seed, "seed", x.device)
        if seed.dtype != torch.int64 or tuple(seed.shape) != (2,) or not seed.is_contiguous():
            raise ValueError("seed must be an integer or a contiguous int64 tensor [2]")
        state, seed = seed, 0
    seed, offset = int(seed) & 0xFFFFFFFFFFFFFFFF, int(offset) & 0xFFFFFFFFFFFFFFFF
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _DropoutAdd.apply(x, residual, threshold, seed, offset, state)
    return _dropout_launch(x, residual, threshold, seed, offset, state)


# --------------------------------------------------------------- feed-forward
@lru_cache(maxsize=1024)
def _feed_forward_plan(shape: tuple, training: bool):
    """(the native shape, its workspace's bytes) of a forward: they depend on
    these integers alone, and a program asks for the same few on every call."""

    hip = _hip()
    library = hip._library()
    native = FeedForwardShape(*shape)
    size = ctypes.c_size_t()
    hip._check(library.lsso_hip_feed_forward_workspace_bytes(
        ctypes.byref(native), int(training), ctypes.byref(size)), library)
    return ctypes.byref(native), size.value


@lru_cache(maxsize=1024)
def _feed_forward_backward_plan(shape: tuple, grad_stride: int, weights: int):
    hip = _hip()
    library = hip._library()
    native = FeedForwardShape(*shape)
    size = ctypes.c_size_t()
    hip._check(library.lsso_hip_feed_forward_backward_workspace_bytes(
        ctypes.byref(native), grad_stride, weights, ctypes.byref(size)), library)
    return ctypes.byref(native), size.value


def _aligned(value: torch.Tensor) -> torch.Tensor:
    """value at a 16-byte aligned address (a view may begin anywhere)."""

    return value if value.data_ptr() % 16 == 0 else value.clone()


def _feed_forward_kept(rows: int, hidden: int, dtype: torch.dtype, fine: bool) -> tuple[int, int]:
    """Values of the kept gates, and a row of the kept product
    (``lsso_hip_feed_forward_kept``)."""

    pitch = (hidden + 7) // 8 * 8
    lower = (hidden + 31) // 32 * (16 if dtype == torch.bfloat16 else 32) if fine else 0
    return rows * (2 * pitch + lower), pitch


def _feed_forward_inputs(x, gate_weight, up_weight, down_weight, activation, fine):
    """(rows of x, weights, their addresses, the shape's fields)."""

    hidden, in_features = gate_weight.shape
    flat = _hip()._rows(x, in_features)
    if flat.data_ptr() % 16 != 0:
        flat = flat.clone()
    weights, pointers = (gate_weight, up_weight, down_weight), []
    if not (gate_weight.is_contiguous() and up_weight.is_contiguous() and down_weight.is_contiguous()):
        weights = tuple(w.contiguous() for w in weights)
    for w in weights:
        pointers.append(w.data_ptr())
    if (pointers[0] | pointers[1] | pointers[2]) % 16 != 0:
        weights = tuple(_aligned(w) for w in weights)
        pointers = [w.data_ptr() for w in weights]
    rows = flat.shape[0]
    shape = (
        rows, in_features, hidden, down_weight.shape[0], flat.stride(0) if rows > 1 else in_features,
        _HALF_CODES[x.dtype], _VALUE_CODES[gate_weight.dtype], activation, int(fine),
    )
    return flat, weights, pointers, shape


def _feed_forward_launch(x, gate_weight, up_weight, down_weight, activation, row_mask, training, fine=False):
    """y, and with ``training`` the kept gates and product."""

    hip = _hip()
    library = hip._library()
    device = x.device
    mask_ptr = None
    if row_mask is not None:
        _mask, mask_ptr = _mask_pointer(row_mask, x.shape[:-1], device)
    flat, _weights, pointers, shape = _feed_forward_inputs(
        x, gate_weight, up_weight, down_weight, activation, fine
    )
    gates = product = None
    if training:
        kept, pitch = _feed_forward_kept(shape[0], shape[2], x.dtype, fine)
        gates = torch.empty(kept, dtype=x.dtype, device=device)
        product = torch.empty((shape[0], pitch), dtype=x.dtype, device=device)
    y = torch.empty((*x.shape[:-1], shape[3]), dtype=x.dtype, device=device)
    native, size = _feed_forward_plan(shape, training)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    status = hip._launch(
        library.lsso_hip_feed_forward, device,
        native, flat.data_ptr(), *pointers, mask_ptr, gates.data_ptr() if training else None,
        product.data_ptr() if training else None, y.data_ptr(), workspace.data_ptr() if size else None, size,
    )
    hip._check(status, library)
    return y, gates, product


class _FeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, down_weight, activation, row_mask, fine):
        y, gates, product = _feed_forward_launch(
            x, gate_weight, up_weight, down_weight, activation, row_mask, True, fine
        )
        ctx.save_for_backward(x, gate_weight, up_weight, down_weight, row_mask, gates, product)
        ctx.activation = activation
        ctx.fine = fine
        ctx.like = tuple((tuple(v.shape), v.dtype) for v in (x, gate_weight, up_weight, down_weight))
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        hip = _hip()
        library = hip._library()
        device = grad_y.device
        x, *weights, row_mask, gates, product = ctx.saved_tensors
        for value, name, (shape, dtype) in zip((x, *weights), ("x", "gate_weight", "up_weight", "down_weight"), ctx.like):
            if value.device != device or value.dtype != dtype or tuple(value.shape) != shape:
                _saved(value, name, dtype, shape, device)
        flat, weights, pointers, shape = _feed_forward_inputs(x, *weights, ctx.activation, ctx.fine)
        rows, in_features, hidden, out_features = shape[:4]
        kept, pitch = _feed_forward_kept(rows, hidden, x.dtype, ctx.fine)
        gates = _aligned(_saved(gates, "gates", x.dtype, (kept,), device))
        product = _aligned(_saved(product, "product", x.dtype, (rows, pitch), device))
        mask_ptr = None
        if row_mask is not None:
            row_mask = _saved(row_mask, "row_mask", torch.bool, x.shape[:-1], device)
            mask_ptr = row_mask.data_ptr()
        flat_grad = _aligned(hip._rows(grad_y, out_features))
        grad_stride = flat_grad.stride(0) if rows > 1 else out_features
        needs = ctx.needs_input_grad[:4]
        grads = [
            torch.empty(like, dtype=dtype, device=device) if need else None
            for need, (like, dtype) in zip(needs, ctx.like)
        ]
        if not any(needs):
            return (None,) * 7
        native, size = _feed_forward_backward_plan(
            shape, grad_stride, needs[1] + 2 * needs[2] + 4 * needs[3]
        )
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        status = hip._launch(
            library.lsso_hip_feed_forward_backward, device,
            native, flat_grad.data_ptr(), grad_stride, flat.data_ptr(), *pointers, mask_ptr, gates.data_ptr(), product.data_ptr(),
            *[None if grad is None else grad.data_ptr() for grad in grads], workspace.data_ptr(), size,
        )
        hip._check(status, library)
        return (*grads, None, None, None)


def gated_feed_forward(
    x: torch.Tensor,
    gate_weight: torch.Tensor,
    up_weight: torch.Tensor,
    down_weight: torch.Tensor,
    *,
    activation: str = "silu",
    row_mask: torch.Tensor | None = None,
    fine_factors: bool = True,
) -> torch.Tensor:
    """Gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) Wd^T.

    x: [..., K] float16/bfloat16; gate_weight, up_weight: [F, K]; down_weight:
    [N, F]; all three of x's type or all float32 (rounded to x's type once per
    call); y: contiguous [..., N] of x's type.  ``activation``: "silu" (g *
    sigmoid(g)) or "gelu" (g * Phi(g), exact).  ``row_mask`` (bool,
    x.shape[:-1]): the rows it excludes give zeros and reach no gradient,
    whatever they hold.

    Products accumulate in FP32 from 16-bit operands; the product act(g) * u
    is rounded to x's type once (so in float16 it must stay below 65,504); of up
    to 32 rows y's product takes it in two 16-bit parts.  Differentiable (first
    order) in x and the weights, deterministically.  For the backward u * act'(g)
    and act(g) are kept: with ``fine_factors`` as FP32 values rounded to their
    upper 20 bits for bfloat16 and 24 for float16 (7 F and 8 F bytes per row with
    the product), else rounded to x's type (6 F bytes; in float16 they must then
    stay below 65,504 too, and gradients of both types are off by sqrt(3) instead
    of sqrt(2) roundings of their own)."""

    hip = _hip()
    hip.require_available()
    _without_tangents(x, gate_weight, up_weight, down_weight)
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA (ROCm device) tensor")
    if x.dtype not in _HALF_CODES:
        raise TypeError(f"the feed-forward block supports float16 and bfloat16 x, got {x.dtype}")
    weights = (gate_weight, up_weight, down_weight)
    if x.dim() == 0 or any(w.dim() != 2 for w in weights):
        raise ValueError("x must have at least one dimension and the weights two")
    dtype = gate_weight.dtype
    if dtype not in (x.dtype, torch.float32) or up_weight.dtype != dtype or down_weight.dtype != dtype:
        raise TypeError(f"the weights must all be {x.dtype} or all float32")
    hidden, in_features = gate_weight.shape
    if (
        x.shape[-1] != in_features or up_weight.shape != gate_weight.shape or down_weight.shape[1] != hidden
        or hidden == 0 or in_features == 0 or down_weight.shape[0] == 0
    ):
        raise ValueError(
            "x [..., K], gate_weight and up_weight [F, K] and down_weight [N, F] must agree, got "
            f"{list(x.shape)}, {list(gate_weight.shape)}, {list(up_weight.shape)} and {list(down_weight.shape)}"
        )
    kind = _ACTIVATIONS.get(activation)
    if kind is None:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    for name, value in zip(("gate_weight", "up_weight", "down_weight"), weights):
        _on_device(value, name, x.device)
    if torch.is_grad_enabled() and (x.requires_grad or any(w.requires_grad for w in weights)):
        return _FeedForward.apply(x, *weights, kind, row_mask, bool(fine_factors))
    return _feed_forward_launch(x, *weights, kind, row_mask, False)[0]


__all__ = ["dropout_add", "embedding", "gated_feed_forward"]
