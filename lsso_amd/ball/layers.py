"""Modules around the mixer: token embedding, gated feed-forward block and
residual dropout.

Like ``LSSO``, each takes ``implementation``: the device-agnostic PyTorch path
("reference", the default) or the gfx950 native path ("hip", or "cuda" as the
same request), which never falls back; and parameters are float32 whatever
type the activations have."""

from __future__ import annotations

import torch
import torch.nn as nn

from . import reference as canonical

_NATIVE_IMPLEMENTATIONS = ("hip", "cuda")


def _native(implementation: str) -> bool:
    if implementation in _NATIVE_IMPLEMENTATIONS:
        return True
    if implementation != "reference":
        raise ValueError(f"implementation must be 'reference', 'hip' or 'cuda', got {implementation!r}")
    return False


def _positive(**sizes: int) -> None:
    for name, value in sizes.items():
        if not isinstance(value, int) or isinstance(value, bool):
            raise TypeError(f"{name} must be an integer, got {type(value).__name__}")
        if value <= 0:
            raise ValueError(f"{name} must be positive, got {value}")


class TokenEmbedding(nn.Module):
    """x = scale * weight[tokens] in ``dtype``, the input of a stack of mixers."""

    def __init__(self, vocabulary: int, dim: int, *, scale: float = 1.0, padding_index: int | None = None) -> None:
        super().__init__()
        _positive(vocabulary=vocabulary, dim=dim)
        if padding_index is not None and not 0 <= padding_index < vocabulary:
            raise ValueError(f"padding_index must be a row of the table, got {padding_index}")
        self.scale = float(scale)
        self.padding_index = padding_index
        self.weight = nn.Parameter(torch.randn(vocabulary, dim) * (dim**-0.5))
        if padding_index is not None:
            with torch.no_grad():
                self.weight[padding_index].zero_()

    def forward(
        self,
        tokens: torch.Tensor,
        valid_mask: torch.Tensor | None = None,
        *,
        dtype: torch.dtype | None = None,
        implementation: str = "reference",
    ) -> torch.Tensor:
        if _native(implementation):
            from . import hip

            path = hip.embedding
        else:
            path = canonical.embedding
        return path(
            tokens, self.weight, scale=self.scale, row_mask=valid_mask, padding_index=self.padding_index,
            output_dtype=dtype,
        )

    def extra_repr(self) -> str:
        return f"{self.weight.shape[0]}, {self.weight.shape[1]}, scale={self.scale}, padding_index={self.padding_index}"


class GatedFeedForward(nn.Module):
    """y = (act(x gate^T) * (x up^T)) down^T, the channel mixing beside LSSO's
    token mixing; rows that ``valid_mask`` excludes are zeros."""

    def __init__(self, dim: int, hidden: int, *, activation: str = "silu") -> None:
        super().__init__()
        _positive(dim=dim, hidden=hidden)
        if activation not in ("silu", "gelu"):
            raise ValueError(f"activation must be 'silu' or 'gelu', got {activation!r}")
        self.activation = activation
        self.gate = nn.Linear(dim, hidden, bias=False)
        self.up = nn.Linear(dim, hidden, bias=False)
        self.down = nn.Linear(hidden, dim, bias=False)

    def forward(
        self, x: torch.Tensor, valid_mask: torch.Tensor | None = None, *, implementation: str = "reference"
    ) -> torch.Tensor:
        if _native(implementation):
            from . import hip

            path = hip.gated_feed_forward
        else:
            path = canonical.gated_feed_forward
        return path(
            x, self.gate.weight, self.up.weight, self.down.weight, activation=self.activation, row_mask=valid_mask
        )

    def extra_repr(self) -> str:
        return f"activation={self.activation}"


class ResidualDropout(nn.Module):
    """residual + dropout(x), with a mask that is a function of ``seed`` and
    ``offset`` alone; in evaluation the plain sum (on the native path the same
    kernel, with nothing dropped, and the same arguments refused)."""

    def __init__(self, probability: float) -> None:
        super().__init__()
        from .block import dropout_threshold

        self.probability = float(probability)
        self._threshold = dropout_threshold(self.probability)

    def forward(
        self,
        x: torch.Tensor,
        residual: torch.Tensor | None = None,
        *,
        seed: int | torch.Tensor,
        offset: int = 0,
        implementation: str = "reference",
    ) -> torch.Tensor:
        if _native(implementation):
            from . import hip

            return hip.dropout_add(x, residual, self.probability if self.training else 0.0, seed, offset)
        if not self.training:
            return x if residual is None else residual + x
        if isinstance(seed, torch.Tensor):
            key, step = (int(value) for value in seed.tolist())
            seed, offset = key, offset + step
        return canonical.dropout_add(x, residual, self._threshold, seed, offset)

    def extra_repr(self) -> str:
        return f"probability={self.probability}"


__all__ = ["GatedFeedForward", "ResidualDropout", "TokenEmbedding"]
