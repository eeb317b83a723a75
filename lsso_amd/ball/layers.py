"""Modules around the mixer: token embedding, gated feed-forward block, residual
dropout and group norm; and the causal mixer, which mixes each token with those
before it where LSSO mixes all of a sequence.

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


class GroupNorm(nn.Module):
    """y = act((x - mean) / sqrt(var + eps) * weight + bias) of [B, ..., C], statistics
    over the tokens that ``valid_mask`` leaves and the channels of each group; the
    other tokens are zeros.  [B * N, C] normalises each token by itself."""

    def __init__(self, groups: int, channels: int, *, eps: float = 1e-5, activation: str | None = None) -> None:
        super().__init__()
        _positive(groups=groups, channels=channels)
        if channels % groups:
            raise ValueError(f"groups must divide the channels, got {groups} and {channels}")
        if activation not in (None, "silu", "gelu"):
            raise ValueError(f"activation must be None, 'silu' or 'gelu', got {activation!r}")
        self.groups = groups
        self.eps = float(eps)
        self.activation = activation
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels))

    def forward(
        self, x: torch.Tensor, valid_mask: torch.Tensor | None = None, *, implementation: str = "reference"
    ) -> torch.Tensor:
        if _native(implementation):
            from . import hip

            path = hip.group_norm
        else:
            path = canonical.group_norm
        return path(
            x, self.groups, self.weight, self.bias, eps=self.eps, activation=self.activation, row_mask=valid_mask
        )

    def extra_repr(self) -> str:
        return f"{self.groups}, {self.weight.shape[0]}, eps={self.eps}, activation={self.activation}"


class CausalMixer(nn.Module):
    """Causal token mixing with a state of fixed size, for sequences that go on
    token by token:

        q, k, v = W_in x;  q, k turned by their positions;
        o = linear attention with a decay for each head;
        y = W_o act(group norm over each head of each token of o).

    ``forward`` takes whole sequences (training, prompts), ``step`` one token of
    each with the state in place.  Heads forget over ``shortest`` to ``longest``
    tokens.  Tokens that ``valid_mask`` excludes are as if they were not there, but
    for the positions of those behind them; their y is zero.  position_ids are
    0 .. N - 1 by default: a call that goes on from a state gives its own.
    ``frequencies``: float64 radians a position (``rotary_frequencies``); of half a
    head's features by default."""

    def __init__(
        self,
        dim: int,
        num_heads: int,
        *,
        kv_heads: int | None = None,
        frequencies: torch.Tensor | None = None,
        amplitude: float = 1.0,
        layout: str = "interleaved",
        activation: str | None = "silu",
        shortest: float = 8.0,
        longest: float = 1024.0,
        bias: bool = False,
    ) -> None:
        super().__init__()
        kv_heads = num_heads if kv_heads is None else kv_heads
        _positive(dim=dim, num_heads=num_heads, kv_heads=kv_heads)
        if dim % num_heads or num_heads % kv_heads:
            raise ValueError(f"num_heads must divide dim and kv_heads num_heads, got {dim}, {num_heads} and {kv_heads}")
        if not 1.0 < shortest <= longest:
            raise ValueError(f"shortest must be above 1 and at most longest, got {shortest} and {longest}")
        if layout not in ("interleaved", "half"):
            raise ValueError(f"layout must be 'interleaved' or 'half', got {layout!r}")
        self.num_heads, self.kv_heads, self.head_dim = num_heads, kv_heads, dim // num_heads
        if frequencies is None:
            frequencies = canonical.rotary_frequencies(max(2, self.head_dim // 4 * 2))
        if not 1 <= frequencies.shape[0] <= self.head_dim // 2:
            raise ValueError(f"frequencies must be 1 to {self.head_dim // 2}, got {frequencies.shape[0]}")
        self.layout, self.amplitude = layout, float(amplitude)
        device = torch.empty(0).device   # where the layers below are made
        frequencies = frequencies.detach().to(device=device, dtype=torch.float64, copy=True)
        self.register_buffer("frequencies", frequencies, persistent=False)
        self.register_buffer("log_decay", self._decays(num_heads, shortest, longest), persistent=False)
        self.w_in = nn.Linear(dim, (num_heads + 2 * kv_heads) * self.head_dim, bias=bias)
        self.norm = GroupNorm(num_heads, dim, activation=activation)
        self.w_o = nn.Linear(dim, dim, bias=bias)

    @staticmethod
    def _decays(heads: int, shortest: float, longest: float) -> torch.Tensor:
        spread = torch.arange(heads, dtype=torch.float64) / max(1, heads - 1)
        return torch.log1p(-1.0 / (shortest * (longest / shortest) ** spread)).float()

    def _apply(self, *arguments, **keywords):
        # Of a moved module only the device changes: both lose what they are for in a
        # type of fewer bits.  What the program wrote into them goes with them.
        fixed = {name: getattr(self, name) for name in ("frequencies", "log_decay")}
        result = super()._apply(*arguments, **keywords)
        device = self.w_o.weight.device
        for name, value in fixed.items():
            setattr(self, name, value.to(device))
        return result

    def initial_state(self, batch: int) -> torch.Tensor:
        """The state before the first token: float32 zeros [B, H, D, D]."""

        return torch.zeros(
            batch, self.num_heads, self.head_dim, self.head_dim, dtype=torch.float32, device=self.w_o.weight.device
        )

    def _paths(self, implementation: str):
        if _native(implementation):
            from . import hip

            def linear(x, layer, mask):
                return hip.linear(x, layer.weight, layer.bias, x.dtype, mask)

            return hip, linear

        def linear(x, layer, mask):
            y = canonical.linear(x, layer.weight, layer.bias, output_dtype=x.dtype)
            return y if mask is None else torch.where(mask[..., None], y, torch.zeros_like(y))

        return canonical, linear

    def _heads(self, projected: torch.Tensor, path, position_ids: torch.Tensor | None):
        """(query, key, value) [B, N, heads, head_dim], query and key turned."""

        split = projected.unflatten(-1, (-1, self.head_dim))
        q, k, v = split.split((self.num_heads, self.kv_heads, self.kv_heads), dim=-2)
        q, k = path.rotary(q, k, position_ids, self.frequencies, layout=self.layout, amplitude=self.amplitude)
        return q, k, v

    def forward(
        self,
        x: torch.Tensor,
        valid_mask: torch.Tensor | None = None,
        position_ids: torch.Tensor | None = None,
        *,
        state: torch.Tensor | None = None,
        return_state: bool = False,
        implementation: str = "reference",
    ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
        """y [B, N, dim] of x [B, N, dim], and with ``return_state`` the state behind it."""

        path, linear = self._paths(implementation)
        batch, length, dim = x.shape
        q, k, v = self._heads(linear(x, self.w_in, valid_mask), path, position_ids)
        mixed = path.linear_attention(
            q, k, v, self.log_decay, row_mask=valid_mask, initial_state=state, return_state=return_state
        )
        mixed, last = mixed if return_state else (mixed, None)
        normal = self.norm(
            mixed.reshape(batch * length, dim), None if valid_mask is None else valid_mask.reshape(-1),
            implementation=implementation,
        )
        y = linear(normal.view(batch, length, dim), self.w_o, valid_mask)
        return (y, last) if return_state else y

    def step(
        self,
        x: torch.Tensor,
        state: torch.Tensor,
        position_ids: torch.Tensor,
        valid_mask: torch.Tensor | None = None,
        *,
        implementation: str = "reference",
    ) -> torch.Tensor:
        """y [B, dim] of one token x [B, dim] of each sequence at position_ids [B]; its
        state is updated in place.  Sequences that ``valid_mask`` [B] excludes keep
        theirs.  Runs without gradients."""

        path, linear = self._paths(implementation)
        with torch.no_grad():
            projected = linear(x, self.w_in, valid_mask)
            q, k, v = self._heads(projected[:, None], path, position_ids[:, None])
            mixed = path.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], self.log_decay, state, row_mask=valid_mask)
            normal = self.norm(mixed.flatten(1), valid_mask, implementation=implementation)
            return linear(normal, self.w_o, valid_mask)

    def extra_repr(self) -> str:
        return f"num_heads={self.num_heads}, kv_heads={self.kv_heads}, layout={self.layout}"


__all__ = ["CausalMixer", "GatedFeedForward", "GroupNorm", "ResidualDropout", "TokenEmbedding"]
