"""Rotary positions for the KV-cache path: the frequencies (plain, or scaled for contexts longer
than a model was trained on), their table on the device, and the rotation as a differentiable
operation.  The reference's models take keys and queries that were rotated elsewhere; here a
cache can rotate the keys while it stores them (``PagedFP8KVCache(rope=...)``) and
``QuantizedRingAttention`` then rotates the queries."""
from __future__ import annotations

import math

import torch
import torch.autograd.forward_ad as fwAD

from .. import kv
from .._native import ensure_gpu


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None):
    """(float64 ``[rotary_dim / 2]`` angle per position of every pair, factor of the table).

    Pair i turns by base^(-2 i / rotary_dim) per position.  ``scaling``:

    * ``{"type": "linear", "factor": f}``: positions divided by f;
    * ``{"type": "ntk", "factor": f}``: the base times f^(d / (d - 2)), which leaves the fastest
      pair alone and divides the slowest one's angle by f;
    * ``{"type": "yarn", "factor": f, "original_positions": n}``: pairs that turn more than
      ``beta_fast`` (32) times within n positions are left alone, those that turn less than
      ``beta_slow`` (1) times are divided by f, a linear ramp over the pairs between; cosines
      and sines times ``attention_factor`` (0.1 ln f + 1).
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even")
    if not base > 1:
        raise ValueError("base must be above 1")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if scaling is None:
        return base ** (-2 * i / rotary_dim), 1.0
    kind, known = scaling.get("type"), {"type", "factor"}
    factor = float(scaling.get("factor", 0.0))
    if not factor >= 1:
        raise ValueError("scaling needs a factor of at least 1")
    if kind == "yarn":
        known |= {"original_positions", "beta_fast", "beta_slow", "attention_factor"}
    if kind not in ("linear", "ntk", "yarn") or set(scaling) - known:
        raise ValueError(f"unknown scaling {scaling!r}")
    if kind == "linear":
        return base ** (-2 * i / rotary_dim) / factor, 1.0
    if kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs a rotary_dim of at least 4")
        return (base * factor ** (rotary_dim / (rotary_dim - 2))) ** (-2 * i / rotary_dim), 1.0
    n = scaling.get("original_positions")
    if not n or n < 1:
        raise ValueError("yarn scaling needs original_positions")

    def pair(turns):  # the pair that turns so often within the original positions
        return rotary_dim * math.log(n / (2 * math.pi * turns)) / (2 * math.log(base))
    lo = max(math.floor(pair(scaling.get("beta_fast", 32.0))), 0)
    hi = min(math.ceil(pair(scaling.get("beta_slow", 1.0))), rotary_dim - 1)
    ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    freq = base ** (-2 * i / rotary_dim)
    mult = scaling.get("attention_factor")
    return freq * (1 - ramp) + freq / factor * ramp, 0.1 * math.log(factor) + 1 if mult is None else float(mult)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the kernel takes it: the caller has no say in how autograd lays a gradient out (one of a
    slice of a concatenation is a view that begins anywhere)."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class _Rotate(torch.autograd.Function):
    """A linear map: its gradient is the transposed one, its derivative along a tangent the map itself,
    both differentiable in their turn."""

    @staticmethod
    def forward(ctx, x, table, positions, interleaved, transpose):
        ctx.save_for_backward(table, positions)
        ctx.save_for_forward(table, positions)
        ctx.interleaved, ctx.transpose = interleaved, transpose
        return kv.rope(x, table, positions, interleaved=interleaved, transpose=transpose)

    @staticmethod
    def backward(ctx, grad):
        table, positions = ctx.saved_tensors
        return (_Rotate.apply(_rows(grad), table, positions, ctx.interleaved, not ctx.transpose),
                None, None, None, None)

    @staticmethod
    def jvp(ctx, tangent, *_):
        table, positions = ctx.saved_tensors
        return _Rotate.apply(_rows(tangent), table, positions, ctx.interleaved, ctx.transpose)


class RotaryPositions:
    """The rotary positions of one kind of head: ``rotary_dim`` (default: all ``head_dim``
    channels; a multiple of 16) turned in pairs (i, i + rotary_dim / 2), or (2 i, 2 i + 1) when
    ``interleaved``, for positions below ``max_positions``; ``base`` and ``scaling`` as in
    ``rotary_frequencies``.  ``table``: float32 ``[max_positions, rotary_dim]`` on the device."""

    def __init__(self, head_dim: int, max_positions: int, rotary_dim: int | None = None, base: float = 10000.0,
                 interleaved: bool = False, scaling: dict | None = None, device: torch.device | None = None):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if not 16 <= rotary_dim <= head_dim or rotary_dim % 16:
            raise ValueError("rotary_dim must be a multiple of 16, at most head_dim")
        if max_positions < 1:
            raise ValueError("max_positions must be positive")
        freq, factor = rotary_frequencies(rotary_dim, base, scaling)
        self.head_dim, self.rotary_dim, self.max_positions = head_dim, rotary_dim, int(max_positions)
        self.interleaved = bool(interleaved)
        self.table = kv.rope_table(freq.to(device or ensure_gpu()), self.max_positions, factor)

    def __call__(self, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """``x [n, H, head_dim]`` (bf16, f16, f32) at ``positions`` (int32 ``[n]``); differentiable
        in x, in reverse mode (the gradient is rotated back) and in forward mode.  ``kv.rope``
        itself is not: autograd does not see it."""
        if x.shape[-1] != self.head_dim:
            raise ValueError(f"x must have heads of {self.head_dim}")
        # (an autograd function costs a call 5 us of the host's time: only where one is needed)
        if torch.is_grad_enabled() and x.requires_grad or fwAD.unpack_dual(x).tangent is not None or \
                torch.jit.is_tracing():
            return _Rotate.apply(x, self.table, positions, self.interleaved, False)
        return kv.rope(x, self.table, positions, interleaved=self.interleaved)


__all__ = ["RotaryPositions", "rotary_frequencies"]
