"""Rotary positions: interleaved and half layouts, part of the head, scaled frequencies.

``y = R(p) x``: pair ``i`` of a head is turned by the angle ``p * inv_freq[i]``
and multiplied by ``amplitude``.  ``layout="interleaved"`` pairs dimensions
``(2i, 2i + 1)`` (the layout of every model here, `src/titans/attention.py:107-132`),
``"half"`` pairs ``(i, i + n)`` with ``n = len(inv_freq)``; dimensions from
``2n`` on are copied.  The angle is formed in fp64, so positions of millions of
tokens keep their phase; cos and sin are fp32, and the result is rounded once
to the input's type.  The backward pass is the rotation by the opposite angle
(``csrc/rope.cu`` runs both).
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from ._ext import ext, want_kernels

LAYOUTS = ("interleaved", "half")
SCALINGS = ("none", "linear", "ntk", "yarn")


def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                     original_max_position: int = 8192, fast_turns: float = 32.0, slow_turns: float = 1.0,
                     device=None) -> tuple[torch.Tensor, float]:
    """``(inv_freq [rotary_dim / 2] fp32, amplitude)`` for :func:`rotary_embedding`.

    * ``none``: ``base ** (-2i / rotary_dim)``;
    * ``linear``: the same divided by ``factor`` (positions interpolated);
    * ``ntk``: ``base * factor ** (rotary_dim / (rotary_dim - 2))`` as base, which
      leaves the fastest pair alone and stretches the slowest by ``factor``;
    * ``yarn``: pairs that turn at least ``fast_turns`` times within
      ``original_max_position`` tokens keep their frequency, pairs below
      ``slow_turns`` are divided by ``factor``, those between are blended
      linearly in their number of turns; amplitude ``0.1 ln(factor) + 1``.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, not {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, not {scaling!r}")
    if not factor >= 1.0:
        raise ValueError(f"factor must be at least 1, not {factor}")
    if not fast_turns > slow_turns:
        raise ValueError("fast_turns must be greater than slow_turns")
    amplitude = 1.0
    if scaling == "ntk":
        base = base * factor ** (rotary_dim / max(rotary_dim - 2, 1))
    f = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        turns = original_max_position * f / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    return f.float().to(device), amplitude


def rotary_embedding_reference(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                               layout: str = "interleaved", amplitude: float = 1.0) -> torch.Tensor:
    """PyTorch restatement (differentiable in ``x``)."""
    n = inv_freq.numel()
    wide = x.double() if x.dtype == torch.float64 else x.float()
    angle = positions.double()[..., None] * inv_freq.double()
    if positions.dim() == 1:
        angle = angle[None]
    cos = (amplitude * angle.cos()).to(wide.dtype)[:, :, None]
    sin = (amplitude * angle.sin()).to(wide.dtype)[:, :, None]
    if layout == "interleaved":
        a, b = wide[..., 0:2 * n:2], wide[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = wide[..., :n], wide[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, wide[..., 2 * n:]], dim=-1).to(x.dtype)


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, inv_freq, half, amplitude, backward):
        ctx.save_for_backward(positions, inv_freq)
        ctx.save_for_forward(positions, inv_freq)
        ctx.args = (half, amplitude, backward)
        return ext().rotary_embedding(x, positions, inv_freq, half, amplitude, backward)

    @staticmethod
    def backward(ctx, dy):
        positions, inv_freq = ctx.saved_tensors
        half, amplitude, backward = ctx.args
        return _RotaryFn.apply(dy, positions, inv_freq, half, amplitude, not backward), None, None, None, None, None

    @staticmethod
    def jvp(ctx, dx, *_):  # the rotation is linear
        return _RotaryFn.apply(dx, *ctx.saved_tensors, *ctx.args)


def rotary_embedding(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                     layout: str = "interleaved", amplitude: float = 1.0,
                     use_kernels: bool | None = None) -> torch.Tensor:
    """Rotate the first ``2 * len(inv_freq)`` dimensions of every head of ``x`` [B, T, H, d].

    ``positions``: int64 [T] (shared by the batch) or [B, T]; ``inv_freq``,
    ``amplitude``: from :func:`rope_frequencies`.  ``x`` may have any strides
    (a slice of a fused projection needs no copy); the result is contiguous.
    Differentiable in ``x``, backwards (any number of times) and forwards.
    """
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {LAYOUTS}, not {layout!r}")
    if x.dim() != 4:
        raise ValueError(f"x must be [B, T, H, d], not {tuple(x.shape)}")
    if positions.dtype != torch.int64:
        raise TypeError(f"positions must be int64, not {positions.dtype}")
    if positions.shape not in (x.shape[1:2], x.shape[:2]):
        raise ValueError(f"positions must be [T] or [B, T] of {tuple(x.shape)}, not {tuple(positions.shape)}")
    if inv_freq.dim() != 1 or 2 * inv_freq.numel() > x.shape[-1]:
        raise ValueError(f"inv_freq must be [n] with 2n <= {x.shape[-1]}, not {tuple(inv_freq.shape)}")
    if want_kernels(x, use_kernels):
        inv_freq = inv_freq.float().contiguous()
        if (x.requires_grad and torch.is_grad_enabled()) or forward_ad.unpack_dual(x).tangent is not None:
            return _RotaryFn.apply(x, positions, inv_freq, layout == "half", float(amplitude), False)
        return ext().rotary_embedding(x, positions, inv_freq, layout == "half", float(amplitude), False)
    return rotary_embedding_reference(x, positions, inv_freq, layout, amplitude)


__all__ = ["rope_frequencies", "rotary_embedding", "rotary_embedding_reference", "LAYOUTS", "SCALINGS"]
