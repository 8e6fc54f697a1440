"""
Rotary positions with several axes (time, height, width), straight from position ids (``csrc/rotary.cu``).

The fused QKV projection takes its rotation from a table (:func:`nunchaku_rocm_b200.models.embeddings.flux_pos_embed`);
:func:`rotary_table` makes that table in one launch, and :func:`rotary_axes` rotates Q and K that come from elsewhere (a
16-bit attention layer, a training step) without one.  The reference builds tables
with torch operators (``rope`` / ``NunchakuFluxPosEmbed``, nunchaku/models/embeddings.py:11-50, 74-97).
"""

from __future__ import annotations

import functools

import torch

from .. import _lib as L

__all__ = ["rotary_axes", "rotary_table"]


@functools.lru_cache(maxsize=64)
def _ladder(axes_dim: tuple, theta: float):
    """The rates of the axes' pairs, made once per (axes, theta)."""
    if not 1 <= len(axes_dim) <= L.ROTARY_MAX_AXES:
        raise ValueError(f"1 to {L.ROTARY_MAX_AXES} axes, got {len(axes_dim)}")
    if any(d <= 0 or d % 2 for d in axes_dim) or sum(axes_dim) > 2 * L.ROTARY_MAX_PAIRS:
        raise ValueError(f"the axes' channels must be even, positive and at most {2 * L.ROTARY_MAX_PAIRS} together: {axes_dim}")
    return L.binding().Ladder(axes_dim, theta)


def rotary_axes(q: torch.Tensor, k: torch.Tensor | None, ids: torch.Tensor, axes_dim, theta: float = 10000.0,
                interleaved: bool = True, inverse: bool = False):
    """
    Rotate ``q (B, S, H, D)`` and ``k (B, S, Hk, D)`` by the positions ``ids (S, axes)`` or ``(B, S, axes)``; returns new
    contiguous tensors ``(q', k')``, or ``q'`` alone when ``k`` is ``None``.  Differentiable in ``q`` and ``k``.

    Axis ``a`` owns ``axes_dim[a]`` channels of every head, in order; its pair ``j`` turns by
    ``ids[..., a] * theta ** (-2 j / axes_dim[a])`` radians (angles in fp64, the rotation in fp32, one rounding).  A pair is
    two neighbouring channels, or with ``interleaved=False`` channels ``j`` and ``j + R / 2`` of the ``R = sum(axes_dim)``
    rotary ones.  Channels behind those pass through.  ``inverse`` rotates back.

    bfloat16, float16 or float32; any strides; ``ids`` float32, float64, int32 or int64.
    """
    return L.binding().rotary_axes(q, k, ids, _ladder(tuple(axes_dim), float(theta)), not interleaved, inverse)


def rotary_table(ids: torch.Tensor, axes_dim, theta: float = 10000.0) -> torch.Tensor:
    """
    The ``(sin, cos)`` table of ``ids (S, axes)`` -> ``(S, sum(axes_dim) / 2, 1, 2)`` fp32 (or with a leading ``B``): what
    the fused QKV epilogue reads as ``rotary_emb``, with the angles of :func:`rotary_axes`.
    """
    return L.binding().rotary_table(ids, _ladder(tuple(axes_dim), float(theta)))
