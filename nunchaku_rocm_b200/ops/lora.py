"""
Low-rank adapters of many requests at once beside a shared projection (``csrc/lora.cu``).

The reference serves one LoRA set at a time (nunchaku/lora/runtime.py:475-535: the factors become part of the layer).  Here
every request of a batch names its own adapter, and the projection's output gets each row's ``scale (x D^T) U^T``.
:mod:`nunchaku_rocm_b200.lora` attaches stacks of adapters to layers; this is the operator under it.
"""

from __future__ import annotations

import torch

from .. import _lib as L

__all__ = ["lora_batched"]


def lora_batched(x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, offsets: torch.Tensor, adapters: torch.Tensor,
                 base: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, _impl: int = L.IMPL_AUTO) -> torch.Tensor:
    """
    ``out[t] = base[t] + scale[a] * (x[t] @ down[a]^T) @ up[a]^T`` with ``a`` the adapter of row ``t``'s request.

    ``x (..., K)`` and ``base (..., N)`` (zeros when ``None``) are taken as rows, bfloat16 or float16.  Request ``i`` has the
    rows ``offsets[i] .. offsets[i + 1] - 1`` (``offsets (requests + 1,)`` int32, not going down, zero-length requests
    allowed) and uses adapter ``adapters[i]`` (int32); a value outside ``0 .. A - 1``, -1 by convention, is no adapter.
    Rows outside every request have none either: ``out`` is ``base`` there.  Both index tensors stay on the device, so they
    may change between replays of a captured graph (as many requests as at capture).

    ``down (A, R, K)`` and ``up (A, N, R)`` are contiguous stacks of adapters (``R`` a multiple of 16 up to 128, ``K`` and
    ``N`` multiples of 8; smaller ranks are padded with zeros, see :func:`nunchaku_rocm_b200.lora.stack_loras`); ``scale
    (A,)`` is float32.  ``out`` may be given where no gradient is asked for; it may be ``base`` itself, and shares no memory
    with the inputs otherwise.  At most 65535 adapters, and ``rows / 64 + requests`` at most 65000.  A backward pass needs a
    workspace of ``R (K + N)`` floats for every request and every few hundred rows.

    Between the products ``scale * x @ down^T`` and its gradient keep 24 bits in bfloat16; in float16 22 bits and a power of two
    per row, so they may be far beyond float16 (what is below 2^-39 of the largest in a row, or of the rows that a gradient
    sums, is lost).

    Differentiable in ``x``, ``base``, ``down`` and ``up`` (not in ``scale``); gradients of adapters that several requests
    share are summed in a fixed order.
    """
    return L.binding().lora_batched(x, down, up, offsets, adapters, base, scale, out, _impl)
