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


def _rows_ok(t: torch.Tensor) -> bool:
    """Whether the kernel can write ``t (..., C)`` in place: rows evenly strided and apart, each on a 16-byte boundary."""
    if t.data_ptr() % 16 or t.stride(-1) != 1:
        return False
    run, step = 1, t.shape[-1]
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size != 1:
            if run == 1:
                step = stride
            elif stride != run * step:
                return False
            run *= size
    return step % 8 == 0 and (step >= t.shape[-1] or run <= 1)


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

    Differentiable in ``x``, ``base``, ``down`` and ``up`` (not in ``scale``); gradients of adapters that several requests
    share are summed in a fixed order.
    """
    dt = x.dtype
    if (dt not in L.DTYPE_CODE or down.dtype != dt or up.dtype != dt or (base is not None and base.dtype != dt)
            or (out is not None and out.dtype != dt)):
        raise ValueError("x, base, down, up and out must share one dtype, bfloat16 or float16")
    if down.dim() != 3 or up.dim() != 3 or down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2] or down.shape[0] == 0:
        raise ValueError(f"down must be (A, R, K) and up (A, N, R); got {tuple(down.shape)} and {tuple(up.shape)}")
    A, R, K = down.shape
    N = up.shape[1]
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"x must be (..., {K}), got {tuple(x.shape)}")
    out_shape = (*x.shape[:-1], N)
    for name, t in (("base", base), ("out", out)):
        if t is not None and t.shape != out_shape:
            raise ValueError(f"{name} must be {out_shape}, got {tuple(t.shape)}")
    if R == 0 or R % 16 or R > L.LORA_MAX_RANK or K == 0 or K % 8 or N == 0 or N % 8:
        raise NotImplementedError(f"rank {R} must be a multiple of 16 up to {L.LORA_MAX_RANK}, K={K} and N={N} multiples of 8")
    if offsets.dtype != torch.int32 or adapters.dtype != torch.int32 or offsets.dim() != 1 or adapters.dim() != 1:
        raise ValueError("offsets and adapters must be 1-D int32 tensors")
    if offsets.shape[0] != adapters.shape[0] + 1:
        raise ValueError(f"{adapters.shape[0]} adapters need {adapters.shape[0] + 1} offsets, got {offsets.shape[0]}")
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != (A,)):
        raise ValueError(f"scale must be ({A},) float32, got {tuple(scale.shape)} {scale.dtype}")
    grad = torch.is_grad_enabled()
    if grad and scale is not None and scale.requires_grad:
        raise ValueError("lora_batched has no gradient for scale")
    if out is not None and not _rows_ok(out):
        raise ValueError("out must have evenly strided rows on 16-byte boundaries that do not overlap")
    L.require_cuda(x, down, up, offsets, adapters, base, scale, out)
    if out is not None and grad and (out.requires_grad or x.requires_grad or down.requires_grad or up.requires_grad or (base is not None and base.requires_grad)):
        raise ValueError("out cannot be given where a gradient is asked for")
    return L.binding().lora_batched(
        x, down.contiguous(), up.contiguous(), offsets.contiguous(), adapters.contiguous(), base,
        None if scale is None else scale.contiguous(), out, _impl, L.status_word(x.device).data_ptr())
