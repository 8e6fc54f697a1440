"""
Low-rank adapters of many requests at once beside a shared projection (``csrc/lora.cu``).

The reference serves one LoRA set at a time (nunchaku/lora/runtime.py:475-535: the factors become part of the layer).  Here
every request of a batch names its own adapter, and the projection's output gets each row's ``scale (x D^T) U^T``.
:mod:`nunchaku_rocm_b200.lora` attaches stacks of adapters to layers; this is the operator under it.
"""

from __future__ import annotations

import torch

from .. import _lib as L
from .elementwise import _strided_rows

__all__ = ["lora_batched"]


def _aligned_rows(t: torch.Tensor):
    """``t (..., C)`` with rows evenly strided on 16-byte boundaries, and their stride (a copy only if they are not)."""
    t, stride = _strided_rows(t)
    if stride % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        stride = t.shape[-1]
    return t, stride


def _args(T, K, N, down, up, offsets, adapters, scale, impl):
    a = L.LoraArgs()
    a.down, a.up = down.data_ptr(), up.data_ptr()
    a.offsets, a.adapters = offsets.data_ptr(), adapters.data_ptr()
    if scale is not None:
        a.scale = scale.data_ptr()
    a.T, a.K, a.N, a.R, a.A = T, K, N, down.shape[1], down.shape[0]
    a.requests, a.dtype, a.impl = adapters.shape[0], L.DTYPE_CODE[down.dtype], impl
    a.status = L.status_word(down.device).data_ptr()
    return a


def _forward(x, base, down, up, offsets, adapters, scale, out, impl):
    """``out`` and the two 16-bit parts of ``scale x down^T``; the arguments are checked already."""
    K, N = down.shape[2], up.shape[1]
    T = x.numel() // K
    h = x.new_empty((2, T, down.shape[1]))
    if T == 0:
        return h
    x, stride_x = _aligned_rows(x)
    a = _args(T, K, N, down, up, offsets, adapters, scale, impl)
    a.x, a.stride_x = x.data_ptr(), stride_x
    if base is not None:
        base, a.stride_base = _aligned_rows(base)
        a.base = base.data_ptr()
    a.out, a.stride_out = out.data_ptr(), _strided_rows(out)[1]
    a.h = h.data_ptr()
    L.launch(L.lib().nb_lora_forward, "lora_batched", x, a)
    return h


class _LoraBatched(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, base, down, up, offsets, adapters, scale, impl):
        out = x.new_empty((*x.shape[:-1], up.shape[1]))
        h = _forward(x, base, down, up, offsets, adapters, scale, out, impl)
        need = ctx.needs_input_grad
        ctx.save_for_backward(x if need[2] else None, down, up, h if need[3] else None, offsets, adapters, scale)
        ctx.x_shape, ctx.impl = x.shape, impl
        return out

    @staticmethod
    @L.once_differentiable
    def backward(ctx, dy):
        x, down, up, h, offsets, adapters, scale = ctx.saved_tensors
        need_x, need_base, need_down, need_up = ctx.needs_input_grad[:4]
        new = down.new_empty
        dx = new(ctx.x_shape) if need_x else None
        ddown = new(down.shape) if need_down else None
        dup = new(up.shape) if need_up else None
        K, N = down.shape[2], up.shape[1]
        T = dy.numel() // N
        if T == 0:
            for t in (ddown, dup):
                if t is not None:
                    t.zero_()
        elif need_x or need_down or need_up:
            rows, stride_dy = _aligned_rows(dy)
            a = _args(T, K, N, down, up, offsets, adapters, scale, ctx.impl)
            a.dy, a.stride_dy = rows.data_ptr(), stride_dy
            if need_x:
                a.dx = dx.data_ptr()
            if need_down:
                x, a.stride_x = _aligned_rows(x)
                a.x, a.ddown = x.data_ptr(), ddown.data_ptr()
            if need_x or need_down:
                g = new((2, T, down.shape[1]))
                a.g = g.data_ptr()
            if need_up:
                a.h, a.dup = h.data_ptr(), dup.data_ptr()
            lib = L.lib()
            n = lib.nb_lora_workspace_bytes(a) if need_down or need_up else 0
            if n:
                ws = new((n + 1) // 2)
                a.workspace, a.workspace_bytes = ws.data_ptr(), n
            L.launch(lib.nb_lora_backward, "lora_batched backward", down, a)
        return dx, (dy if need_base else None), ddown, dup, None, None, None, None


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
    (A,)`` is float32.  ``out`` may be given where no gradient is asked for, and may be ``base``.

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
    if out is not None:
        rows, stride = _strided_rows(out)
        if rows is not out or stride % 8 or out.data_ptr() % 16:
            raise ValueError("out must have evenly strided rows on 16-byte boundaries")
    L.require_cuda(x, down, up, offsets, adapters, base, scale, out)
    down, up, offsets, adapters = down.contiguous(), up.contiguous(), offsets.contiguous(), adapters.contiguous()
    scale = None if scale is None else scale.contiguous()
    if grad and (x.requires_grad or down.requires_grad or up.requires_grad or (base is not None and base.requires_grad)):
        if out is not None:
            raise ValueError("out cannot be given where a gradient is asked for")
        return _LoraBatched.apply(x, base, down, up, offsets, adapters, scale, _impl)
    if out is None:
        out = x.new_empty((*x.shape[:-1], N))
    _forward(x, base, down, up, offsets, adapters, scale, out, _impl)
    return out
