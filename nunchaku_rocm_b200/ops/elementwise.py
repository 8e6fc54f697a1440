"""
The element-wise steps around the quantised linears of a DiT block, fused to one pass over HBM each
(``csrc/elementwise.cu``).  The reference runs them as torch operators: ``NunchakuAdaLayerNormZero``
(nunchaku/models/normalization.py:60-159) and the gated residuals of the transformer blocks
(nunchaku/models/transformers/transformer_flux_v2.py:174-343).

:func:`layer_norm` is a layer norm with its backward pass (``csrc/norm.cu``), for norms with a weight and a bias and for
training the adaptive ones; :func:`layernorm_modulate` uses the same backward pass where gradients are asked for.
"""

from __future__ import annotations

import ctypes as C

import torch

from .. import _lib as L

__all__ = ["layernorm_modulate", "gated_residual", "layer_norm"]


def _bind():
    lib = L.lib()
    if not getattr(lib, "_ew_bound", False):
        lib.nb_layernorm_modulate.argtypes = [C.c_void_p] * 4 + [C.c_int32] * 3 + [C.c_int64] * 4 + [C.c_float, C.c_float, C.c_int32, C.c_void_p]
        lib.nb_gated_residual.argtypes = [C.c_void_p] * 5 + [C.c_int32] * 3 + [C.c_int64] * 6 + [C.c_int32, C.c_void_p]
        lib._ew_bound = True
    return lib


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``(B, T, dim)`` as a view whose rows are evenly strided (a copy only if they are not)."""
    B, T, D = x.shape
    if x.stride(2) != 1 or (B > 1 and x.stride(0) != T * x.stride(1)) or x.stride(1) % 8 or x.data_ptr() % 16:
        x = x.contiguous()
    return x


def layernorm_modulate(x: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor, scale_add: float = 0.0,
                       eps: float = 1e-6) -> torch.Tensor:
    """``LayerNorm(x) * (scale[:, None] + scale_add) + shift[:, None]`` for ``x (B, T, dim)``, ``scale / shift (B, dim)``
    (any strides), no affine; rounded to the dtype where ``layer_norm``, ``+``, ``*``, ``+`` of the reference round.
    Differentiable in ``x``, ``scale`` and ``shift``."""
    B, T, D = x.shape
    if D % 1024 or D > 4096:
        return torch.nn.functional.layer_norm(x, (D,), eps=eps) * (scale + scale_add)[:, None] + shift[:, None]
    if torch.autograd.forward_ad._current_level >= 0 and any(map(L.binding().has_tangent, (x, scale, shift))):
        raise NotImplementedError("layernorm_modulate has no forward-mode derivative")
    if torch.is_grad_enabled() and (x.requires_grad or scale.requires_grad or shift.requires_grad):
        return _LayerNormModulate.apply(x, scale, shift, scale_add, eps)
    return _layernorm_modulate(x, scale, shift, scale_add, eps)


def _layernorm_modulate(x, scale, shift, scale_add, eps):
    B, T, D = x.shape
    dev = L.require_cuda(x, scale, shift)
    x = _rows(x)
    assert scale.shape == (B, D) and shift.shape == (B, D) and scale.stride() == shift.stride() and scale.dtype == x.dtype == shift.dtype
    out = torch.empty(B, T, D, dtype=x.dtype, device=dev)
    with torch.cuda.device(dev):
        L.check(
            _bind().nb_layernorm_modulate(L.ptr(x), L.ptr(scale), L.ptr(shift), L.ptr(out), B * T, T, D, x.stride(1), D,
                                          scale.stride(0), scale.stride(1), float(scale_add), float(eps), L.DTYPE_CODE[x.dtype],
                                          L.stream_of(out)),
            "layernorm_modulate",
        )
    return out


def gated_residual(x: torch.Tensor, gate: torch.Tensor, y: torch.Tensor, y2: torch.Tensor | None = None) -> torch.Tensor:
    """``x + gate[:, None] * (y [+ y2])`` for ``x, y, y2 (B, T, dim)``, ``gate (B, dim)`` (any strides); rounded to the dtype where the reference's ``+``, ``*``, ``+`` round."""
    B, T, D = x.shape
    dev = L.require_cuda(x, gate, y)
    assert D % 8 == 0 and y.shape == x.shape and gate.shape == (B, D) and gate.dtype == x.dtype == y.dtype
    x, y = _rows(x), _rows(y)
    if y2 is not None:
        assert y2.shape == x.shape and y2.dtype == x.dtype
        y2 = _rows(y2)
    out = torch.empty(B, T, D, dtype=x.dtype, device=dev)
    with torch.cuda.device(dev):
        L.check(
            _bind().nb_gated_residual(L.ptr(x), L.ptr(gate), L.ptr(y), L.ptr(y2) if y2 is not None else None, L.ptr(out), B * T, T,
                                      D, x.stride(1), y.stride(1), y2.stride(1) if y2 is not None else 0, D, gate.stride(0),
                                      gate.stride(1), L.DTYPE_CODE[x.dtype], L.stream_of(out)),
            "gated_residual",
        )
    return out


class _LayerNormModulate(torch.autograd.Function):
    """:func:`layernorm_modulate` as it is without gradients, and the backward pass of the function that it rounds."""

    @staticmethod
    def forward(ctx, x, scale, shift, scale_add, eps):
        ctx.save_for_backward(x, scale, shift)
        ctx.consts = eps, scale_add
        return _layernorm_modulate(x, scale, shift, scale_add, eps)

    @staticmethod
    @L.once_differentiable
    def backward(ctx, dy):
        eps, scale_add = ctx.consts
        x, scale, shift = ctx.saved_tensors
        stats = x.new_empty((2, x.numel() // x.shape[-1]), dtype=torch.float32)
        b = L.binding()
        b.layer_norm_forward(x, None, None, eps, 0.0, None, stats)
        return (*b.layer_norm_backward(x, scale, shift, stats, dy, eps, scale_add, *ctx.needs_input_grad[:3]), None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-6,
               weight_add: float = 0.0) -> torch.Tensor:
    """
    ``(x - mean) / sqrt(var + eps) * (weight + weight_add) + bias`` over the last dimension of ``x (..., D)``, computed in
    fp32 and rounded once to ``x``'s dtype (bfloat16, float16 or float32).  Differentiable in ``x``, ``weight`` and ``bias``.

    ``weight`` and ``bias`` are ``(D,)``, or ``(B, D)`` for ``x (B, T, D)`` (one row per sample, as an adaptive norm's scale
    and shift, then with ``weight_add=1``), both of ``x``'s dtype or both float32; either may be ``None``.  Their gradients
    are summed over the rows in fp32, in a fixed order.  ``D`` is at most 16384, ``B`` with a row per sample at most 65535.
    """
    return L.binding().layer_norm(x, weight, bias, eps, weight_add)
