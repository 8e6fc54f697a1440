"""
Fused host-level operators with the signatures of nunchaku/ops/fused.py:15-253: each is a short sequence of
kernel launches (quantizer, GEMM with a fused epilogue, second GEMM).
"""

from __future__ import annotations

import torch

from .gemm import svdq_gemm_w4a4_cuda
from .quantize import ceil_divide


def _is_rmsnorm(m) -> bool:
    # torch.nn.RMSNorm, or diffusers' RMSNorm without a bias (fused.py:203-208)
    return m is None or (hasattr(m, "weight") and getattr(m, "bias", None) is None)


def fused_gelu_mlp(x: torch.Tensor, fc1, fc2, pad_size: int = 256) -> torch.Tensor:
    """
    ``fc2(gelu_tanh(fc1(x)))`` for two ``SVDQW4A4Linear`` layers: quantize, fc1 GEMM whose epilogue applies the GELU,
    the ``+0.171875`` shift and fc2's unsigned int4 quantisation and LoRA-down, then fc2's GEMM.  ``x (B, S, C_in)``.
    """
    from ..lora.batched import add_lora_batch, has_lora_batch

    batch_size, seq_len, channels = x.shape
    if has_lora_batch(fc1) or has_lora_batch(fc2):
        return _gelu_mlp_lora_batch(x, fc1, fc2, pad_size, add_lora_batch, has_lora_batch)
    x = x.view(batch_size * seq_len, channels)
    quantized_x, ascales, lora_act = fc1.quantize(x)
    batch_size_pad = ceil_divide(batch_size * seq_len, pad_size) * pad_size
    qout_act = torch.empty(batch_size_pad, fc1.out_features // 2, dtype=torch.uint8, device=x.device)
    if fc2.precision == "nvfp4":
        qout_ascales = torch.empty(fc1.out_features // 16, batch_size_pad, dtype=torch.float8_e4m3fn, device=x.device)
    else:
        qout_ascales = torch.empty(fc1.out_features // 64, batch_size_pad, dtype=x.dtype, device=x.device)
    qout_lora_act = torch.empty(batch_size_pad, fc2.proj_down.shape[1], dtype=torch.float32, device=x.device)
    svdq_gemm_w4a4_cuda(
        act=quantized_x, wgt=fc1.qweight, qout=qout_act, ascales=ascales, wscales=fc1.wscales, oscales=qout_ascales,
        lora_act_in=lora_act, lora_up=fc1.proj_up, lora_down=fc2.proj_down, lora_act_out=qout_lora_act, bias=fc1.bias,
        smooth_factor=fc2.smooth_factor, fp4=fc1.precision == "nvfp4", alpha=fc1.wtscale, wcscales=fc1.wcscales,
    )
    output = torch.empty(batch_size * seq_len, fc2.out_features, dtype=x.dtype, device=x.device)
    output = fc2.forward_quant(qout_act, qout_ascales, qout_lora_act, output=output)
    return output.view(batch_size, seq_len, -1)


def _gelu_mlp_lora_batch(x, fc1, fc2, pad_size, add_lora_batch, has_lora_batch):
    """:func:`fused_gelu_mlp` with adapters of the active requests: fc1's are added to its 16-bit output before the
    quantizer applies the GELU, fc2's see the GELU's 16-bit output."""
    from .triton.gemm_w4a4 import GELU_SHIFT, quantize_w4a4_act_fuse_lora

    batch_size, seq_len, _ = x.shape
    rows = batch_size * seq_len
    hidden = fc1(x).view(rows, fc1.out_features)
    if hidden.requires_grad:
        raise NotImplementedError("no backward pass: a fused operator")
    padded, fp4 = ceil_divide(rows, pad_size) * pad_size, fc2.precision == "nvfp4"
    act = torch.empty(padded, fc1.out_features // 2, dtype=torch.uint8, device=x.device)
    scales = torch.empty(fc1.out_features // (16 if fp4 else 64), padded, dtype=torch.float8_e4m3fn if fp4 else x.dtype, device=x.device)
    lora_act = torch.empty(padded, fc2.proj_down.shape[1], dtype=torch.float32, device=x.device)
    quantize_w4a4_act_fuse_lora(hidden, act, scales, fc2.proj_down, lora_act, fc2.smooth_factor, fp4=fp4, fuse_gelu=True,
                                shift_value=0.0 if fp4 else GELU_SHIFT, unsigned=not fp4)
    output = torch.empty(rows, fc2.out_features, dtype=x.dtype, device=x.device)
    output = fc2.forward_quant(act, scales, lora_act, output=output)
    if has_lora_batch(fc2):
        output = add_lora_batch(fc2, torch.nn.functional.gelu(hidden, approximate="tanh"), output, samples=batch_size, fused=True)
    return output.view(batch_size, seq_len, -1)


def interleave_swiglu_linear_(linear, up_first: bool = False) -> None:
    """
    Reorder a SwiGLU input projection's output rows in place (once) for :func:`fused_swiglu_mlp`: ``[gate | up]``
    becomes 16-row blocks of gate and up.  ``up_first=True`` is for projections whose output is ``[up | gate]``.
    """
    from .triton.native.w4a4 import interleave_swiglu

    assert linear.precision != "nvfp4" and linear.out_features % 64 == 0
    idx = interleave_swiglu(linear.out_features, linear.qweight.device)
    if up_first:
        idx = (idx + linear.out_features // 2) % linear.out_features
    with torch.no_grad():
        linear.qweight.data = linear.qweight.data[idx].contiguous()
        linear.wscales.data = linear.wscales.data[:, idx].contiguous()
        linear.proj_up.data = linear.proj_up.data[idx].contiguous()
        if linear.bias is not None:
            linear.bias.data = linear.bias.data[idx].contiguous()


def fused_swiglu_mlp(x: torch.Tensor, fc1, fc2, pad_size: int = 256) -> torch.Tensor:
    """``fc2(silu(gate) * up)`` with ``[gate | up] = fc1(x)``; ``fc1`` must have been interleaved (int4 only)."""
    from ..lora.batched import has_lora_batch
    from .triton.gemm_w4a4 import gemm_w4a4

    if has_lora_batch(fc1) or has_lora_batch(fc2):
        raise NotImplementedError("adapters of several requests on an interleaved SwiGLU projection")
    shape = x.shape
    x = x.reshape(-1, shape[-1])
    M = x.shape[0]
    quantized_x, ascales, lora_act = fc1.quantize(x, pad_size=pad_size)
    M_pad = quantized_x.shape[0]
    H = fc2.in_features
    qout_act = torch.empty(M_pad, H // 2, dtype=torch.uint8, device=x.device)
    qout_ascales = torch.empty(H // 64, M_pad, dtype=x.dtype, device=x.device)
    qout_lora_act = torch.empty(M_pad, fc2.proj_down.shape[1], dtype=torch.float32, device=x.device)
    gemm_w4a4(
        act=quantized_x, wgt=fc1.qweight, ascales=ascales, wscales=fc1.wscales, bias=fc1.bias, lora_act_in=lora_act,
        lora_up=fc1.proj_up, qout=qout_act, oscales=qout_ascales, smooth_factor=fc2.smooth_factor,
        lora_down=fc2.proj_down, lora_act_out=qout_lora_act, act_unsigned=fc1.act_unsigned, out_dtype=x.dtype,
        fuse_swiglu=True,
    )
    output = torch.empty(M, fc2.out_features, dtype=x.dtype, device=x.device)
    output = fc2.forward_quant(qout_act, qout_ascales, qout_lora_act, output=output)
    return output.view(*shape[:-1], fc2.out_features)


def fused_qkv_norm_rottary(x: torch.Tensor, proj, norm_q=None, norm_k=None, rotary_emb: torch.Tensor | None = None,
                           output=None, attn_tokens: int = 0):
    """
    Quantised QKV projection with per-head RMSNorm on Q and K and rotary embedding fused into the GEMM.
    ``rotary_emb`` is the natural ``(S, 64, 1, 2)`` fp32 table; with a batch ``B > 1`` the same ``S``-row table
    serves every batch element.  A tuple ``output`` (packed Q/K/V of the ``nunchaku-fp16`` processor) raises
    ``NotImplementedError`` as in the reference's natural-layout backend.
    """
    from ..lora.batched import add_lora_batch, has_lora_batch

    assert _is_rmsnorm(norm_q) and _is_rmsnorm(norm_k)
    batch_size, seq_len, channels = x.shape
    x = x.view(batch_size * seq_len, channels)
    quantized_x, ascales, lora_act = proj.quantize(x)
    if output is None:
        output = torch.empty(batch_size * seq_len, proj.out_features, dtype=x.dtype, device=x.device)
    common = dict(
        act=quantized_x, wgt=proj.qweight, ascales=ascales, wscales=proj.wscales, lora_act_in=lora_act,
        lora_up=proj.proj_up, bias=proj.bias, fp4=proj.precision == "nvfp4", alpha=proj.wtscale,
        wcscales=proj.wcscales, norm_q=norm_q.weight if norm_q is not None else None,
        norm_k=norm_k.weight if norm_k is not None else None, rotary_emb=rotary_emb,
    )
    if isinstance(output, tuple):
        assert len(output) == 3
        output_q, output_k, output_v = output
        svdq_gemm_w4a4_cuda(**common, out_q=output_q, out_k=output_k, out_v=output_v, attn_tokens=attn_tokens)
        return output_q, output_k, output_v
    if has_lora_batch(proj):
        # adapters of the active requests: they are added to the projection before Q and K are normalised and rotated
        from .triton.gemm_w4a4 import _apply_rmsnorm_rope_qk

        qk = {name: common.pop(name) for name in ("norm_q", "norm_k", "rotary_emb")}
        svdq_gemm_w4a4_cuda(**common, out=output)
        rows = output.view(batch_size * seq_len, proj.out_features)
        added = add_lora_batch(proj, x, rows, samples=batch_size, fused=True)
        if added is not rows:
            rows.copy_(added)
        if all(v is not None for v in qk.values()):
            _apply_rmsnorm_rope_qk(rows, qk["norm_q"], qk["norm_k"], qk["rotary_emb"])
        return output.view(batch_size, seq_len, -1)
    svdq_gemm_w4a4_cuda(**common, out=output)
    return output.view(batch_size, seq_len, -1)
