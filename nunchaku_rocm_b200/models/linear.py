"""
Parameter containers of the two quantised linear layers, with the attribute names, shapes and method
signatures of the reference's ``nunchaku/models/linear.py`` (``SVDQW4A4Linear`` :13-275,
``AWQW4A16Linear`` :278-415).  They are callers of the operators: every forward is two (or one) kernel
launches through :mod:`nunchaku_rocm_b200.ops`.  Parameters are in the natural layout
(:func:`nunchaku_rocm_b200.ops.triton.layout.convert_svdq_linear_to_natural_layout` converts a checkpoint).
"""

from __future__ import annotations

import torch
from torch import nn

from ..lora.batched import add_lora_batch, has_lora_batch
from ..ops.gemm import svdq_gemm_w4a4_cuda
from ..ops.gemv import awq_gemv_w4a16_cuda
from ..ops.quantize import svdq_quantize_w4a4_act_fuse_lora_cuda


class SVDQW4A4Linear(nn.Module):
    """
    ``y = W4A4(quant(x / smooth)) + (x @ proj_down) @ proj_up^T + bias``.

    ``qweight (out, in // 2)`` int8, ``wscales (in // G, out)`` (16-bit for int4, float8_e4m3fn for nvfp4),
    ``smooth_factor (in)``, ``proj_down (in, rank)``, ``proj_up (out, rank)``, optional ``bias (out)``;
    nvfp4 adds ``wcscales (out)`` and the Python float ``wtscale``.
    """

    def __init__(self, in_features: int, out_features: int, rank: int = 32, bias: bool = True, precision: str = "int4",
                 act_unsigned: bool = False, torch_dtype: torch.dtype = torch.bfloat16,
                 device: str | torch.device | None = None):
        super().__init__()
        if device is None:
            device = torch.device("cpu")
        if precision not in ("int4", "nvfp4"):
            raise ValueError(f"Invalid precision: {precision}")
        self.in_features, self.out_features, self.rank = in_features, out_features, rank
        self.precision, self.torch_dtype = precision, torch_dtype
        self.group_size = 16 if precision == "nvfp4" else 64
        sdt = torch_dtype if precision == "int4" else torch.float8_e4m3fn

        def P(*shape, dtype=torch_dtype, grad=False):
            return nn.Parameter(torch.empty(*shape, dtype=dtype, device=device), requires_grad=grad)

        self.qweight = P(out_features, in_features // 2, dtype=torch.int8)
        self.bias = P(out_features) if bias else None
        self.wscales = P(in_features // self.group_size, out_features, dtype=sdt)
        self.smooth_factor = P(in_features)
        self.smooth_factor_orig = P(in_features)
        self.proj_down = P(in_features, rank)
        self.proj_up = P(out_features, rank)
        if precision == "nvfp4":
            self.wcscales = nn.Parameter(torch.ones(out_features, dtype=torch_dtype, device=device), requires_grad=False)
            self.wtscale = 1.0
        else:
            self.wtscale = None
            self.wcscales = None
        self.act_unsigned = act_unsigned

    @classmethod
    def from_linear(cls, linear: nn.Linear, **kwargs):
        in_features = kwargs.pop("in_features", linear.in_features)
        torch_dtype = kwargs.pop("torch_dtype", linear.weight.dtype)
        return cls(in_features=in_features, out_features=linear.out_features, bias=linear.bias is not None,
                   torch_dtype=torch_dtype, device=linear.weight.device, **kwargs)

    def forward(self, x: torch.Tensor, output: torch.Tensor | None = None) -> torch.Tensor:
        batch_size, seq_len, channels = x.shape
        x = x.reshape(batch_size * seq_len, channels)
        given = output is not None
        if not given:
            output = torch.empty(batch_size * seq_len, self.out_features, dtype=x.dtype, device=x.device)
        quantized_x, ascales, lora_act_out = self.quantize(x)
        output = self.forward_quant(quantized_x, ascales, lora_act_out, output)
        if has_lora_batch(self):
            rows = output.view(batch_size * seq_len, self.out_features)
            added = add_lora_batch(self, x, rows, samples=batch_size)
            if not given:
                output = added
            elif added is not rows:
                rows.copy_(added)
        return output.reshape(batch_size, seq_len, -1)

    def quantize(self, x: torch.Tensor, pad_size: int = 256):
        return svdq_quantize_w4a4_act_fuse_lora_cuda(
            x, lora_down=self.proj_down, smooth=self.smooth_factor, fp4=self.precision == "nvfp4", pad_size=pad_size
        )

    def forward_quant(self, quantized_x, ascales, lora_act, output: torch.Tensor | None = None) -> torch.Tensor:
        if output is None:
            output = torch.empty(quantized_x.shape[0], self.out_features, dtype=self.proj_up.dtype,
                                 device=quantized_x.device)
        svdq_gemm_w4a4_cuda(
            act=quantized_x, wgt=self.qweight, out=output, ascales=ascales, wscales=self.wscales, lora_act_in=lora_act,
            lora_up=self.proj_up, bias=self.bias, fp4=self.precision == "nvfp4", alpha=self.wtscale,
            wcscales=self.wcscales, act_unsigned=self.act_unsigned,
        )
        return output

    def __repr__(self):
        return (f"SVDQW4A4Linear(in_features={self.in_features}, out_features={self.out_features}, "
                f"rank={self.rank}, precision={self.precision}, act_unsigned={self.act_unsigned})")


class AWQW4A16Linear(nn.Module):
    """``qweight (out // 4, in // 2)`` int32 TinyChat packing, ``wscales / wzeros (in // group, out)``, optional bias."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, group_size: int = 64,
                 torch_dtype: torch.dtype = torch.bfloat16, device: str | torch.device | None = None):
        super().__init__()
        if device is None:
            device = torch.device("cpu")
        self.in_features, self.out_features, self.group_size = in_features, out_features, group_size
        self.qweight = nn.Parameter(
            torch.empty(out_features // 4, in_features // 2, dtype=torch.int32, device=device), requires_grad=False
        )
        self.bias = nn.Parameter(torch.empty(out_features, dtype=torch_dtype, device=device)) if bias else None
        self.wscales = nn.Parameter(
            torch.empty(in_features // group_size, out_features, dtype=torch_dtype, device=device), requires_grad=False
        )
        self.wzeros = nn.Parameter(
            torch.empty(in_features // group_size, out_features, dtype=torch_dtype, device=device), requires_grad=False
        )

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        output = awq_gemv_w4a16_cuda(
            in_feats=x, kernel=self.qweight, scaling_factors=self.wscales, zeros=self.wzeros, m=x.shape[0],
            n=self.out_features, k=self.in_features, group_size=self.group_size,
        )
        if self.bias is not None:
            view_shape = [1] * (output.ndim - 1) + [-1]
            output.add_(self.bias.view(view_shape))
        return output

    @classmethod
    def from_linear(cls, linear: nn.Linear, group_size: int = 64, torch_dtype: torch.dtype = torch.bfloat16,
                    device: str = "cpu", **kwargs):
        return cls(in_features=linear.in_features, out_features=linear.out_features, bias=linear.bias is not None,
                   group_size=group_size, torch_dtype=torch_dtype, device=device)

    def __repr__(self):
        return (f"AWQW4A16Linear(in_features={self.in_features}, out_features={self.out_features}, "
                f"group_size={self.group_size})")
