"""Calls that the differentiable operators refuse, because they would answer them wrongly: on the CPU, before any launch."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from nunchaku_rocm_b200.ops.elementwise import layer_norm, layernorm_modulate
from nunchaku_rocm_b200.ops.lora import lora_batched
from nunchaku_rocm_b200.ops.rotary import rotary_axes, rotary_table

BF16 = torch.bfloat16


def dual(t):
    return fwad.make_dual(t, torch.ones_like(t))


def test_forward_mode_is_refused():
    x, w = torch.zeros(2, 3, 16), torch.ones(16)
    q, ids = torch.zeros(1, 5, 2, 64), torch.zeros(5, 2)
    a, down, up, base = (torch.zeros(s, dtype=BF16) for s in ((4, 64), (1, 16, 64), (1, 32, 16), (4, 32)))
    off, ad, scale = torch.tensor([0, 4], dtype=torch.int32), torch.tensor([0], dtype=torch.int32), torch.ones(1)
    m, mod = torch.zeros(1, 2, 1024, dtype=BF16), torch.zeros(1, 1024, dtype=BF16)
    calls = [(layer_norm, (x, w, w)), (rotary_axes, (q, q.clone(), ids, (32, 32))), (rotary_table, (ids, (32, 32))),
             (lora_batched, (a, down, up, off, ad, base, scale)), (layernorm_modulate, (m, mod, mod.clone()))]
    with fwad.dual_level():
        for fn, args in calls:
            for i, t in enumerate(args):
                if isinstance(t, torch.Tensor) and t.is_floating_point():
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        fn(*args[:i], dual(t), *args[i + 1 :])
            with pytest.raises(RuntimeError, match="no CPU path"):  # without a tangent: the call itself
                fn(*args)
