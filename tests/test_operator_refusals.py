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


def test_sizes_beyond_32_bits_are_refused():
    # views without memory of their own: 2^32 + something would be something to the C entries
    far = 2**32 + 3
    q, ids = torch.zeros(1, 1, 1, 64), torch.zeros(1, 2)
    with pytest.raises(RuntimeError, match="2\\^31 rows"):
        rotary_axes(q.expand(1, far, 1, 64), None, ids.expand(far, 2), (32, 32))
    with pytest.raises(RuntimeError, match="2\\^31 rows"):
        rotary_axes(q.expand(far, 1, 1, 64), None, ids, (32, 32))
    with pytest.raises(RuntimeError, match="channels per row"):
        rotary_axes(q, q.expand(1, 1, far, 64), ids, (32, 32))
    for t in (ids.expand(far, 2), ids.expand(far, 1, 2)):
        with pytest.raises(RuntimeError, match="2\\^31 rows"):
            rotary_table(t, (32, 32))
    w = torch.zeros(1, 8)
    for samples in (65536, 2**32):
        with pytest.raises(RuntimeError, match="65535 samples"):
            layer_norm(torch.zeros(1, 1, 8).expand(samples, 1, 8), w.expand(samples, 8))
        with pytest.raises(RuntimeError, match="65535 samples"):
            layer_norm(torch.zeros(1, 1, 8).expand(samples, 1, 8), None, w.expand(samples, 8))
    x, down, up, one = torch.zeros(4, 64, dtype=BF16), torch.zeros(1, 16, 64, dtype=BF16), torch.zeros(1, 32, 16, dtype=BF16), torch.zeros(1, dtype=torch.int32)
    off = torch.tensor([0, 4], dtype=torch.int32)
    wide = 2**32 + 64
    for args in ((x[:, :1].expand(4, wide), down[..., :1].expand(1, 16, wide), up, off, one), (x, down, up[:, :1].expand(1, wide, 16), off, one),
                 (x, down.expand(65536, 16, 64), up.expand(65536, 32, 16), off, one), (x, down, up, one.expand(far + 1), one.expand(far))):
        with pytest.raises(RuntimeError, match="65535 adapters or requests, or 2\\^24 columns"):
            lora_batched(*args)
