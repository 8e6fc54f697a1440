"""The rotation's cosines and sines: one fp32 rounding of the 64-bit values."""

import pytest
import torch

from nunchaku_rocm_b200.ops.rotary import rotary_table

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("axes,theta", [((16, 56, 56), 10000.0), ((64, 64), 500.0), ((256,), 1e6)])
def test_the_table_is_rounded_once(cuda_dev, axes, theta):
    ids = torch.stack([torch.arange(-700, 1300, device=cuda_dev) * (i + 1) for i in range(len(axes))], -1)
    table = rotary_table(ids, axes, theta)[:, :, 0].double()
    ang = torch.cat([ids[:, i, None].double() * theta ** (-2.0 * torch.arange(d // 2, device=cuda_dev, dtype=torch.float64) / d) for i, d in enumerate(axes)], -1)
    want = torch.stack([ang.sin(), ang.cos()], -1)
    # half a step of the value's own binade; a cosine of at least 0.7 (step 2^-24) lacks at most (pi / 4)^12 / 12! = 2^-33, a sine
    # y of at least 2^-9 y^13 / 13! = 2^-37 (step 2^-24): under 1/16 of a step; angles in 64 bits are 4000 x 2^-53 x 2 pi off
    step = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(2.0**-60))) - 23)
    off = (table - want).abs() - step * (0.5 + 1 / 16) - 2.0**-38
    assert off.max() <= 0, (off / step).max().item()
    # on the average no more than the rounding of the true values
    assert (table - want).norm() <= 1.02 * (want.float().double() - want).norm()
