"""
Layer norm of rows whose mean is far above their deviation: the mean is taken off before anything else, and what its rounding
leaves goes into the result too.
"""

import pytest
import torch

from nunchaku_rocm_b200.ops.elementwise import layer_norm

F32 = 2.0**-24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu

# a warp per row, one team of warps (with threads that have no columns, with partial warps), four groups of columns per thread,
# and sizes that are no whole 16-byte pieces
DIMS = [1, 64, 256, 264, 512, 520, 1000, 1001, 1152, 4100, 5120, 8192, 8200, 8456, 12800, 16384]


@gpu
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype,values", [(FP32, [0.0, 300.1, -0.1, 7.3e-30, 1e20, -3.3e30, 1.7e37]), (BF16, [3.0, -1.1e20, 2e30]), (FP16, [300.1, -6e4, 6e-8])])
def test_rows_of_one_value_give_the_bias(cuda_dev, dim, dtype, values):
    g = torch.Generator(device=cuda_dev).manual_seed(dim)
    x = torch.tensor(values, dtype=dtype, device=cuda_dev)[:, None].expand(len(values), dim)
    x = x.repeat(5, 1).requires_grad_(True)  # more rows than a round takes
    w, b = (torch.randn(dim, generator=g, device=cuda_dev).requires_grad_(True) for _ in range(2))
    dy = torch.randn(x.shape, generator=g, device=cuda_dev).to(dtype)
    y = layer_norm(x, w, b)
    assert torch.equal(y.detach(), b.detach().to(dtype).expand_as(y))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert not dw.any()  # dy times zero
    total = dy.double().sum(0)
    assert ((db.double() - total).abs() <= F32 * (len(x) + 2) * dy.double().abs().sum(0)).all()
    if dtype == FP32 and dim > 1:  # dx = (v - mean v) / sqrt(eps), as there is no deviation
        v = dy.double() * w.detach().double()
        want = (v - v.mean(-1, keepdim=True)) * 1e3
        # eps in fp32, the root, v and the mean of v (at most dim / 32 + 40 additions one after the other)
        tol = 1e3 * F32 * (8 * v.abs() + (dim / 32 + 40) * v.abs().mean(-1, keepdim=True))
        assert ((dx.double() - want).abs() <= tol).all()


@gpu
@pytest.mark.parametrize("dim", [d for d in DIMS if d > 1])
@pytest.mark.parametrize("mean", [1000.0, 4096.0, -30000.0])
def test_a_large_mean_costs_nothing(cuda_dev, dim, mean):
    g = torch.Generator(device=cuda_dev).manual_seed(dim)
    x = torch.randn(37, dim, generator=g, device=cuda_dev) + mean
    w, b = (torch.randn(dim, generator=g, device=cuda_dev) for _ in range(2))
    d = x.double() - x.double().mean(-1, keepdim=True)
    xh = d * (d.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    want = xh * w.double() + b.double()
    # differences from a value near the mean are exact; their mean and that of their squares take at most dim / 32 + 40 additions
    # one after the other, of which the mean's weigh by |xh| (about 1); the rest are six roundings
    chain = dim / 32 + 40
    tol = F32 * ((chain + 6) * xh.abs() * w.abs() + (chain + 2) * xh.abs().mean(-1, keepdim=True) * w.abs() + 2 * want.abs())
    off = (layer_norm(x, w, b).double() - want).abs() - tol
    assert off.max() <= 0, off.max().item()


@gpu
@pytest.mark.parametrize("dim", [64, 1152, 1001, 5120, 8456])
def test_an_outlier_keeps_the_others(cuda_dev, dim):
    # one value of a row 10000 times the others, in every position that is a first one of a thread, a warp or the row
    g = torch.Generator(device=cuda_dev).manual_seed(dim)
    x = torch.randn(40, dim, generator=g, device=cuda_dev)
    at = [0, 1, 8, 9, 31, 32, 63]
    for i, c in enumerate(at):
        x[i, c] = 1e4
    d = x.double() - x.double().mean(-1, keepdim=True)
    xh = d * (d.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    # as above, but a difference is rounded where the outlier is what it is taken from, relative to xh's largest
    tol = F32 * ((dim / 32 + 46) * (xh.abs() + xh.abs().mean(-1, keepdim=True)) + 4 * xh.abs().amax(-1, keepdim=True) / dim**0.5 + 2)
    off = (layer_norm(x).double() - xh).abs() - tol
    assert off.max() <= 0, off.max().item()
