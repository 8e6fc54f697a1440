"""
Layer norm with its backward pass and rotary positions with several axes, against their definitions in 64 bits.

Tolerances count roundings: ``half`` is half a step of the output type relative to the value; what is computed in fp32
before that rounding is off by a few 2^-24 of the terms that enter it.
"""

import pytest
import torch

from nunchaku_rocm_b200 import _lib as L
from nunchaku_rocm_b200.models.embeddings import flux_image_ids, flux_pos_embed
from nunchaku_rocm_b200.ops.elementwise import layer_norm, layernorm_modulate
from nunchaku_rocm_b200.ops.rotary import rotary_axes, rotary_table

F32 = 2.0**-24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu


def half(dt):
    return torch.finfo(dt).eps / 2


def within(got, ref, tol):
    off = ((got.double() - ref).abs() - tol).max().item() if ref.numel() else -1.0
    assert off <= 0, f"over the tolerance by {off:.3g} (largest difference {(got.double() - ref).abs().max().item():.3g})"


# --------------------------------------------------------------------------------------------------------------- refusals
def test_layer_norm_refuses():
    x = torch.zeros(2, 3, 16, dtype=BF16)
    w = torch.zeros(16, dtype=BF16)
    for args, kw in [((x.double(),), {}), ((x, w[:8]), {}), ((x, w.to(FP16)), {}), ((x, w, w.float()), {}),
                     ((x, torch.zeros(3, 16, dtype=BF16)), {}), ((x[0], torch.zeros(3, 16, dtype=BF16)), {}),
                     ((x, w, torch.zeros(2, 16, dtype=BF16)), {}), ((x,), {"weight_add": 1.0}), ((x[..., :0],), {})]:
        with pytest.raises(ValueError):
            layer_norm(*args, **kw)
    with pytest.raises(NotImplementedError):
        layer_norm(torch.zeros(1, 16385))
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer_norm(x, w)


def test_rotary_refuses():
    q, ids = torch.zeros(1, 5, 2, 64, dtype=BF16), torch.zeros(5, 2)
    for args, kw in [((q.double(), None, ids, (32, 32)), {}), ((q[0], None, ids, (32, 32)), {}), ((q, q.float(), ids, (32, 32)), {}),
                     ((q, q[:, :4], ids, (32, 32)), {}), ((q, None, ids, (32, 34)), {}), ((q, None, ids, (31, 33)), {}),
                     ((q, None, ids, ()), {}), ((q, None, ids, (16, 16, 16, 8, 8)), {}), ((q, None, ids, (64,)), {}),
                     ((q, None, ids[:4], (32, 32)), {}), ((q, None, ids.half(), (32, 32)), {}), ((q[:, :, :0], None, ids, (32, 32)), {}),
                     ((q, None, ids, (32, 32)), {"theta": -1.0}), ((q, None, ids, (32, 0)), {})]:
        with pytest.raises(ValueError):
            rotary_axes(*args, **kw)
    with pytest.raises(ValueError):
        rotary_table(torch.zeros(5), (64,))
    learned = torch.zeros(5, 2, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        rotary_axes(q, None, learned, (32, 32))
    with pytest.raises(ValueError, match="gradient"):
        rotary_table(learned, (32, 32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        rotary_axes(q, None, ids, (32, 32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        rotary_table(ids, (32, 32))


def test_the_c_entries_refuse_bad_sizes():
    # before any launch: these return without touching a device
    lib, a = L.lib(), L.LayerNormArgs(groups=1, rows=1, dim=0)
    assert lib.nb_layer_norm(a, None) == L.NB_ERR_INVALID
    a.dim, a.dtype = 20000, 2
    assert lib.nb_layer_norm(a, None) == L.NB_ERR_UNSUPPORTED
    a.dim = 64
    assert lib.nb_layer_norm(a, None) == L.NB_ERR_INVALID  # no x
    assert lib.nb_layer_norm_backward(L.LayerNormArgs(groups=0, rows=1, dim=8), None) == L.NB_ERR_INVALID
    assert lib.nb_layer_norm_workspace_bytes(1, 0, 64, 0) == 0
    r = L.RotaryArgs(B=1, S=1, H=1, D=8)
    assert lib.nb_rotary_axes(r, L.RotaryLadder(), None) == L.NB_ERR_INVALID  # no axes
    ladder = L.RotaryLadder()
    assert lib.nb_rotary_ladder_init(ladder, (L.C.c_int32 * 1)(16), 1, 1e4) == L.NB_OK
    assert lib.nb_rotary_axes(r, ladder, None) == L.NB_ERR_INVALID  # 16 channels of 8
    assert list(ladder.pair_end)[:1] == [8] and abs(ladder.turns[0] * 6.283185307179586 - 1) < 1e-15


# ------------------------------------------------------------------------------------------------------------- layer norm
def ln_ref(x, w, b, dy, eps, add, grouped):
    x, dy = x.double(), dy.double()
    per = (lambda v: v.double()[:, None]) if grouped else (lambda v: v.double())
    scale = (per(w) + add) if w is not None else torch.ones((), dtype=torch.float64, device=x.device)
    shift = per(b) if b is not None else torch.zeros((), dtype=torch.float64, device=x.device)
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh, v = (x - mean) * rstd, dy * scale
    y = xh * scale + shift
    dx = rstd * (v - v.mean(-1, keepdim=True) - xh * (v * xh).mean(-1, keepdim=True))
    over = tuple(range(1, x.dim() - 1)) if grouped else tuple(range(x.dim() - 1))
    total = (lambda t: t.sum(over)) if over else (lambda t: t)  # a single row is its own sum
    rows = x.shape[1] if grouped else x.numel() // x.shape[-1]
    # fp32: xh is off by the mean's and rstd's error, the sums by one rounding per term
    e = F32 * (8 + 4 * mean.abs() * rstd)
    return {"y": (y, e * (xh.abs() * scale.abs() + scale.abs()) + F32 * 4 * shift.abs()),
            "dx": (dx, rstd * 4 * e * (v.abs() + v.abs().mean(-1, keepdim=True) + (1 + xh.abs()) * (1 + (v * xh).abs().mean(-1, keepdim=True)))),
            "dw": (total(dy * xh), F32 * (rows + 8) * total((dy * xh).abs() + dy.abs()) + total(e * (1 + xh.abs()) * dy.abs())),
            "db": (total(dy), F32 * (rows + 8) * total(dy.abs()))}


def ln_check(x, w, b, dy, eps=1e-6, add=0.0):
    grouped = w is not None and w.dim() == 2
    leaves = [t if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, eps=eps, weight_add=add)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps=eps, weight_add=add), y.detach())
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    got = dict(zip(["dx"] + ["dw"] * (w is not None) + ["db"] * (b is not None), grads), y=y.detach())
    ref = ln_ref(x, w, b, dy, eps, add, grouped)
    for name, t in got.items():
        r, tol = ref[name]
        assert t.shape == r.shape and t.dtype == (x.dtype if name in ("y", "dx") else w.dtype if w is not None else b.dtype)
        within(t, r, tol + half(t.dtype) * (r.abs() + tol) + torch.finfo(t.dtype).smallest_normal)
    again = torch.autograd.grad(layer_norm(*leaves, eps=eps, weight_add=add), [t for t in leaves if t is not None], dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))  # fixed order of the sums
    return got


@gpu
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP16, FP32), (FP32, FP32)])
@pytest.mark.parametrize("dim", [1, 7, 8, 256, 257, 320, 512, 520, 1152, 4096, 4100, 5121, 8192, 8200, 16384])
def test_layer_norm_dims_and_types(cuda_dev, dtype, wdtype, dim):
    g = torch.Generator(device=cuda_dev).manual_seed(dim)
    x = (torch.randn(37, dim, generator=g, device=cuda_dev) * 2 + 0.5).to(dtype)
    w, b = (torch.randn(dim, generator=g, device=cuda_dev).to(wdtype) for _ in range(2))
    ln_check(x, w, b, torch.randn(37, dim, generator=g, device=cuda_dev).to(dtype), eps=1e-3 if dim == 1 else 1e-6)


@gpu
@pytest.mark.parametrize("B,T,dim", [(1, 1, 64), (3, 1, 1024), (2, 701, 96), (5, 33, 2048), (200, 3, 40), (2, 2500, 1000)])
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (FP16, FP32), (FP32, FP32)])
def test_layer_norm_per_sample(cuda_dev, B, T, dim, dtype, wdtype):
    g = torch.Generator(device=cuda_dev).manual_seed(B * T)
    x, dy = (torch.randn(B, T, dim, generator=g, device=cuda_dev).to(dtype) for _ in range(2))
    mod = torch.randn(B, 3 * dim + 8, generator=g, device=cuda_dev).to(wdtype)
    ln_check(x, mod[:, :dim], mod[:, dim : 2 * dim], dy, add=1.0)      # views of one projection
    ln_check(x, mod[:, 1 : dim + 1], mod[:, dim : 2 * dim], dy, add=1.0)  # and one off every alignment


@gpu
def test_layer_norm_layouts(cuda_dev):
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    big = torch.randn(4, 60, 3, 128, generator=g, device=cuda_dev).to(BF16)
    w, b = torch.randn(128, generator=g, device=cuda_dev), torch.randn(128, generator=g, device=cuda_dev)
    for x in (big[:, :, 1], big[:, 5:40, 0], big.transpose(0, 1)[:, :, 2], big[..., ::2].repeat_interleave(2, -1)[:, 0], big[0, 0, 0],
              big[:1, :1, 0], big[0].transpose(0, 1), big[:, :1].expand(4, 7, 3, 128)[..., 0, :], big.reshape(-1)[3:643].view(5, 128)):
        dy = torch.randn(x.shape, generator=g, device=cuda_dev).to(BF16)
        ln_check(x, w, b, dy)
    x = big[:, :, 0].contiguous()
    ln_check(x, None, None, torch.randn(x.shape, generator=g, device=cuda_dev).to(BF16))
    ln_check(x, w.to(BF16), None, torch.randn(x.shape, generator=g, device=cuda_dev).to(BF16))
    ln_check(x, None, b, torch.randn(x.shape, generator=g, device=cuda_dev).to(BF16))
    ln_check(x, w, b, torch.randn(60, 4, 128, generator=g, device=cuda_dev).to(BF16).transpose(0, 1))
    ln_check(x, w, b, torch.randn(1, 1, 128, generator=g, device=cuda_dev).to(BF16).expand(4, 60, 128))


@gpu
def test_layer_norm_empty_constant_and_non_finite_rows(cuda_dev):
    w, b = torch.randn(64, device=cuda_dev, requires_grad=True), torch.randn(64, device=cuda_dev, requires_grad=True)
    x = torch.zeros(0, 64, device=cuda_dev, requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 64, device=cuda_dev))
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()
    x = torch.full((3, 64), 7.25, device=cuda_dev)  # no variance: y is the bias
    assert torch.equal(layer_norm(x, w, b).detach(), b.detach().expand(3, 64))
    x[1, 5], x[2, 9] = float("inf"), float("nan")
    y = layer_norm(x, w, b).detach()
    assert torch.equal(y[0], b.detach()) and y[1:].isnan().all()
    # one row's NaN stays in that row of dx
    xg = torch.randn(5, 64, device=cuda_dev)
    xg[3, 1] = float("nan")
    xg.requires_grad_(True)
    (dx,) = torch.autograd.grad(layer_norm(xg, w, b), xg, torch.ones(5, 64, device=cuda_dev))
    assert dx[3].isnan().all() and torch.isfinite(dx[[0, 1, 2, 4]]).all()


@gpu
def test_layer_norm_large_mean_keeps_the_variance(cuda_dev):
    # the mean is 4096 times the deviation: squares are summed after it is taken off
    x = torch.randn(9, 512, device=cuda_dev) + 4096.0
    ln_check(x, torch.ones(512, device=cuda_dev), torch.zeros(512, device=cuda_dev), torch.randn(9, 512, device=cuda_dev))


@gpu
def test_layer_norm_gradient_against_differences(cuda_dev):
    g = torch.Generator(device=cuda_dev).manual_seed(11)
    x, dy, d = (torch.randn(6, 40, generator=g, device=cuda_dev) for _ in range(3))
    w, b, dwt = (torch.randn(40, generator=g, device=cuda_dev) for _ in range(3))
    got = ln_check(x, w, b, dy)

    def value(x, w):
        return (ln_ref(x, w, b, dy, 1e-6, 0.0, False)["y"][0] * dy.double()).sum()

    # central differences in 64 bits: off by h^2 of a third derivative of order one per element; fp32 gradients by ~2^-20
    h = 1e-4
    num = (value(x.double() + h * d, w) - value(x.double() - h * d, w)) / (2 * h)
    assert abs(num - (got["dx"].double() * d).sum()) <= 1e-6 * 240 + 2.0**-20 * (got["dx"] * d).abs().sum()
    num = (value(x, w.double() + h * dwt) - value(x, w.double() - h * dwt)) / (2 * h)
    assert abs(num - (got["dw"].double() * dwt).sum()) <= 2.0**-20 * (got["dw"] * dwt).abs().sum() + 1e-9


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_layernorm_modulate_keeps_its_values_and_has_gradients(cuda_dev, dtype):
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    x = torch.randn(2, 50, 1024, generator=g, device=cuda_dev).to(dtype)
    mod = (torch.randn(2, 6 * 1024, generator=g, device=cuda_dev) * 0.3).to(dtype)
    dy = torch.randn(2, 50, 1024, generator=g, device=cuda_dev).to(dtype)
    interleaved = mod.view(2, 1024, 6)
    for scale, shift in ((interleaved[..., 1], interleaved[..., 0]), (mod[:, 1024:2048], mod[:, :1024])):
        plain = layernorm_modulate(x, scale, shift, scale_add=1.0)
        leaves = [t.detach().requires_grad_(True) for t in (x, scale, shift)]
        y = layernorm_modulate(*leaves, scale_add=1.0)
        assert torch.equal(y, plain)
        ref = ln_ref(x, scale, shift, dy, 1e-6, 1.0, True)
        for name, t in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy)):
            r, tol = ref[name]
            within(t, r, tol + half(dtype) * (r.abs() + tol) + torch.finfo(dtype).smallest_normal)
    only = shift.detach().requires_grad_(True)
    (db,) = torch.autograd.grad(layernorm_modulate(x, scale, only, scale_add=1.0), only, dy)
    within(db, ref["db"][0], ref["db"][1] + half(dtype) * (ref["db"][0].abs() + ref["db"][1]))


@gpu
def test_layer_norm_captured_on_another_stream(cuda_dev):
    x = torch.randn(64, 768, device=cuda_dev).to(BF16)
    w, b, dy = torch.randn(768, device=cuda_dev), torch.randn(768, device=cuda_dev), torch.randn(64, 768, device=cuda_dev).to(BF16)
    ops = L.binding()
    stats = torch.empty(2, 64, device=cuda_dev)
    y = torch.empty_like(x)
    ops.layer_norm_forward(x, w, b, 1e-6, 0.0, y, stats)
    backward = lambda: ops.layer_norm_backward(x, w, b, stats, dy, 1e-6, 0.0, True, True, True)  # noqa: E731
    s = torch.cuda.Stream()
    graphs, outs = [], []
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):  # two graphs, each with a workspace of its own
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                outs.append((layer_norm(x, w, b), *backward()))
            graphs.append(gr)
    torch.cuda.current_stream().wait_stream(s)
    x.copy_(torch.randn(64, 768, device=cuda_dev))
    ops.layer_norm_forward(x, w, b, 1e-6, 0.0, None, stats)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for gr, st in zip(graphs, streams):
        with torch.cuda.stream(st):
            gr.replay()
    torch.cuda.synchronize()
    want = (layer_norm(x, w, b), *backward())
    for out in outs:
        assert all(torch.equal(p, q) for p, q in zip(out, want))


# ----------------------------------------------------------------------------------------------------------------- rotary
def rot_ref(x, ids, axes, theta, half_split, inverse):
    if ids.dim() == 2:
        ids = ids[None]
    ang = torch.cat([ids[..., i, None].double() * theta ** (-2.0 * torch.arange(d // 2, device=x.device, dtype=torch.float64) / d)
                     for i, d in enumerate(axes)], -1)[:, :, None]
    c, s = torch.cos(ang), torch.sin(ang) * (-1 if inverse else 1)
    xd, r = x.double(), 2 * ang.shape[-1]
    u, v = (xd[..., : r // 2], xd[..., r // 2 : r]) if half_split else (xd[..., :r:2], xd[..., 1:r:2])
    p, q = u * c - v * s, u * s + v * c
    m = u.abs() + v.abs()
    join = (lambda a, b: torch.cat([a, b], -1)) if half_split else (lambda a, b: torch.stack([a, b], -1).flatten(-2))
    # cos and sin are off by a step or two of fp32, each product and the sum by half a step; the rest is copied
    return torch.cat([join(p, q), xd[..., r:]], -1), torch.cat([join(m, m) * 6 * F32, torch.zeros_like(xd[..., r:])], -1)


def rot_check(q, k, ids, axes, theta=10000.0, interleaved=True):
    ql, kl = q.detach().requires_grad_(True), None if k is None else k.detach().requires_grad_(True)
    for inverse in (False, True):
        out = rotary_axes(ql, kl, ids, axes, theta, interleaved, inverse)
        outs, leaves = ([out], [ql]) if k is None else (list(out), [ql, kl])
        with torch.no_grad():
            plain = rotary_axes(q, k, ids, axes, theta, interleaved, inverse)
            assert all(torch.equal(p, o) for p, o in zip([plain] if k is None else plain, outs))
        grads = torch.autograd.grad(outs, leaves, [t.detach().flip(1) for t in outs])
        for o, leaf, d in zip(outs, leaves, grads):
            ref, tol = rot_ref(leaf.detach(), ids, axes, theta, not interleaved, inverse)
            assert o.shape == leaf.shape and o.is_contiguous()
            within(o.detach(), ref, tol + half(o.dtype) * (ref.abs() + tol) + torch.finfo(o.dtype).smallest_normal)
            ref, tol = rot_ref(o.detach().flip(1), ids, axes, theta, not interleaved, not inverse)
            within(d, ref, tol + half(o.dtype) * (ref.abs() + tol) + torch.finfo(o.dtype).smallest_normal)


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,axes", [(128, (16, 56, 56)), (64, (64,)), (128, (44, 42, 42)), (72, (24, 24, 24)), (96, (16, 16)),
                                    (70, (2, 4, 6, 8)), (33, (32,)), (256, (128, 128)), (128, (30, 30, 4))])
def test_rotary_heads_and_axes(cuda_dev, dtype, interleaved, D, axes):
    g = torch.Generator(device=cuda_dev).manual_seed(D)
    for B, S, H, Hk in ((1, 1, 1, 1), (2, 37, 3, 1), (1, 701, 5, 5)):
        q, k = torch.randn(B, S, H, D, generator=g, device=cuda_dev).to(dtype), torch.randn(B, S, Hk, D, generator=g, device=cuda_dev).to(dtype)
        ids = torch.randint(0, 200, (S, len(axes)), generator=g, device=cuda_dev)
        rot_check(q, k, ids, axes, interleaved=interleaved)
        rot_check(q, None, ids[None].expand(B, S, len(axes)).float() + 0.25, axes, theta=500.0, interleaved=interleaved)


@gpu
@pytest.mark.parametrize("idt", [torch.float32, torch.float64, torch.int32, torch.int64])
def test_rotary_far_positions_and_id_types(cuda_dev, idt):
    ids = torch.tensor([[0, -3], [1, 70000], [12345678, -16777215], [2**24, 1]], device=cuda_dev).to(idt)
    q = torch.randn(2, 4, 3, 64, device=cuda_dev)
    # 64-bit angles of the definition: a position of 2^24 turns by 2^24 2^-53 radians of error, far under fp32
    rot_check(q, None, ids, (32, 32))
    rot_check(q, None, torch.stack([ids, ids.flip(0)]).transpose(0, 1).contiguous().transpose(0, 1), (32, 32))
    bad = rotary_axes(q, None, torch.full((4, 2), float("nan"), device=cuda_dev), (32, 16))
    assert bad[..., :48].isnan().all() and torch.equal(bad[..., 48:], q[..., 48:])


@gpu
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_layouts(cuda_dev, interleaved):
    g = torch.Generator(device=cuda_dev).manual_seed(8)
    B, S, H, D = 2, 45, 4, 128
    ids = torch.randint(0, 64, (S, 3), generator=g, device=cuda_dev).float()
    qkv = torch.randn(B, S, 3 * H * D + 1, generator=g, device=cuda_dev).to(BF16)
    packed = qkv[..., : 3 * H * D].contiguous().view(B, S, 3, H, D)
    rot_check(packed[:, :, 0], packed[:, :, 1], ids, (16, 56, 56), interleaved=interleaved)
    odd = qkv[..., 1 : H * D + 1].unflatten(-1, (H, D))  # every row off its alignment
    rot_check(odd, packed[:, :, 1], ids, (16, 56, 56), interleaved=interleaved)
    bhsd = torch.randn(B, H, S, D, generator=g, device=cuda_dev).to(BF16).transpose(1, 2)
    rot_check(bhsd, bhsd[:, :, :1], ids, (16, 56, 56), interleaved=interleaved)
    rot_check(bhsd, bhsd[:, :, :1].expand(B, S, 3, D), ids, (16, 56, 56), interleaved=interleaved)
    rot_check(bhsd.flip(3)[..., ::2].repeat_interleave(2, 3)[..., ::2], None, ids, (16, 24, 24), interleaved=interleaved)
    assert rotary_axes(bhsd[:, :0], None, ids[:0], (16, 56, 56)).shape == (B, 0, H, D)
    # only K's gradient is asked for
    k = bhsd.detach().requires_grad_(True)
    _, ko = rotary_axes(packed[:, :, 0], k, ids, (16, 56, 56), interleaved=interleaved)
    (dk,) = torch.autograd.grad(ko, k, ko.detach())
    back = rotary_axes(ko.detach(), None, ids, (16, 56, 56), interleaved=interleaved, inverse=True)
    assert torch.equal(dk, back)


@gpu
def test_rotary_gradient_against_differences(cuda_dev):
    g = torch.Generator(device=cuda_dev).manual_seed(2)
    q, d, dy = (torch.randn(1, 9, 2, 24, generator=g, device=cuda_dev) for _ in range(3))
    ids = torch.randint(0, 50, (9, 2), generator=g, device=cuda_dev)
    ql = q.clone().requires_grad_(True)
    (dq,) = torch.autograd.grad(rotary_axes(ql, None, ids, (8, 16)), ql, dy)
    # the operator is linear: a difference over a step of one has no truncation error, only fp32 roundings of each side
    up, down = rotary_axes(q + d, None, ids, (8, 16)).double(), rotary_axes(q - d, None, ids, (8, 16)).double()
    num = ((up - down) / 2 * dy).sum()
    assert abs(num - (dq.double() * d).sum()) <= 16 * F32 * ((q.abs() + d.abs()) * dy.abs()).sum() * 2


@gpu
@pytest.mark.parametrize("txt,h,w", [(0, 1, 1), (5, 7, 9), (512, 64, 64)])
def test_rotary_table(cuda_dev, txt, h, w):
    ids = flux_image_ids(txt, h, w, device=cuda_dev)
    table = rotary_table(ids, (16, 56, 56))
    want = flux_pos_embed(ids, (16, 56, 56))
    assert table.shape == want.shape and table.is_contiguous()
    ang = torch.cat([ids[:, i, None].double() * 10000.0 ** (-2.0 * torch.arange(d // 2, device=cuda_dev, dtype=torch.float64) / d)
                     for i, d in enumerate((16, 56, 56))], -1)
    within(table, torch.stack([ang.sin(), ang.cos()], -1)[:, :, None], 3 * F32)
    batched = rotary_table(torch.stack([ids, ids + 3]), (16, 56, 56))
    assert torch.equal(batched[0], table) and torch.equal(batched[1], rotary_table(ids + 3, (16, 56, 56)))


@gpu
def test_rotary_captured(cuda_dev):
    ids = torch.randint(0, 60, (33, 3), device=cuda_dev).float()
    q = torch.randn(1, 33, 2, 128, device=cuda_dev).to(BF16)
    rotary_axes(q, q, ids, (16, 56, 56))
    gr, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(gr, stream=s):
        a, b = rotary_axes(q, q, ids, (16, 56, 56))
        t = rotary_table(ids, (16, 56, 56))
    ids.add_(5)
    q.mul_(-2)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, rotary_axes(q, None, ids, (16, 56, 56))) and torch.equal(a, b)
    assert torch.equal(t, rotary_table(ids, (16, 56, 56)))


def test_struct_fields_match_the_header():
    import pathlib
    import re

    text = (pathlib.Path(__file__).parent.parent / "include" / "nunchaku_b200.h").read_text()
    text = re.sub(r"/\*.*?\*/|//[^\n]*", "", text, flags=re.S)
    for name, ctype in (("nb_lora_args", L.LoraArgs), ("nb_layer_norm_args", L.LayerNormArgs), ("nb_rotary_args", L.RotaryArgs),
                        ("nb_rotary_ladder", L.RotaryLadder)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        fields = [re.search(r"(\w+)\s*(\[[^\]]*\])?$", f.strip()).group(1) for line in body.split(";") if line.strip() for f in line.split(",")]
        assert fields == [f[0] for f in ctype._fields_], name


@gpu
def test_norm_and_rotary_training_steps_captured(cuda_dev):
    x, w, b, dy = (torch.randn(s, device=cuda_dev).to(FP16) for s in ((2, 50, 320), (2, 320), (2, 320), (2, 50, 320)))
    q, k, dq, dk = (torch.randn(2, 50, h, 64, device=cuda_dev).to(FP16) for h in (4, 1, 4, 1))
    ids = torch.randint(0, 90, (50, 2), device=cuda_dev).float()

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b, q, k)]
        y = layer_norm(*leaves[:3], weight_add=1.0)
        r = rotary_axes(*leaves[3:], ids, (32, 32), interleaved=False)
        return (y.detach(), *(t.detach() for t in r), *torch.autograd.grad((y, *r), leaves, (dy, dq, dk)))

    step()
    s, gr = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(gr, stream=s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    ids.add_(3)
    for t in (x, w, dy, q, dk):
        t.mul_(-0.5)
    for _ in range(2):
        gr.replay()
    assert all(torch.equal(a, c) for a, c in zip(got, step()))


@gpu
def test_more_than_2_31_elements(cuda_dev):
    # the last rows, whose offsets pass 32 bits, are those of a call on these rows alone
    T, D, tail = (1 << 19) + 5, 4104, 37
    assert T * D > 1 << 31
    x, dy = torch.empty(T, D, dtype=FP16, device=cuda_dev).normal_(), torch.empty(T, D, dtype=FP16, device=cuda_dev).normal_()
    y, dx = [], []
    for rows in (slice(None), slice(T - tail, None)):
        leaf = x[rows].detach().requires_grad_(True)
        y.append(layer_norm(leaf))
        dx += torch.autograd.grad(y[-1], leaf, dy[rows])
    assert torch.equal(y[0][-tail:], y[1]) and torch.equal(dx[0][-tail:], dx[1])
    del dy, y, dx
    H = 4104 // 8
    q = x.view(T, 1, H, 8)  # more than 2^19 samples of one token
    ids = torch.randint(0, 500, (T, 1, 2), device=cuda_dev)
    got = rotary_axes(q, None, ids, (4, 4))
    assert torch.equal(got[-tail:], rotary_axes(q[-tail:], None, ids[-tail:], (4, 4)))


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,axes", [(128, (42, 42, 42)), (72, (24, 24, 24)), (72, (20, 24, 22)), (64, (2,)), (66, (22, 22, 22)), (68, (8, 26))])
def test_rotary_splits_inside_a_piece(cuda_dev, dtype, interleaved, D, axes):
    # channel counts that no 16-byte piece divides; what is behind the axes passes through, whatever it holds
    q, k = torch.randn(2, 37, 3, D, device=cuda_dev).to(dtype), torch.randn(2, 37, 1, D, device=cuda_dev).to(dtype)
    if sum(axes) < D:
        q[0, 3, 1, sum(axes):] = float("inf")
    ids = torch.randint(-50, 50, (37, len(axes)), device=cuda_dev)
    got = rotary_axes(q, k, ids, axes, interleaved=interleaved)
    for t, out in zip((q, k), got):
        R = sum(axes)
        rates = torch.cat([10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=cuda_dev) / d) for d in axes])
        angle = torch.cat([ids[:, i : i + 1].double().expand(-1, d // 2) for i, d in enumerate(axes)], 1) * rates
        c, s = angle.cos()[None, :, None], angle.sin()[None, :, None]
        x = t[..., :R].double()
        u, v = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., : R // 2], x[..., R // 2 :])
        a, b = u * c - v * s, u * s + v * c
        ref = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
        # one rounding; cos and sin off by 2^-24 of a turn's part (4 of fp32's half steps), the rotation's own two roundings
        big = torch.stack([u.abs() + v.abs()] * 2, -1).flatten(-2) if interleaved else torch.cat([u.abs() + v.abs()] * 2, -1)
        tol = torch.finfo(dtype).eps / 2 * ref.abs() + 8 * 2.0**-24 * big + torch.finfo(dtype).smallest_normal
        assert ((out[..., :R].double() - ref).abs() <= tol * (1 + 2.0**-10)).all()
        assert torch.equal(out[..., R:], t[..., R:])
