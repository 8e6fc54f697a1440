"""
Batched adapters where the 16-bit types are narrow: h = s x D^T and g = s dy U far beyond and far below float16's own values.

h and g are fp32 sums that the second products read in 16-bit parts: bfloat16's three hold all of their 24 bits, float16's two
follow a power of two that brings a row's largest value below 2^15.  What float16's cost, and the tolerances count:

* 2^-22 of each value (half a step of 2^-11, twice);
* 2^-39 of the row's largest (of the adapter's largest, where rows are summed): half of float16's smallest step, 2^-25, beside
  2^14 or more;
* fp32 sums, 2^-24 per term;
* one rounding of the result, half a step or half of the smallest step.
"""

import pytest
import torch

from nunchaku_rocm_b200 import _lib as L
from nunchaku_rocm_b200.ops.lora import lora_batched

F32 = 2.0**-24
BF16, FP16 = torch.bfloat16, torch.float16
IMPLS = {"generic": L.IMPL_GENERIC, "tcgen05": L.IMPL_TCGEN05, "auto": L.IMPL_AUTO}
gpu = pytest.mark.gpu


def part(v, dim, dtype):
    """What the parts of `v` lose: rows (dim=-1) or all of an adapter's rows (dim=(0, 1)) share a power of two in float16."""
    if dtype == BF16:
        return torch.zeros_like(v)
    return 2.0**-22 * v.abs() + 2.0**-39 * v.abs().amax(dim, keepdim=True)


def rounded(v, tol, dtype):
    info = torch.finfo(dtype)
    return tol + info.eps / 2 * (v.abs() + tol) + info.smallest_normal * info.eps / 2


def reference(p, offsets, adapters):
    """{name: (value, tolerance)} of the definition in 64 bits."""
    d, dt = {k: v.double() for k, v in p.items()}, p["x"].dtype
    (T, K), (A, N, R) = p["x"].shape, p["up"].shape
    zero = {"out": d["base"], "dx": d["x"], "ddown": d["down"], "dup": d["up"]}
    val = {k: d["base"].clone() if k == "out" else torch.zeros_like(v) for k, v in zero.items()}
    tol = {k: torch.zeros_like(v) for k, v in zero.items()}
    whole = {}
    for i, a in enumerate(adapters):
        rows = slice(offsets[i], offsets[i + 1])
        if offsets[i] == offsets[i + 1] or not 0 <= a < A:
            continue
        s, x, dy, D, U = d["scale"][a], d["x"][rows], d["dy"][rows], d["down"][a], d["up"][a]
        h, g = s * x @ D.t(), s * dy @ U
        eh, eg = F32 * (K + 4) * (s * x.abs() @ D.t().abs()), F32 * (N + 4) * (s * dy.abs() @ U.abs())
        val["out"][rows] += h @ U.t()
        tol["out"][rows] += (eh + part(h, -1, dt)) @ U.t().abs() + F32 * (R + 4) * (h.abs() @ U.t().abs()) + F32 * val["out"][rows].abs()
        val["dx"][rows] = g @ D
        tol["dx"][rows] = (eg + part(g, -1, dt)) @ D.abs() + F32 * (R + 4) * (g.abs() @ D.abs())
        whole.setdefault(a, []).append((h, g, eh, eg, x, dy))
    for a, parts in whole.items():
        h, g, eh, eg, x, dy = (torch.cat(t) for t in zip(*parts))
        val["ddown"][a], val["dup"][a] = g.t() @ x, dy.t() @ h
        tol["ddown"][a] = (eg + part(g, -1, dt) + part(g, (0, 1), dt)).t() @ x.abs() + F32 * (T + 4) * (g.t().abs() @ x.abs())
        tol["dup"][a] = dy.t().abs() @ (eh + part(h, -1, dt) + part(h, (0, 1), dt)) + F32 * (T + 4) * (dy.t().abs() @ h.abs())
    return {k: (val[k], rounded(val[k], tol[k], dt)) for k in val}


def run(p, off, ad, impl):
    leaves = [p[k].detach().requires_grad_(True) for k in ("x", "down", "up")]
    out = lora_batched(*leaves, off, ad, base=p["base"], scale=p["scale"], _impl=impl)
    return dict(zip(("out", "dx", "ddown", "dup"), (out.detach(), *torch.autograd.grad(out, leaves, p["dy"]))))


def check(p, offsets, adapters, impl):
    dev = p["x"].device
    off, ad = torch.tensor(offsets, dtype=torch.int32, device=dev), torch.tensor(adapters, dtype=torch.int32, device=dev)
    got, want = run(p, off, ad, impl), reference(p, offsets, adapters)
    for name, (ref, tol) in want.items():
        over = (got[name].double() - ref).abs() - tol
        assert over.isfinite().all() and over.max() <= 0, (name, over.max().item(), (got[name].double() - ref).abs().max().item())
    assert L.device_status(dev) == 0


def make(dev, T, K, N, R, A, dtype, x=1.0, down=1.0, up=1.0, dy=1.0, base=1.0, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = lambda k, *s: (torch.randn(s, generator=g, device=dev) * k).to(dtype)  # noqa: E731
    return {"x": n(x, T, K), "base": n(base, T, N), "down": n(down * K**-0.5, A, R, K), "up": n(up, A, N, R), "dy": n(dy, T, N),
            "scale": torch.rand(A, generator=g, device=dev) + 0.5}


@gpu
@pytest.mark.parametrize("impl", IMPLS.values(), ids=IMPLS)
@pytest.mark.parametrize("up,dy", [(1e-4, 1e-2), (1e-4, 1e-4), (6e-2, 1e-6), (6e-5, 6e-5)])
def test_small_gradients_of_float16(cuda_dev, up, dy, impl):
    # adapters that have just begun to train: dy U is far below float16's normal numbers, the sums over the rows are not
    p = make(cuda_dev, 1333, 520, 1032, 16, 2, FP16, up=up, dy=dy, x=300.0, base=0.0, seed=3)
    check(p, [0, 700, 1333], [1, 0], impl)


@gpu
@pytest.mark.parametrize("impl", IMPLS.values(), ids=IMPLS)
@pytest.mark.parametrize("R", [16, 32, 48, 64, 96, 128])
@pytest.mark.parametrize("T,offsets,adapters", [(21, [0, 9, 21], [1, 0]), (400, [0, 130, 390], [0, 1])])
def test_rows_of_unlike_size(cuda_dev, R, T, offsets, adapters, impl):
    # neighbouring rows, and the ranks of a row, many powers of two apart: every row keeps its own power
    p = make(cuda_dev, T, 328, 264, R, 2, FP16, up=0.05, seed=R)
    g = torch.Generator(device=cuda_dev).manual_seed(R)
    for name, high in (("x", 5), ("dy", 2)):
        p[name] = (p[name].float() * torch.exp2(torch.randint(-14, high, (T, 1), generator=g, device=cuda_dev).float())).to(FP16)
    p["down"] = (p["down"].float() * torch.exp2(torch.randint(-6, 3, (2, R, 1), generator=g, device=cuda_dev).float())).to(FP16)
    check(p, offsets, adapters, impl)


@gpu
@pytest.mark.parametrize("impl", IMPLS.values(), ids=IMPLS)
@pytest.mark.parametrize("T", [1, 16, 300])
def test_h_beyond_float16(cuda_dev, T, impl):
    K, N, R = 1024, 64, 16
    off, ad = torch.tensor([0, T], dtype=torch.int32, device=cuda_dev), torch.tensor([0], dtype=torch.int32, device=cuda_dev)
    x, down = torch.full((T, K), 6e4, dtype=FP16, device=cuda_dev), torch.ones(1, R, K, dtype=FP16, device=cuda_dev)
    base = torch.randn(T, N, generator=torch.Generator(device=cuda_dev).manual_seed(1), device=cuda_dev).to(FP16)
    call = lambda up, **kw: lora_batched(x, down, up, off, ad, _impl=impl, **kw)  # noqa: E731
    # h is 6.1e7 in every rank; one that up leaves out leaves base as it is, two of unlike sign cancel
    up = torch.zeros(1, N, R, dtype=FP16, device=cuda_dev)
    assert torch.equal(call(up, base=base), base)
    up[0, :, 3], up[0, :, 9] = 1.0, -1.0
    assert torch.equal(call(up, base=base), base)
    up.zero_()[0, :, 5] = 2.0**-14
    h = float(x[0, 0]) * K  # exact in fp32: 60000 x 2^10
    assert (call(up) == torch.tensor(h * 2.0**-14).to(FP16).item()).all()
    assert (call(up.neg()) == -torch.tensor(h * 2.0**-14).to(FP16).item()).all()
    assert (call(up * 64) == float("inf")).all()  # 2.3e5: the result itself is beyond float16
    # a scale that carries h there
    assert torch.equal(call(up * 2.0**-10, scale=torch.full((1,), 1024.0, device=cuda_dev)), call(up))
    # g and the gradients: dy U and the sums over the rows are as far out, their products with the factors are not
    up = torch.full((1, N, R), 2.0**10, dtype=FP16, device=cuda_dev)
    leaves = [t.detach().requires_grad_(True) for t in (torch.full((T, K), 2.0**-10, dtype=FP16, device=cuda_dev), torch.full((1, R, K), 2.0**-14, dtype=FP16, device=cuda_dev), up)]
    dx, ddown, dup = torch.autograd.grad(lora_batched(*leaves, off, ad, _impl=impl), leaves, torch.ones(T, N, dtype=FP16, device=cuda_dev))
    assert (dx == 64.0).all()  # g = 2^16 in every rank: 16 x 2^16 x 2^-14
    assert (ddown == torch.tensor(T * 64.0).to(FP16).item()).all() and (dup == torch.tensor(T * 2.0**-14).to(FP16).item()).all()


@gpu
@pytest.mark.parametrize("impl", IMPLS.values(), ids=IMPLS)
def test_a_row_that_is_not_finite_keeps_its_kind(cuda_dev, impl):
    # one infinite rank among finite ones: infinite with its sign where up reads it, finite where it does not
    T, K, N, R = 40, 64, 32, 16
    off, ad = torch.tensor([0, T], dtype=torch.int32, device=cuda_dev), torch.tensor([0], dtype=torch.int32, device=cuda_dev)
    x, down, up = torch.zeros(T, K, dtype=FP16, device=cuda_dev), torch.zeros(1, R, K, dtype=FP16, device=cuda_dev), torch.zeros(1, N, R, dtype=FP16, device=cuda_dev)
    x[:, 0], x[7, 0] = 1.0, float("inf")
    down[0, 0, 0], up[0, :, 0] = 1.0, 1.0
    up[0, 5, 0] = -2.0
    out = lora_batched(x, down, up, off, ad, _impl=impl)
    rest = [t for t in range(T) if t != 7]
    keep = [n for n in range(N) if n != 5]
    assert (out[rest][:, keep] == 1).all() and (out[rest, 5] == -2).all()
    # row 7: inf x 0 in the other ranks of down is NaN by the definition too
    assert not out[7].isfinite().any()


def test_h_has_room_for_the_rows_powers():
    lib, a = L.lib(), L.LoraArgs(T=5, K=64, N=32, R=16, A=1, requests=1, dtype=1)  # float16
    rows = 5 * 16 * 2  # bytes of a part
    assert lib.nb_lora_h_bytes(a) >= 2 * rows + 5 * 4
    assert lib.nb_lora_h_bytes(L.LoraArgs(T=5, K=64, N=32, R=16, A=1, requests=1, dtype=0)) >= 3 * rows
    a.R = 24
    assert lib.nb_lora_h_bytes(a) == 0  # refused sizes


@gpu
@pytest.mark.parametrize("impl", IMPLS.values(), ids=IMPLS)
@pytest.mark.parametrize("R", [16, 32, 64, 128])
@pytest.mark.parametrize("T", [2, 70, 300])
def test_bfloat16_keeps_all_bits_of_h(cuda_dev, T, R, impl):
    # two ranks (rows) whose first sixteen bits cancel: what is left is the last eight of h (g), exact in every step
    K, N = 64, 96
    off, ad = torch.tensor([0, T], dtype=torch.int32, device=cuda_dev), torch.tensor([0], dtype=torch.int32, device=cuda_dev)
    z = lambda *s: torch.zeros(*s, dtype=BF16, device=cuda_dev)  # noqa: E731
    digits, powers = (torch.tensor(v, dtype=BF16, device=cuda_dev) for v in ([0xAB, 0xCD, 0xEF], [2.0**16, 2.0**8, 1.0]))
    upper = powers * torch.tensor([-1.0, -1.0, 0.0], dtype=BF16, device=cuda_dev)
    x, down, up = z(T, K), z(1, R, K), z(1, N, R)
    x[:, 8:11] = digits
    down[0, 3, 8:11], down[0, R - 2, 8:11] = powers, upper  # h = 0xABCDEF and -0xABCD00
    up[0, :, 3], up[0, :, R - 2] = 1.0, 1.0
    assert (lora_batched(x, down, up, off, ad, _impl=impl) == 0xEF).all()
    # g likewise through dy and up, read back by dx; and the sums over two rows
    dy, up = z(T, N), z(1, N, R)
    dy[:, 40:43] = digits
    up[0, 40:43, 3], up[0, 40:43, R - 2] = powers, upper
    down = z(1, R, K)
    down[0, 3], down[0, R - 2] = 1.0, 1.0
    leaves = [t.requires_grad_(True) for t in (z(T, K), down, up)]
    (dx,) = torch.autograd.grad(lora_batched(*leaves, off, ad, _impl=impl), leaves[:1], dy)
    assert (dx == 0xEF).all()
    x, dy, down, up = z(T, K), z(T, N), z(1, R, K), z(1, N, R)
    x[0, 8:11], x[T - 1, 8:11] = digits, digits * torch.tensor([-1.0, -1.0, 0.0], dtype=BF16, device=cuda_dev)
    down[0, 5, 8:11] = powers
    dy[0, 7], dy[T - 1, 7] = 1.0, 1.0
    leaves = [t.requires_grad_(True) for t in (x, down, up)]
    (dup,) = torch.autograd.grad(lora_batched(*leaves, off, ad, _impl=impl), leaves[2:], dy)
    assert dup[0, 7, 5] == 0xEF and dup.count_nonzero() == 1
    x, dy, down, up = z(T, K), z(T, N), z(1, R, K), z(1, N, R)
    dy[0, 40:43], dy[T - 1, 40:43] = digits, digits * torch.tensor([-1.0, -1.0, 0.0], dtype=BF16, device=cuda_dev)
    up[0, 40:43, 5] = powers
    x[0, 9], x[T - 1, 9] = 1.0, 1.0
    leaves = [t.requires_grad_(True) for t in (x, down, up)]
    (ddown,) = torch.autograd.grad(lora_batched(*leaves, off, ad, _impl=impl), leaves[1:2], dy)
    assert ddown[0, 5, 9] == 0xEF and ddown.count_nonzero() == 1


@gpu
@pytest.mark.parametrize("impl", IMPLS.values(), ids=IMPLS)
@pytest.mark.parametrize("R", [16, 48, 64, 80, 128])
@pytest.mark.parametrize("T,offsets,adapters", [(21, [0, 9, 21], [1, 0]), (700, [0, 330, 690], [0, 1])])
def test_bfloat16_differs_by_fp32_roundings_alone(cuda_dev, R, T, offsets, adapters, impl):
    p = make(cuda_dev, T, 328, 264, R, 2, BF16, up=0.1, seed=R)
    check(p, offsets, adapters, impl)


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_long_contractions_do_not_drift(cuda_dev, dtype):
    # the tensor cores' accumulators truncate: sums of one sign fall short by up to 2^-23 of what is there in each step.  A chain
    # of 64 steps loses at most sum(i / 64) = 32.5 of those, a product of 16 terms is rounded once (2 more allowed), and the
    # nine chains are added with rounding.  One chain of 576 steps loses some 1.5e-5.
    T, K, N, R = 9600, 9216, 64, 64
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    x, down = (torch.rand(s, generator=g, device=cuda_dev).add_(0.5).to(dtype) for s in ((T, K), (1, R, K)))
    up, out = torch.zeros(1, N, R, dtype=dtype, device=cuda_dev), torch.empty(T, N, dtype=dtype, device=cuda_dev)
    off, ad = torch.tensor([0, T], dtype=torch.int32, device=cuda_dev), torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    parts = 2 if dtype == FP16 else 3
    a = L.LoraArgs(T=T, K=K, N=N, R=R, A=1, requests=1, dtype=1 if dtype == FP16 else 0, stride_x=K, stride_out=N,
                   **{n: t.data_ptr() for n, t in (("x", x), ("down", down), ("up", up), ("offsets", off), ("adapters", ad), ("out", out))})
    h = torch.empty(L.lib().nb_lora_h_bytes(a), dtype=torch.uint8, device=cuda_dev)
    a.h = h.data_ptr()
    assert L.lib().nb_lora_forward(a, L.stream_of(x)) == L.NB_OK
    value = h[: parts * T * R * 2].view(dtype).view(parts, T, R).double().sum(0)
    if dtype == FP16:
        value = value * h[parts * T * R * 2 :].view(torch.float32)[:T].double()[:, None]
    want = x.double() @ down[0].double().t()
    assert ((value - want).abs() / want).max() <= 35 * 2.0**-23 + 16 * F32 + (0 if dtype == BF16 else 2.0**-22)


@gpu
@pytest.mark.parametrize("impl", [L.IMPL_TCGEN05, L.IMPL_AUTO])
def test_long_sums_over_rows_do_not_drift(cuda_dev, impl):
    # all rows but the last three add up with one sign, and these take the sum off again up to its last bit, so that the error of
    # a sum of 9213 terms is what is left.  Chains of at most 48 steps: sum(i / 48) = 24.5 truncations of 2^-23, nine more where
    # the sum is taken off, and some twenty rounded additions; one chain of 432 steps loses some 1.3e-5.
    T, K, N, R = 9216, 64, 9216, 64
    off, ad = torch.tensor([0, T], dtype=torch.int32, device=cuda_dev), torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    x, down = torch.zeros(T, K, dtype=BF16, device=cuda_dev), torch.zeros(1, R, K, dtype=BF16, device=cuda_dev)
    x[:, 8:11], down[0, 3, 8:11] = torch.tensor([0xAB, 0xCD, 0xEF]), torch.tensor([2.0**16, 2.0**8, 1.0])  # h = 0xABCDEF
    up = torch.zeros(1, N, R, dtype=BF16, device=cuda_dev, requires_grad=True)
    dy = torch.rand(T, N, generator=torch.Generator(device=cuda_dev).manual_seed(0), device=cuda_dev).add_(0.5).to(BF16)
    total = dy[:-3].sum(0, dtype=torch.float64)
    left = total.clone()
    for t in (T - 3, T - 2, T - 1):
        dy[t] = -left.to(BF16)
        left += dy[t].double()
    (dup,) = torch.autograd.grad(lora_batched(x, down, up, off, ad, _impl=impl), up, dy)
    off_by = (dup[0, :, 3].double() - left * 0xABCDEF).abs() / (total * 0xABCDEF)
    assert off_by.max() <= 34 * 2.0**-23 + 20 * F32
