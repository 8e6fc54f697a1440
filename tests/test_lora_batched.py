"""
Adapters of many requests beside a shared projection, against the definition in 64 bits.

Tolerances: one rounding of the output (half a step), fp32 sums (one 2^-24 per term, taken over the longest chain), and the
two-part 16-bit operands (half a step of T squared, relative to each term of the second product).
"""

import pytest
import torch

from nunchaku_rocm_b200 import _lib as L
from nunchaku_rocm_b200.ops.lora import lora_batched

F32 = 2.0**-24
BF16, FP16 = torch.bfloat16, torch.float16
gpu = pytest.mark.gpu


def half(dt):
    return torch.finfo(dt).eps / 2


def within(got, ref, tol):
    off = ((got.double() - ref).abs() - tol).max().item() if ref.numel() else -1.0
    assert off <= 0, f"over the tolerance by {off:.3g} (largest difference {(got.double() - ref).abs().max().item():.3g})"


def make(dev, T, K, N, R, A, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s, k=1.0: (torch.randn(s, generator=g, device=dev) * k).to(dtype)  # noqa: E731
    return {"x": n(T, K), "base": n(T, N), "down": n(A, R, K, k=K**-0.5), "up": n(A, N, R, k=R**-0.5), "dy": n(T, N),
            "scale": torch.rand(A, generator=g, device=dev) + 0.5}


def index(dev, offsets, adapters):
    return torch.tensor(offsets, dtype=torch.int32, device=dev), torch.tensor(adapters, dtype=torch.int32, device=dev)


def reference(p, offsets, adapters, scale=True, base=True):
    """{name: (value, tolerance)} in 64 bits, one request after the other."""
    d = {k: v.double() for k, v in p.items()}
    dt, (T, K), (A, N, R) = p["x"].dtype, p["x"].shape, p["up"].shape
    out, dx = (d["base"].clone() if base else torch.zeros_like(d["base"])), torch.zeros_like(d["x"])
    dd, du = torch.zeros_like(d["down"]), torch.zeros_like(d["up"])
    t = {"out": F32 * out.abs(), "dx": torch.zeros_like(dx), "ddown": torch.zeros_like(dd), "dup": torch.zeros_like(du)}
    two = half(dt) ** 2  # what is left of a value after its two 16-bit parts
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps  # the parts of very small values are subnormal
    for i, a in enumerate(adapters):
        rows = slice(offsets[i], offsets[i + 1])
        n = offsets[i + 1] - offsets[i]
        if n == 0 or not 0 <= a < A:
            continue
        s = d["scale"][a] if scale else 1.0
        x, dy, D, U = d["x"][rows], d["dy"][rows], d["down"][a], d["up"][a]
        h, g = s * x @ D.t(), s * dy @ U
        eh = F32 * (K + 4) * (s * x.abs() @ D.t().abs()) + two * h.abs() + tiny
        eg = F32 * (N + 4) * (s * dy.abs() @ U.abs()) + two * g.abs() + tiny
        out[rows] += h @ U.t()
        t["out"][rows] += eh @ U.t().abs() + F32 * (R + 4) * (h.abs() @ U.t().abs())
        dx[rows] = g @ D
        t["dx"][rows] = eg @ D.abs() + F32 * (R + 4) * (g.abs() @ D.abs())
        dd[a] += g.t() @ x
        t["ddown"][a] += eg.t() @ x.abs() + F32 * (T + 4) * (g.t().abs() @ x.abs())
        du[a] += dy.t() @ h
        t["dup"][a] += dy.t().abs() @ eh + F32 * (T + 4) * (dy.t().abs() @ h.abs())
    return {k: (v, t[k] + half(dt) * (v.abs() + t[k]) + torch.finfo(dt).smallest_normal) for k, v in {"out": out, "dx": dx, "ddown": dd, "dup": du}.items()}


IMPLS = {"generic": L.IMPL_GENERIC, "tcgen05": L.IMPL_TCGEN05}


def check(dev, p, offsets, adapters, scale=True, base=True):
    for impl in IMPLS.values():
        check_impl(dev, p, offsets, adapters, scale, base, impl)
    assert L.device_status(dev) == 0


def check_impl(dev, p, offsets, adapters, scale, base, impl):
    off, ad = index(dev, offsets, adapters)
    ref = reference(p, offsets, adapters, scale, base)
    kw = {"base": p["base"] if base else None, "scale": p["scale"] if scale else None, "_impl": impl}
    plain = lora_batched(p["x"], p["down"], p["up"], off, ad, **kw)
    within(plain, *ref["out"])
    leaves = [p[k].detach().requires_grad_(True) for k in ("x", "down", "up")]
    if base:
        kw["base"] = p["base"].detach().requires_grad_(True)
        leaves.append(kw["base"])
    out = lora_batched(*leaves[:3], off, ad, **kw)
    assert torch.equal(out, plain)
    got = torch.autograd.grad(out, leaves, p["dy"])
    for name, t in zip(("dx", "ddown", "dup"), got):
        within(t, *ref[name])
    if base:
        assert torch.equal(got[3], p["dy"])
    again = torch.autograd.grad(lora_batched(*leaves[:3], off, ad, **kw), leaves, p["dy"])
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # fixed order of the sums
    covered = torch.zeros(len(p["x"]), dtype=torch.bool, device=dev)
    for i, a in enumerate(adapters):
        if 0 <= a < len(p["down"]):
            covered[offsets[i] : offsets[i + 1]] = True
    assert torch.equal(plain[~covered], p["base"][~covered] if base else torch.zeros_like(plain[~covered])) and not got[0][~covered].any()


# --------------------------------------------------------------------------------------------------------------- refusals
def test_refuses():
    x, down, up = torch.zeros(4, 64, dtype=BF16), torch.zeros(2, 16, 64, dtype=BF16), torch.zeros(2, 32, 16, dtype=BF16)
    off, ad = torch.tensor([0, 4], dtype=torch.int32), torch.tensor([0], dtype=torch.int32)
    base = torch.zeros(4, 32, dtype=BF16)
    bad = [(x.float(), down, up, off, ad), (x, down.to(FP16), up, off, ad), (x, down, up[:1], off, ad), (x, down[0], up, off, ad),
           (x[:, :56], down, up, off, ad), (x, down, up, off.long(), ad), (x, down, up, off, ad.long()), (x, down, up, off[:1], ad),
           (x, down, up, off[None], ad), (x, down[:0], up[:0], off, ad)]
    for args in bad:
        with pytest.raises(ValueError):
            lora_batched(*args)
    for kw in ({"base": base[:3]}, {"base": base.float()}, {"scale": torch.ones(3)}, {"scale": torch.ones(2, dtype=BF16)},
               {"scale": torch.ones(2, requires_grad=True)}, {"out": torch.zeros(4, 40, dtype=BF16)}, {"out": torch.zeros(4, 34, dtype=BF16)[:, :32]}):
        with pytest.raises(ValueError):
            lora_batched(x, down, up, off, ad, **kw)
    with pytest.raises(ValueError, match="overlap"):
        lora_batched(x, down, up, off, ad, out=torch.zeros(1, 32, dtype=BF16).expand(4, 32))
    for r, k, n in ((8, 64, 32), (144, 64, 32), (16, 60, 32), (16, 64, 36), (0, 64, 32)):
        with pytest.raises(NotImplementedError):
            lora_batched(torch.zeros(4, k, dtype=BF16), torch.zeros(1, r, k, dtype=BF16), torch.zeros(1, n, r, dtype=BF16), off, ad)
    with pytest.raises(RuntimeError, match="no CPU path"):
        lora_batched(x, down, up, off, ad, base=base)


def test_the_c_entries_refuse_bad_sizes():
    lib = L.lib()
    a = L.LoraArgs(T=4, K=64, N=32, R=16, A=1, requests=1, dtype=0)
    assert lib.nb_lora_forward(a, None) == L.NB_ERR_INVALID  # null pointers
    a.R = 24
    assert lib.nb_lora_forward(a, None) == L.NB_ERR_UNSUPPORTED
    a.R, a.K = 16, 60
    assert lib.nb_lora_backward(a, None) == L.NB_ERR_UNSUPPORTED
    a.K, a.T = 64, 1 << 29
    assert lib.nb_lora_forward(a, None) == L.NB_ERR_TOO_LARGE
    a.T, a.dtype = 4, 2
    assert lib.nb_lora_forward(a, None) == L.NB_ERR_INVALID
    a.T, a.dtype = 0, 0
    assert lib.nb_lora_forward(a, None) == L.NB_OK and lib.nb_lora_workspace_bytes(a) == 0


# --------------------------------------------------------------------------------------------------------------- on the GPU
@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("R", [16, 32, 48, 64, 96, 128])
def test_ranks_and_types(cuda_dev, dtype, R):
    p = make(cuda_dev, 200, 520, 328, R, 3, dtype, seed=R)
    check(cuda_dev, p, [0, 70, 71, 190], [2, 0, 2])


@gpu
@pytest.mark.parametrize("K,N", [(8, 8), (64, 128), (72, 136), (1024, 40), (40, 1032), (2048, 2048)])
@pytest.mark.parametrize("T,offsets,adapters", [
    (1, [0, 1], [0]),
    (16, list(range(17)), [i % 5 - 1 for i in range(16)]),          # one row each, some without an adapter
    (130, [0, 64, 128, 130], [1, 0, 1]),                            # borders on tile borders
    (257, [3, 3, 20, 20, 101, 250], [0, 3, 7, 1, 2]),               # empty requests, an unknown adapter, rows before and behind
    (97, [97, 97], [0]), (65, [0, 0, 0, 65], [0, 1, 2]), (40, [0], []),
])
def test_sizes_and_borders(cuda_dev, K, N, T, offsets, adapters):
    check(cuda_dev, make(cuda_dev, T, K, N, 32, 4, BF16, seed=T), offsets, adapters)


@gpu
@pytest.mark.parametrize("T,requests", [(3000, 7), (2049, 130), (700, 300), (4500, 2)])
def test_many_rows_and_requests(cuda_dev, T, requests):
    g = torch.Generator().manual_seed(T)
    cuts = sorted(torch.randint(0, T + 1, (requests - 1,), generator=g).tolist())
    adapters = torch.randint(-1, 6, (requests,), generator=g).tolist()
    check(cuda_dev, make(cuda_dev, T, 1280, 384, 16, 6, FP16, seed=T), [0, *cuts, T], adapters)


@gpu
@pytest.mark.parametrize("R,K,N,offsets,adapters", [
    (16, 64, 6016, [0, 2944, 6000], [1, 0]),         # long walks over the columns, whole and partial tiles
    (64, 4096, 72, [0, 1000, 1003, 6000], [0, -1, 1]),  # long contractions
    (128, 72, 4104, [0, 6000], [0]),
])
def test_long_rows_and_columns(cuda_dev, R, K, N, offsets, adapters):
    check(cuda_dev, make(cuda_dev, 6000, K, N, R, 2, BF16, seed=R), offsets, adapters)


@gpu
def test_without_base_and_scale(cuda_dev):
    p = make(cuda_dev, 90, 128, 256, 64, 2, BF16)
    check(cuda_dev, p, [10, 50, 80], [1, 0], scale=False, base=False)
    check(cuda_dev, p, [10, 50, 80], [1, 0], scale=True, base=False)
    check(cuda_dev, p, [10, 50, 80], [1, 0], scale=False, base=True)


@gpu
def test_layouts_and_out(cuda_dev):
    p = make(cuda_dev, 96, 128, 256, 32, 2, BF16)
    off, ad = index(cuda_dev, [0, 33, 96], [1, 0])
    want = lora_batched(p["x"], p["down"], p["up"], off, ad, base=p["base"], scale=p["scale"])
    wide = torch.zeros(96, 3 * 128, dtype=BF16, device=cuda_dev)
    wide[:, 128:256] = p["x"]
    assert torch.equal(lora_batched(wide[:, 128:256], p["down"], p["up"], off, ad, base=p["base"], scale=p["scale"]), want)
    odd = torch.zeros(96, 129, dtype=BF16, device=cuda_dev)
    odd[:, 1:] = p["x"]
    got = lora_batched(odd[:, 1:].view(2, 48, 128), p["down"], p["up"], off, ad, base=p["base"].view(2, 48, 256), scale=p["scale"])
    assert torch.equal(got.view(96, 256), want)
    t = p["x"].view(2, 48, 128).transpose(0, 1).contiguous().transpose(0, 1)  # rows not evenly strided
    assert torch.equal(lora_batched(t, p["down"], p["up"], off, ad, base=p["base"].view(2, 48, 256), scale=p["scale"]).view(96, 256), want)
    fat = torch.full((96, 3 * 256), 7.0, dtype=BF16, device=cuda_dev)  # out: columns of a larger buffer, in place
    fat[:, 256:512] = p["base"]
    got = lora_batched(p["x"], p["down"], p["up"], off, ad, base=fat[:, 256:512], scale=p["scale"], out=fat[:, 256:512])
    assert got.data_ptr() == fat[:, 256:512].data_ptr() and torch.equal(fat[:, 256:512], want)
    assert (fat[:, :256] == 7).all() and (fat[:, 512:] == 7).all()
    # gradients through views, a broadcast gradient, and a shared base
    x = wide.detach().requires_grad_(True)
    row = p["base"][:1].detach().requires_grad_(True)
    y = lora_batched(x[:, 128:256], p["down"], p["up"], off, ad, base=row.expand(96, 256))
    dx, drow = torch.autograd.grad(y.sum(), (x, row))
    ones = {**p, "dy": torch.ones_like(p["dy"])}
    within(dx[:, 128:256], *reference(ones, [0, 33, 96], [1, 0], scale=False)["dx"])
    assert not dx[:, :128].any() and (drow == 96).all()


@gpu
def test_out_is_an_in_place_change(cuda_dev):
    p = make(cuda_dev, 40, 64, 64, 16, 1, BF16)
    off, ad = index(cuda_dev, [0, 40], [0])
    w = torch.ones(40, 64, dtype=BF16, device=cuda_dev, requires_grad=True)
    y = (w * p["base"]).sum()  # keeps base for w's gradient
    lora_batched(p["x"], p["down"], p["up"], off, ad, base=p["base"], out=p["base"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with pytest.raises(ValueError, match="gradient"):
        lora_batched(p["x"], p["down"], p["up"], off, ad, out=w)


@gpu
def test_captured_training_step(cuda_dev):
    p = make(cuda_dev, 300, 256, 384, 32, 3, FP16)
    off, ad = index(cuda_dev, [0, 120, 120, 300], [0, 1, 2])

    def step():
        leaves = [p[k].detach().requires_grad_(True) for k in ("x", "down", "up")]
        out = lora_batched(*leaves, off, ad, base=p["base"], scale=p["scale"])
        return (out.detach(), *torch.autograd.grad(out, leaves, p["dy"]))

    step()
    s, gr = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(gr, stream=s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    ad.copy_(torch.tensor([2, 0, 2], dtype=torch.int32))
    off.copy_(torch.tensor([0, 7, 190, 290], dtype=torch.int32))
    p["dy"].neg_()
    for _ in range(2):
        gr.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ref = reference(p, [0, 7, 190, 290], [2, 0, 2])
    for name, t in zip(("out", "dx", "ddown", "dup"), got):
        within(t, *ref[name])


@gpu
def test_rows_stay_apart_when_values_are_not_finite(cuda_dev):
    p = make(cuda_dev, 70, 64, 64, 16, 2, BF16)
    clean = lora_batched(p["x"], p["down"], p["up"], *index(cuda_dev, [0, 20, 70], [0, 1]), base=p["base"])
    p["x"][25, 3] = float("nan")
    p["x"][3, 0] = float("inf")
    got = lora_batched(p["x"], p["down"], p["up"], *index(cuda_dev, [0, 20, 70], [0, 1]), base=p["base"])
    others = [i for i in range(70) if i not in (3, 25)]
    assert got[25].isnan().all() and not torch.isfinite(got[3]).any() and torch.equal(got[others], clean[others])
    # masked rows: their NaN reaches neither the output nor the gradients of the adapters
    x, down, up = (p[k].detach().requires_grad_(True) for k in ("x", "down", "up"))
    out = lora_batched(x, down, up, *index(cuda_dev, [4, 20, 26, 70], [0, -1, 1]), base=p["base"])
    dx, dd, du = torch.autograd.grad(out, (x, down, up), p["dy"])
    assert torch.isfinite(out).all() and torch.isfinite(dx).all() and torch.isfinite(dd).all() and torch.isfinite(du).all()
    # an adapter that is not finite reaches the rows of its requests alone
    p = make(cuda_dev, 70, 64, 64, 16, 2, FP16)
    p["up"][1] = float("inf")
    got = lora_batched(p["x"], p["down"], p["up"], *index(cuda_dev, [0, 20, 70], [0, 1]), base=p["base"])
    assert torch.isfinite(got[:20]).all() and not torch.isfinite(got[20:]).any()
    # h beyond fp16: infinite with its sign, as one 16-bit rounding of it would be, not NaN
    x = torch.full((1, 64), 6e4, dtype=FP16, device=cuda_dev)
    down, up = torch.ones(1, 16, 64, dtype=FP16, device=cuda_dev), torch.full((1, 8, 16), -1.0, dtype=FP16, device=cuda_dev)
    assert (lora_batched(x, down, up, *index(cuda_dev, [0, 1], [0])) == float("-inf")).all()


@gpu
def test_gradients_against_differences(cuda_dev):
    # the output is linear in each of x, down and up: a difference over a step of the tensors' own size has no truncation
    # error, only one rounding of each output element on each side
    p = make(cuda_dev, 60, 64, 48, 16, 2, FP16)
    off, ad = index(cuda_dev, [0, 25, 60], [1, 0])
    leaves = {k: p[k].detach().requires_grad_(True) for k in ("x", "down", "up")}
    grads = dict(zip(leaves, torch.autograd.grad(lora_batched(*leaves.values(), off, ad, scale=p["scale"]), list(leaves.values()), p["dy"])))
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    for k in leaves:
        d = (torch.randn(p[k].shape, generator=g, device=cuda_dev) * p[k].std()).to(FP16)
        side = [(p[k].float() + s * d.float()).to(FP16) for s in (1, -1)]
        step = (side[0].double() - side[1].double()) / 2  # what the rounded arguments really differ by
        y = [lora_batched(*[v if n == k else p[n] for n in leaves], off, ad, scale=p["scale"]).double() for v in side]
        num = ((y[0] - y[1]) / 2 * p["dy"].double()).sum()
        tol = (half(FP16) * 1.01 * (y[0].abs() + y[1].abs()) / 2 * p["dy"].double().abs()).sum() + (half(FP16) * 1.01 * grads[k].double().abs() * step.abs()).sum()
        assert abs(num - (grads[k].double() * step).sum()) <= tol


@gpu
def test_captured_with_changing_requests(cuda_dev):
    p = make(cuda_dev, 150, 256, 384, 32, 3, BF16)
    off, ad = index(cuda_dev, [0, 50, 100, 150], [0, 1, 2])
    lora_batched(p["x"], p["down"], p["up"], off, ad, base=p["base"], scale=p["scale"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                graphs.append((gr, lora_batched(p["x"], p["down"], p["up"], off, ad, base=p["base"], scale=p["scale"])))
    torch.cuda.current_stream().wait_stream(s)
    off.copy_(torch.tensor([5, 5, 77, 140], dtype=torch.int32))
    ad.copy_(torch.tensor([2, 2, -1], dtype=torch.int32))
    p["x"].mul_(-1.5)
    torch.cuda.synchronize()
    for gr, _ in graphs:  # side by side: each has scratch of its own
        with torch.cuda.stream(torch.cuda.Stream()):
            gr.replay()
    torch.cuda.synchronize()
    want = lora_batched(p["x"], p["down"], p["up"], off, ad, base=p["base"], scale=p["scale"])
    assert all(torch.equal(out, want) for _, out in graphs)


@gpu
def test_on_a_stream_of_its_own(cuda_dev):
    p = make(cuda_dev, 500, 512, 512, 32, 2, BF16)
    off, ad = index(cuda_dev, [0, 250, 500], [0, 1])
    want = lora_batched(p["x"], p["down"], p["up"], off, ad, base=p["base"])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [lora_batched(p["x"], p["down"], p["up"], off, ad, base=p["base"]) for _ in range(8)]
    s.synchronize()
    assert all(torch.equal(t, want) for t in got)


@gpu
@pytest.mark.parametrize("impl", IMPLS.values(), ids=IMPLS)
def test_more_than_2_31_elements(cuda_dev, impl):
    # the last rows, whose offsets pass 32 bits, against 64 bits
    T, K, N, tail = 3_000_000, 16, 728, 200
    assert T * N > 1 << 31
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    p = make(cuda_dev, tail, K, N, 16, 2, BF16)
    x, dy = torch.zeros(T, K, dtype=BF16, device=cuda_dev), torch.zeros(T, N, dtype=BF16, device=cuda_dev)
    x[:-tail].normal_(generator=g)
    x[-tail:], dy[-tail:] = p["x"], p["dy"]
    off, ad = index(cuda_dev, [0, 1_000_001, T - 90, T], [1, 0, 1])
    x.requires_grad_(True)
    out = lora_batched(x, p["down"], p["up"], off, ad, _impl=impl)
    dx, = torch.autograd.grad(out, x, dy)
    ref = reference(p, [0, tail - 90, tail], [0, 1], scale=False, base=False)
    within(out[-tail:], *ref["out"])
    within(dx[-tail:], *ref["dx"])
    assert L.device_status(cuda_dev) == 0


@gpu
@pytest.mark.parametrize("R", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("K,N", [(8, 8), (40, 264), (2048, 18432), (12288, 72)])
@pytest.mark.parametrize("T,offsets,adapters", [
    (1, [0, 1], [0]),
    (17, [0, 16, 17], [1, 0]),
    (24, list(range(25)), [i % 4 - 1 for i in range(24)]),
    (70, [2, 2, 3, 20, 20, 69], [2, 0, -1, 1, 2]),
])
def test_few_rows(cuda_dev, R, K, N, T, offsets, adapters):
    # the forward pass in one kernel, and the adapters' part added in place
    p = make(cuda_dev, T, K, N, R, 3, BF16 if R % 32 else FP16, seed=T + R)
    check_impl(cuda_dev, p, offsets, adapters, True, True, L.IMPL_AUTO)
    out = p["base"].clone()
    lora_batched(p["x"], p["down"], p["up"], *index(cuda_dev, offsets, adapters), base=out, scale=p["scale"], out=out)
    assert torch.equal(out, lora_batched(p["x"], p["down"], p["up"], *index(cuda_dev, offsets, adapters), base=p["base"], scale=p["scale"]))


@gpu
@pytest.mark.parametrize("K,N", [(520, 328), (72, 136), (40, 1032)])
@pytest.mark.parametrize("R", [16, 32, 48, 64, 96, 128])
def test_more_than_a_few_rows(cuda_dev, R, K, N):
    # too many for the one kernel: the shrink and the expand of their own, with odd sizes and short items among long ones
    p = make(cuda_dev, 1301, K, N, R, 3, BF16 if R % 32 else FP16, seed=R + N)
    check(cuda_dev, p, [3, 3, 20, 21, 149, 640, 640, 1290], [1, 0, 2, -1, 1, 5, 2])
