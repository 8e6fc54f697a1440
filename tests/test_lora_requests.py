"""
Adapters of several requests on the layers of a model, and the adapter, norm and rotary operators in a run together.

The layers' tests compare with the layer without adapters plus the adapters' product in 64 bits: one rounding of the base
output and one of the sum (half a step each), and the operator's own fp32 error, far below.
"""

import pytest
import torch
from torch import nn

from nunchaku_rocm_b200.lora import attach_lora, attach_lora_batch, detach_lora_batch, lora_requests, stack_loras
from nunchaku_rocm_b200.lora import batched
from nunchaku_rocm_b200.models.embeddings import flux_pos_embed, qwen_image_ids
from nunchaku_rocm_b200.models.linear import AWQW4A16Linear, SVDQW4A4Linear

gpu = pytest.mark.gpu
BF16 = torch.bfloat16
HALF = torch.finfo(BF16).eps / 2


def pair(r, n_in, n_out, seed, dev="cpu", dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(r, n_in, generator=g) * n_in**-0.5).to(dtype).to(dev), (torch.randn(n_out, r, generator=g) * 0.5 * r**-0.5).to(dtype).to(dev))


def layer(cin, cout, dev, seed, precision="int4", unsigned=False):
    g = torch.Generator().manual_seed(seed)
    lin = SVDQW4A4Linear(cin, cout, rank=32, precision=precision, act_unsigned=unsigned, torch_dtype=BF16)
    with torch.no_grad():
        lin.qweight.copy_(torch.randint(-128, 128, lin.qweight.shape, dtype=torch.int8, generator=g))
        lin.wscales.copy_((torch.rand(lin.wscales.shape, generator=g) * 0.015 + 0.005).to(lin.wscales.dtype))
        lin.bias.copy_((torch.randn(cout, generator=g) * 0.1).to(BF16))
        lin.smooth_factor.copy_((torch.rand(cin, generator=g) + 0.5).to(BF16))
        lin.proj_down.copy_((torch.randn(cin, 32, generator=g) * 0.05).to(BF16))
        lin.proj_up.copy_((torch.randn(cout, 32, generator=g) * 0.05).to(BF16))
    return lin.to(dev)


def delta(x, stack, scale, adapters):
    """The adapters' part of the output in 64 bits, sample by sample."""
    down, up = (t.double() for t in stack)
    out = torch.zeros(*x.shape[:-1], up.shape[1], dtype=torch.float64, device=x.device)
    for b, a in enumerate(adapters):
        if 0 <= a < len(down):
            out[b] = (1.0 if scale is None else scale[a]) * ((x[b].double() @ down[a].t()) @ up[a].t())
    return out


def near(got, base, d):
    tol = HALF * (base.double().abs() + got.double().abs()) + 2.0**-15 * (d.abs() + 1)
    off = ((got.double() - base.double() - d).abs() - tol).max().item()
    assert off <= 0, off


# ------------------------------------------------------------------------------------------------------------------- CPU
def test_stack_loras_pads_ranks_and_adds_lists():
    a, b, c = pair(4, 64, 32, 1), pair(20, 64, 32, 2), pair(9, 64, 32, 3)
    down, up = stack_loras([a, [b, c]])
    assert down.shape == (2, 32, 64) and up.shape == (2, 32, 32)
    assert torch.equal(down[0, :4], a[0]) and not down[0, 4:].any() and torch.equal(up[1, :, 20:29], c[1]) and not up[1, :, 29:].any()
    for bad in ([], [a, pair(4, 60, 32, 1)], [(a[0], a[1][:, :3])]):
        with pytest.raises(ValueError):
            stack_loras(bad)


def test_attach_and_requests_refuse():
    lin = layer(64, 128, "cpu", 0)
    for bad in ([pair(4, 60, 128, 1)], [pair(4, 64, 120, 1)], (torch.zeros(2, 8, 64), torch.zeros(2, 128, 8)), (torch.zeros(2, 16, 64), torch.zeros(3, 128, 16))):
        with pytest.raises(ValueError):
            attach_lora_batch(lin, bad)
    with pytest.raises(ValueError):
        attach_lora_batch(lin, [pair(4, 64, 128, 1)], scale=[1.0, 2.0])
    with pytest.raises(NotImplementedError):
        attach_lora_batch(lin, [pair(129, 64, 128, 1)])
    with pytest.raises(ValueError):
        attach_lora_batch(nn.GELU(), [pair(4, 64, 128, 1)])
    assert not hasattr(lin, "_lora_stack")
    for bad in (torch.zeros(2), torch.zeros(2, dtype=torch.int64), torch.zeros(1, 2, dtype=torch.int32)):
        with pytest.raises(ValueError), lora_requests(bad):
            pass
    plain = nn.Linear(16, 8)
    attach_lora_batch(plain, [pair(2, 16, 8, 1, dtype=torch.float32)])
    x = torch.randn(3, 16)
    y = plain(x)  # no requests are active: the stack is not used
    with pytest.raises(ValueError, match="samples"), lora_requests(torch.zeros(2, dtype=torch.int32)):
        plain(x)
    with pytest.raises(ValueError, match="samples"), lora_requests(torch.zeros(2, dtype=torch.int32)):
        plain(input=x)  # found by name too
    detach_lora_batch(plain)
    detach_lora_batch(plain)
    with lora_requests(torch.zeros(2, dtype=torch.int32)):
        assert torch.equal(plain(x), y)


def test_qwen_image_ids():
    ids = qwen_image_ids(3, 2, 5, 4)
    assert ids.shape == (43, 3) and ids[:3].tolist() == [[2, 2, 2], [3, 3, 3], [4, 4, 4]]
    assert ids[3].tolist() == [0, -3, -2] and ids[-1].tolist() == [1, 1, 1]


def test_a_stack_follows_its_module():
    lin = nn.Linear(16, 8)
    attach_lora_batch(lin, [pair(2, 16, 8, 1, dtype=torch.float32)], scale=[0.5])
    x = torch.zeros(3, 16, dtype=torch.float64, device="cpu")
    with torch.inference_mode():
        down, up, scale = batched._stack_on(lin, x)
    assert lin._lora_stack == (down, up) and down.dtype == up.dtype == x.dtype and not down.is_inference() and scale is lin._lora_stack_scale
    assert batched._stack_on(lin, torch.zeros(1, 16, device="meta", dtype=BF16))[2].device.type == "meta"  # the scale moves too
    # leaves that are trained stay the module's stack: every step converts them with a graph of its own
    leaves = tuple(torch.zeros(s, requires_grad=True) for s in ((1, 16, 16), (1, 8, 16)))
    attach_lora_batch(lin, leaves)
    for _ in range(2):
        down, up, _ = batched._stack_on(lin, x)
        (down.sum() + up.sum()).backward()
    assert lin._lora_stack[0] is leaves[0] and (leaves[0].grad == 2).all() and (leaves[1].grad == 2).all()


def test_offsets_are_kept_for_each_stream_and_may_be_saved():
    cpu = torch.device("cpu")
    with torch.inference_mode():
        a = batched._even_offsets(3, 7, cpu, 1)
    assert a.tolist() == [0, 7, 14, 21] and a.dtype == torch.int32 and not a.is_inference()
    assert batched._even_offsets(3, 7, cpu, 1) is a and batched._even_offsets(3, 7, cpu, 2) is not a


# ------------------------------------------------------------------------------------------------------------------- GPU
@gpu
@pytest.mark.parametrize("precision", ["int4", "nvfp4"])
@pytest.mark.parametrize("S", [1, 37, 300])
def test_quantised_linear(cuda_dev, precision, S):
    lin = layer(256, 384, cuda_dev, 1, precision)
    pairs = [pair(8, 256, 384, 2, cuda_dev), pair(30, 256, 384, 3, cuda_dev)]
    x = torch.randn(3, S, 256, generator=torch.Generator().manual_seed(4)).to(BF16).to(cuda_dev)
    base = lin(x)
    attach_lora_batch(lin, pairs, scale=[0.5, 2.0])
    assert torch.equal(lin(x), base)  # outside of requests
    ids = torch.tensor([1, -1, 0], dtype=torch.int32, device=cuda_dev)
    with lora_requests(ids):
        y = lin(x)
        with lora_requests(ids.flip(0).contiguous()):  # innermost counts
            z = lin(x)
    near(y, base, delta(x, lin._lora_stack, [0.5, 2.0], [1, -1, 0]))
    near(z, base, delta(x, lin._lora_stack, [0.5, 2.0], [0, -1, 1]))
    assert torch.equal(y[1], base[1]) and torch.equal(lin(x), base)
    # with one adapter for all samples: the layer with that LoRA appended to its own branch, up to where that one rounds
    detach_lora_batch(lin)
    attach_lora(lin, [(pairs[0][0], pairs[0][1] * 0.5)])
    one = lin(x)
    assert ((one - z)[:1].float().norm() / one[:1].float().norm()) < 1e-2


@gpu
def test_modulation_and_plain_linears(cuda_dev):
    g = torch.Generator().manual_seed(0)
    awq = AWQW4A16Linear(128, 768, torch_dtype=BF16)
    with torch.no_grad():
        awq.qweight.copy_(torch.randint(-(2**31), 2**31 - 1, awq.qweight.shape, dtype=torch.int32, generator=g))
        awq.wscales.copy_((torch.rand(awq.wscales.shape, generator=g) * 0.01).to(BF16))
        awq.wzeros.zero_()
        awq.bias.zero_()
    awq = awq.to(cuda_dev)
    lin = nn.Linear(128, 768, dtype=BF16, device=cuda_dev)
    ids = torch.tensor([0, 1, -1, 1], dtype=torch.int32, device=cuda_dev)
    x = torch.randn(4, 128, generator=g).to(BF16).to(cuda_dev)
    with torch.no_grad():
        for m in (awq, lin):
            base = m(x)
            attach_lora_batch(m, [pair(16, 128, 768, 2), pair(3, 128, 768, 3)])
            with lora_requests(ids):
                near(m(x), base, delta(x, m._lora_stack, None, ids.tolist()))
            detach_lora_batch(m)
            with lora_requests(ids):
                assert torch.equal(m(x), base)


@gpu
@pytest.mark.parametrize("precision", ["int4", "nvfp4"])
def test_fused_operators(cuda_dev, precision):
    from types import SimpleNamespace

    from nunchaku_rocm_b200.ops.fused import fused_gelu_mlp, fused_qkv_norm_rottary
    from oracle import w4a4

    B, S, C = 2, 64, 256
    x = torch.randn(B, S, C, generator=torch.Generator().manual_seed(1)).to(BF16).to(cuda_dev)
    ids = torch.tensor([1, 0], dtype=torch.int32, device=cuda_dev)
    proj = layer(C, 3 * 256, cuda_dev, 2, precision)
    attach_lora_batch(proj, [pair(16, C, 768, 3), pair(16, C, 768, 4)])
    norm = SimpleNamespace(weight=torch.ones(128, dtype=BF16, device=cuda_dev))
    rot = flux_pos_embed(torch.randint(0, 30, (S, 3), device=cuda_dev))
    plain = fused_qkv_norm_rottary(x, proj, norm, norm, rot)
    with lora_requests(ids):
        raw = proj(x)
        out = fused_qkv_norm_rottary(x, proj, norm, norm, rot)
        buf = torch.empty(B * S, 768, dtype=BF16, device=cuda_dev)
        into = fused_qkv_norm_rottary(x, proj, norm, norm, rot, output=buf)
    assert torch.equal(into, out) and into.data_ptr() == buf.data_ptr() and not torch.equal(out, plain)
    one = torch.ones(128, dtype=BF16)
    ref = w4a4.qk_norm_rope(raw.view(-1, 768).float().cpu(), one, one, rot.cpu().reshape(S, 128).repeat(B, 1))
    assert w4a4.rel_fro(out.view(-1, 768).float().cpu(), ref.float()) < 1e-2

    fc1, fc2 = layer(C, 512, cuda_dev, 5, precision), layer(512, C, cuda_dev, 6, precision, unsigned=precision == "int4")
    plain = fused_gelu_mlp(x, fc1, fc2)
    attach_lora_batch(fc1, [pair(16, C, 512, 7), pair(16, C, 512, 8)])
    attach_lora_batch(fc2, [pair(16, 512, C, 9), pair(16, 512, C, 10)])
    none = torch.full((2,), -1, dtype=torch.int32, device=cuda_dev)
    with lora_requests(none):  # the separate kernels without an adapter: the fused result up to the 16-bit hidden tile
        assert w4a4.rel_fro(fused_gelu_mlp(x, fc1, fc2).float().cpu(), plain.float().cpu()) < 2e-2
    with lora_requests(ids):
        y = fused_gelu_mlp(x, fc1, fc2)
        hidden = torch.nn.functional.gelu(fc1(x), approximate="tanh")
    with lora_requests(ids):
        saved = fc2._lora_stack
        fc2._lora_stack = (saved[0], torch.zeros_like(saved[1]))
        near(y, fused_gelu_mlp(x, fc1, fc2), delta(hidden, saved, None, [1, 0]))
    assert torch.equal(fused_gelu_mlp(x, fc1, fc2), plain)


@gpu
def test_flux_block_serves_two_adapters_and_replays(cuda_dev):
    from nunchaku_rocm_b200.models.flux_dit import FluxDiT, FluxDiTConfig

    cfg = FluxDiTConfig(hidden=256, heads=2, n_double=1, n_single=1)
    model = FluxDiT(cfg, device=cuda_dev).random_init(3)
    B, S, St = 2, 48, 16
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    args = [torch.randn(*s, generator=g, device=cuda_dev).to(BF16) for s in ((B, S, 64), (B, St, 4096), (B, 768))]
    args += [torch.ones(B, device=cuda_dev) * 0.5, torch.zeros(S, 3, device=cuda_dev), torch.zeros(St, 3, device=cuda_dev)]
    with torch.no_grad():
        base = model(*args)
        layers = [m for m in model.modules() if isinstance(m, (SVDQW4A4Linear, AWQW4A16Linear))]
        for i, m in enumerate(layers):
            attach_lora_batch(m, [pair(8, m.in_features, m.out_features, 2 * i), pair(16, m.in_features, m.out_features, 2 * i + 1)])
        assert torch.equal(model(*args), base)

        def run(*adapters):
            with lora_requests(torch.tensor(adapters, dtype=torch.int32, device=cuda_dev)):
                return model(*args)

        both, first, second = run(0, 1), run(0, 0), run(1, 1)
        assert torch.equal(both[0], first[0]) and torch.equal(both[1], second[1])  # a sample does not see the others'
        assert not torch.equal(first[0], base[0]) and not torch.equal(first, second)
        ids = torch.tensor([0, 1], dtype=torch.int32, device=cuda_dev)
        graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s), lora_requests(ids), torch.cuda.graph(graph, stream=s):
            out = model(*args)
        torch.cuda.current_stream().wait_stream(s)
        for want, v in ((both, (0, 1)), (second, (1, 1)), (first, (0, 0))):
            ids.copy_(torch.tensor(v, dtype=torch.int32))
            graph.replay()
            assert torch.equal(out, want)


@gpu
def test_quantised_layers_refuse_gradients_that_they_do_not_have(cuda_dev):
    from nunchaku_rocm_b200.ops.fused import fused_gelu_mlp

    lin, fc2 = layer(128, 256, cuda_dev, 1), layer(256, 128, cuda_dev, 2, unsigned=True)
    down, up = (t.requires_grad_(True) for t in stack_loras([pair(8, 128, 256, 1, cuda_dev), pair(8, 128, 256, 2, cuda_dev)]))
    attach_lora_batch(lin, (down, up))
    x = torch.randn(2, 20, 128, device=cuda_dev).to(BF16)
    ids = torch.tensor([1, 0], dtype=torch.int32, device=cuda_dev)
    with lora_requests(ids):
        y = lin(x)  # the adapters' own gradients are there
        dd, du = torch.autograd.grad(y, (down, up), torch.ones_like(y))
        assert dd.abs().sum() >= 0 and du.any() and torch.isfinite(du).all()
        with pytest.raises(NotImplementedError):
            lin(x.requires_grad_(True))
        with pytest.raises(NotImplementedError):
            fused_gelu_mlp(x.detach(), lin, fc2)


@gpu
def test_qwen_rotary_tables(cuda_dev):
    from nunchaku_rocm_b200.models.qwen_dit import QwenDiT, QwenDiTConfig

    model = QwenDiT(QwenDiTConfig(hidden=256, heads=2, n_blocks=1), device=cuda_dev).random_init(1)
    img, txt = model.rotary_tables(5, 1, 6, 8)
    ids = qwen_image_ids(5, 1, 6, 8, device=cuda_dev)
    want = flux_pos_embed(ids, (16, 56, 56), 10000)
    assert torch.allclose(img, want[5:], rtol=0, atol=2.0**-22) and torch.allclose(txt, want[:5], rtol=0, atol=2.0**-22)
    h, e = torch.randn(1, 48, 64, device=cuda_dev).to(BF16), torch.randn(1, 5, 3584, device=cuda_dev).to(BF16)
    with torch.no_grad():
        out = model(h, e, torch.ones(1, device=cuda_dev), img, txt)
    assert out.shape == (1, 48, 64) and torch.isfinite(out).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, BF16])
def test_operators_in_a_run_together(cuda_dev, dtype):
    """Adaptive norm -> projection with two samples' adapters -> rotation of Q and K -> attention, and all the gradients,
    against the same chain in 64 bits (one 16-bit rounding per operator: a few half steps of the result's norm)."""
    from nunchaku_rocm_b200.ops.elementwise import layer_norm
    from nunchaku_rocm_b200.ops.lora import lora_batched
    from nunchaku_rocm_b200.ops.rotary import rotary_axes

    B, S, H, D = 2, 90, 2, 64
    C = H * D
    g = torch.Generator(device=cuda_dev).manual_seed(7)
    n = lambda *s, k=1.0: (torch.randn(*s, generator=g, device=cuda_dev) * k).to(dtype)  # noqa: E731
    leaves = {"x": n(B, S, C), "scale": n(B, C, k=0.2), "shift": n(B, C, k=0.2), "weight": n(3 * C, C, k=C**-0.5),
              "down": n(2, 16, C, k=C**-0.5), "up": n(2, 3 * C, 16, k=0.25)}
    ids = torch.randint(0, 20, (S, 3), generator=g, device=cuda_dev)
    off, ad = torch.tensor([0, S, 2 * S], dtype=torch.int32, device=cuda_dev), torch.tensor([1, 0], dtype=torch.int32, device=cuda_dev)
    dy = n(B, H, S, D)

    def attention(qkv):
        q, k, v = (t.transpose(1, 2) for t in qkv)
        return torch.softmax(q @ k.transpose(-1, -2) * D**-0.5, -1) @ v

    def ours(p):
        x = layer_norm(p["x"], p["scale"], p["shift"], weight_add=1.0)
        qkv = lora_batched(x, p["down"], p["up"], off, ad, base=x @ p["weight"].t()).view(B, S, 3, H, D)
        q, k = rotary_axes(qkv[:, :, 0], qkv[:, :, 1], ids, (16, 24, 24))
        return attention((q, k, qkv[:, :, 2]))

    def exact(p):
        x = torch.nn.functional.layer_norm(p["x"], (C,), eps=1e-6) * (p["scale"][:, None] + 1) + p["shift"][:, None]
        d = torch.stack([(x[b] @ p["down"][a].t()) @ p["up"][a].t() for b, a in enumerate((1, 0))])
        qkv = (x @ p["weight"].t() + d).view(B, S, 3, H, D)
        ang = torch.cat([ids[:, i, None].double() * 10000.0 ** (-2.0 * torch.arange(w // 2, device=cuda_dev, dtype=torch.float64) / w)
                         for i, w in enumerate((16, 24, 24))], -1)[:, None]
        z = torch.polar(torch.ones_like(ang), ang)
        turn = lambda t: torch.view_as_real(torch.view_as_complex(t.reshape(*t.shape[:-1], -1, 2).contiguous()) * z).flatten(-2)  # noqa: E731
        return attention((turn(qkv[:, :, 0]), turn(qkv[:, :, 1]), qkv[:, :, 2]))

    p16 = {k: v.detach().requires_grad_(True) for k, v in leaves.items()}
    p64 = {k: v.detach().double().requires_grad_(True) for k, v in leaves.items()}
    y, ref = ours(p16), exact(p64)
    got = [y, *torch.autograd.grad(y, list(p16.values()), dy)]
    want = [ref, *torch.autograd.grad(ref, list(p64.values()), dy.double())]
    # forward: norm, projection, sum, rotation, scores, softmax, product = 7 roundings; backward as many again per path
    bound = 14 * torch.finfo(dtype).eps / 2
    for name, a, b in zip(["y", *leaves], got, want):
        err = ((a.double() - b).norm() / b.norm()).item()
        assert err <= bound, (name, err, bound)


@gpu
def test_training_after_serving_in_inference_mode(cuda_dev):
    lin = nn.Linear(64, 48, dtype=BF16, device=cuda_dev).requires_grad_(False)
    down, up = stack_loras([pair(16, 64, 48, 1, cuda_dev), pair(16, 64, 48, 2, cuda_dev)])
    down, up = down.requires_grad_(True), up.requires_grad_(True)
    attach_lora_batch(lin, (down, up))
    x = torch.randn(2, 29, 64, generator=torch.Generator().manual_seed(3)).to(BF16).to(cuda_dev)
    ids = torch.tensor([1, 0], dtype=torch.int32, device=cuda_dev)
    with torch.inference_mode(), lora_requests(ids):
        served = lin(x)
    with lora_requests(ids):
        y = lin(x)
    assert torch.equal(y, served)
    y.float().sum().backward()
    assert down.grad.any() and up.grad.any()
