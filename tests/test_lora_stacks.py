"""
Stacks of adapters over time: what their owner changes is seen, conversions start from what was attached, and a layer that is
recomputed in a backward pass uses the requests of its forward pass.
"""

import pytest
import torch
from torch import nn

from nunchaku_rocm_b200.lora import attach_lora_batch, batched, detach_lora_batch, lora_requests, stack_loras

gpu = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def factors(A, R, n_in, n_out, dtype, dev="cpu", seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(A, R, n_in, generator=g) * n_in**-0.5).to(dev, dtype), (torch.randn(A, n_out, R, generator=g) * 0.25).to(dev, dtype)


# ------------------------------------------------------------------------------------------------------------ conversions
@pytest.mark.parametrize("change", ["in place", "data", "trained later"])
def test_a_given_stack_is_read_in_every_call(change):
    lin = nn.Linear(32, 24)
    down, up = factors(2, 16, 32, 24, torch.float32)
    attach_lora_batch(lin, (down, up), scale=[1.0, 0.5])
    x = torch.zeros(3, 32, dtype=BF16)
    first = batched._stack_on(lin, x)  # converted: the stack is float32
    assert first[0].dtype == BF16 and torch.equal(first[0], down.to(BF16))
    if change == "in place":
        down.mul_(5)
        up[1].zero_()
    elif change == "data":
        down.data.mul_(5)
        up.data[1].zero_()
    else:
        down.requires_grad_(True)
        up.requires_grad_(True)
    d, u, scale = batched._stack_on(lin, x)
    assert torch.equal(d, down.to(BF16)) and torch.equal(u, up.to(BF16)) and scale.tolist() == [1.0, 0.5]
    if change == "trained later":
        (d.float().sum() + u.float().sum()).backward()
        assert (down.grad == 1).all() and (up.grad == 1).all()
    assert lin._lora_stack[0] is down and lin._lora_stack[1] is up
    # in the input's own dtype it is that very tensor
    assert batched._stack_on(lin, x.float())[0] is down


def test_conversions_start_from_what_was_attached():
    lin = nn.Linear(32, 24)
    g = torch.Generator().manual_seed(1)
    attach_lora_batch(lin, [(torch.randn(16, 32, generator=g), torch.randn(24, 16, generator=g)) for _ in range(2)])
    down, up = lin._lora_stack
    for dtype in (BF16, FP16, torch.float32, torch.float64, FP16):
        d, u, _ = batched._stack_on(lin, torch.zeros(1, 32, dtype=dtype))
        assert torch.equal(d, down.to(dtype)) and torch.equal(u, up.to(dtype))
        assert batched._stack_on(lin, torch.zeros(1, 32, dtype=dtype))[0] is d  # kept while the dtype stays
    leaf = torch.randn(16, 32, requires_grad=True)
    attach_lora_batch(lin, [(leaf, torch.randn(24, 16))])
    with torch.no_grad():
        batched._stack_on(lin, torch.zeros(1, 32, dtype=BF16))  # not kept: the next call may train
    batched._stack_on(lin, torch.zeros(1, 32, dtype=BF16))[0].float().sum().backward()
    assert (leaf.grad == 1).all()
    detach_lora_batch(lin)
    assert not hasattr(lin, "_lora_stack_made")


@gpu
def test_a_replayed_graph_reads_a_given_stack(cuda_dev):
    lin = nn.Linear(64, 48, dtype=BF16, device=cuda_dev).requires_grad_(False)
    down, up = factors(2, 16, 64, 48, torch.float32, cuda_dev)
    attach_lora_batch(lin, (down, up))
    ids = torch.tensor([1, 0], dtype=torch.int32, device=cuda_dev)
    x = torch.randn(2, 9, 64, device=cuda_dev).to(BF16)
    with lora_requests(ids):
        lin(x)
        graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
            out = lin(x)
        torch.cuda.current_stream().wait_stream(s)
        for factor in (3.0, -0.5):
            down.mul_(factor)
            graph.replay()
            want = lin(x)
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    base = lin(x)
    down.zero_()
    with lora_requests(ids):
        assert torch.equal(lin(x), base)


@gpu
def test_a_converted_stack_on_several_streams(cuda_dev):
    x = torch.randn(2, 30, 64, device=cuda_dev).to(FP16)
    ids = torch.tensor([1, 0], dtype=torch.int32, device=cuda_dev)
    g = torch.Generator().manual_seed(2)
    pairs = [(torch.randn(16, 64, generator=g) / 8, torch.randn(48, 16, generator=g) / 8) for _ in range(2)]
    results = []
    for _ in range(4):
        lin = nn.Linear(64, 48, device=cuda_dev).requires_grad_(False)
        attach_lora_batch(lin, pairs)  # float32, from the layer
        lin.half().weight.zero_()
        lin.bias.zero_()
        torch.cuda.synchronize()
        with lora_requests(ids):
            for _ in range(3):
                with torch.cuda.stream(torch.cuda.Stream()):
                    results.append(lin(x))
    torch.cuda.synchronize()
    down, up = stack_loras(pairs, cuda_dev, FP16)
    want = torch.stack([(x[b].double() @ down[a].double().t()) @ up[a].double().t() for b, a in enumerate((1, 0))])
    # fp32 sums of 64 and 16 terms, 2^-22 of h for its parts, one rounding of the result
    terms = torch.stack([(x[b].double().abs() @ down[a].double().abs().t()) @ up[a].double().abs().t() for b, a in enumerate((1, 0))])
    tol = (2.0**-24 * 90 + 2.0**-22) * terms
    tol = tol + torch.finfo(FP16).eps / 2 * (want.abs() + tol) + 2.0**-25
    assert all(torch.equal(r, results[0]) for r in results) and ((results[0].double() - want).abs() <= tol).all()


# ---------------------------------------------------------------------------------------------------------- recomputation
def plain_lora(x, down, up, offsets, adapters, base=None, scale=None, out=None):
    rows, y = x.reshape(-1, x.shape[-1]), []
    for i, a in enumerate(adapters.tolist()):
        r = rows[offsets[i] : offsets[i + 1]]
        y.append((r @ down[a].t()) @ up[a].t() if 0 <= a < len(down) else r @ torch.zeros_like(down[0]).t() @ up[0].t())
    y = torch.cat(y).view(*x.shape[:-1], -1)
    return y if base is None else base + y


def block(dev, dtype, seed=3):
    g = torch.Generator().manual_seed(seed)
    lin = nn.Linear(32, 32, dtype=dtype, device=dev)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(32, 32, generator=g) / 6)
        lin.bias.zero_()
    stack = tuple(t.requires_grad_(True) for t in factors(2, 16, 32, 32, dtype, dev, seed))
    attach_lora_batch(lin.requires_grad_(False), stack)
    return (lambda x: torch.tanh(lin(torch.tanh(x)))), lin, stack


def recomputed(dev, dtype, reentrant, after, wrap):
    """The gradients of x, down and up with and without torch.utils.checkpoint."""
    from torch.utils.checkpoint import checkpoint

    fn, _, stack = block(dev, dtype)
    ids = torch.tensor([1, 0, -1], dtype=torch.int32, device=dev)
    x = torch.randn(3, 5, 32, generator=torch.Generator().manual_seed(4)).to(dev, dtype).requires_grad_(True)
    dy = torch.randn(3, 5, 32, generator=torch.Generator().manual_seed(5)).to(dev, dtype)
    grads = []
    for run in (lambda: fn(x), lambda: checkpoint(wrap(fn), x, use_reentrant=reentrant)):
        for t in (x, *stack):
            t.grad = None
        with lora_requests(ids):
            y = run()
            if not after:
                y.backward(dy)
        if after:
            with lora_requests(ids.flip(0).contiguous()):  # another step's
                y.backward(dy)
        grads.append([t.grad for t in (x, *stack)])
    return grads


@pytest.mark.parametrize("after", [False, True])
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_layers_use_their_requests_or_refuse(monkeypatch, reentrant, after):
    from nunchaku_rocm_b200.lora import keep_lora_requests

    monkeypatch.setattr(batched, "lora_batched", plain_lora)
    want, got = recomputed("cpu", torch.float64, reentrant, after, keep_lora_requests)
    assert all(g is not None and torch.equal(w, g) for w, g in zip(want, got)) and want[1].any()
    with pytest.raises(RuntimeError, match="keep_lora_requests"):
        recomputed("cpu", torch.float64, reentrant, after, lambda fn: fn)


def test_kept_requests(monkeypatch):
    from torch.utils.checkpoint import checkpoint

    from nunchaku_rocm_b200.lora import keep_lora_requests

    monkeypatch.setattr(batched, "lora_batched", plain_lora)
    fn, lin, stack = block("cpu", torch.float64)
    x = torch.randn(2, 4, 32, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([0, 1], dtype=torch.int32)
    # a layer that no requests have used yet may be recomputed as it is, and with none kept afterwards too
    checkpoint(fn, x, use_reentrant=True).sum().backward()
    want = x.grad.clone()
    none = keep_lora_requests(fn)
    with lora_requests(ids):
        kept = keep_lora_requests(fn)
        y = fn(x)
        assert torch.equal(none(x), lin_only(lin, x))
    assert torch.equal(kept(x), y) and torch.equal(fn(x), lin_only(lin, x))
    x.grad = None
    checkpoint(none, x, use_reentrant=True).sum().backward()
    assert torch.equal(x.grad, want)
    with pytest.raises(RuntimeError, match="keep_lora_requests"):
        checkpoint(fn, x, use_reentrant=True).sum().backward()
    ids.flip(0)
    assert torch.equal(kept(x), y)
    ids.copy_(ids.flip(0))
    with pytest.raises(RuntimeError, match="in place"):
        kept(x)
    detach_lora_batch(lin)
    checkpoint(fn, x, use_reentrant=True).sum().backward()  # without a stack there is nothing to know


def lin_only(lin, x):
    return torch.tanh(torch.nn.functional.linear(torch.tanh(x), lin.weight, lin.bias))


@gpu
@pytest.mark.parametrize("after", [False, True])
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_on_the_gpu(cuda_dev, reentrant, after):
    from nunchaku_rocm_b200.lora import keep_lora_requests

    want, got = recomputed(cuda_dev, BF16, reentrant, after, keep_lora_requests)
    assert all(g is not None and torch.equal(w, g) for w, g in zip(want, got)) and want[1].any()
    with pytest.raises(RuntimeError, match="keep_lora_requests"):
        recomputed(cuda_dev, BF16, reentrant, after, lambda fn: fn)


# ------------------------------------------------------------------------------------------------------------- the outputs
@gpu
@pytest.mark.parametrize("precision", ["int4", "nvfp4"])
def test_a_given_output_gets_the_adapters(cuda_dev, precision):
    from nunchaku_rocm_b200.models.linear import SVDQW4A4Linear

    B, S, n_in, n_out = 2, 21, 128, 256
    g = torch.Generator().manual_seed(6)
    lin = SVDQW4A4Linear(n_in, n_out, rank=16, precision=precision)
    with torch.no_grad():
        for name, t in lin.named_parameters():
            t.copy_(torch.randint(-128, 128, t.shape, dtype=torch.int8, generator=g) if t.dtype == torch.int8 else (torch.rand(t.shape, generator=g) * 0.02 + 0.01).to(t.dtype))
    lin.to(cuda_dev)
    stack = factors(2, 16, n_in, n_out, BF16, cuda_dev)
    attach_lora_batch(lin, stack)
    x = torch.randn(B, S, n_in, generator=g).to(BF16).to(cuda_dev)
    with lora_requests(torch.tensor([1, 0], dtype=torch.int32, device=cuda_dev)):
        want = lin(x)
        rows, samples = (torch.zeros(s, dtype=BF16, device=cuda_dev) for s in ((B * S, n_out), (B, S, n_out)))
        for buf in (rows, samples):
            got = lin(x, output=buf)
            assert got.shape == want.shape and torch.equal(got, want) and torch.equal(buf.view_as(want), want)
            assert got.data_ptr() == buf.data_ptr()
        # where a gradient is asked for, the buffer holds the sum as well
        for t in stack:
            t.requires_grad_(True)
        buf = torch.zeros(B * S, n_out, dtype=BF16, device=cuda_dev)
        got = lin(x, output=buf)
        assert torch.equal(buf.detach().view_as(want), want) and torch.equal(got.detach(), want)
        ref = torch.autograd.grad(lin(x), stack, torch.ones_like(want))
        assert all(torch.equal(a, b) and a.any() for a, b in zip(torch.autograd.grad(got, stack, torch.ones_like(want)), ref))
