"""
Adapters of many requests at once on the layers of a model.

:func:`nunchaku_rocm_b200.lora.attach_lora` makes one LoRA set part of a layer.  Here a layer gets a STACK of adapters
(:func:`attach_lora_batch`), and while :func:`lora_requests` is active every sample of the batch uses its own::

    for layer in (block.to_qkv, block.to_out, block.ff.fc1, block.ff.fc2):
        attach_lora_batch(layer, [(down_a, up_a), (down_b, up_b)])
    with lora_requests(torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")):   # sample 1 has none
        model(...)

Outside of it the layers compute what they did without the stack, and for samples with -1 a layer's own output is that too.
The quantised weight is read once for all samples; the adapters are added to its 16-bit output by
:func:`nunchaku_rocm_b200.ops.lora.lora_batched`, so the fused paths that work on the output before it is rounded (Q/K
normalisation and rotation, GELU and re-quantisation) run as their separate kernels, for ALL samples, on layers that have a
stack while requests are active: what they compute is then rounded to 16 bits once more, for samples with -1 as well.
"""

from __future__ import annotations

import contextlib
import functools
import threading

import torch
from torch import nn

from .. import _lib as L
from ..ops.lora import lora_batched
from .runtime import RANK_GRANULARITY, _is_svdq

__all__ = ["add_lora_batch", "attach_lora_batch", "detach_lora_batch", "has_lora_batch", "keep_lora_requests", "lora_requests",
           "stack_loras"]


class _Active(threading.local):
    adapters = None  # of the innermost lora_requests
    task = -1        # the backward pass that it was entered in, -1: none


_active = _Active()


def _task() -> int:
    """The backward pass that runs on this thread, -1: none."""
    return torch._C._current_graph_task_id()


def stack_loras(adapters, device=None, dtype=None) -> tuple[torch.Tensor, torch.Tensor]:
    """
    ``[(down (r_i, in), up (out, r_i)), ...]`` -> ``down (A, R, in)``, ``up (A, out, R)`` with ``R`` the largest rank rounded up to
    a multiple of 16 and the ranks behind an adapter's own zero; an entry may also be a list of such pairs, added up.
    """
    merged = []
    for entry in adapters:
        pairs = [entry] if isinstance(entry[0], torch.Tensor) else list(entry)
        for down, up in pairs:
            if down.dim() != 2 or up.dim() != 2 or down.shape[0] != up.shape[1]:
                raise ValueError(f"LoRA factors must be (r, in) and (out, r); got {tuple(down.shape)} and {tuple(up.shape)}")
        merged.append((torch.cat([d for d, _ in pairs], 0), torch.cat([u for _, u in pairs], 1)))
    if not merged:
        raise ValueError("no adapters")
    n_in, n_out = merged[0][0].shape[1], merged[0][1].shape[0]
    if any(d.shape[1] != n_in or u.shape[0] != n_out for d, u in merged):
        raise ValueError("the adapters belong to layers of different sizes")
    device, dtype = device or merged[0][0].device, dtype or merged[0][0].dtype
    rank = max(d.shape[0] for d, _ in merged)
    rank = max(RANK_GRANULARITY, -(-rank // RANK_GRANULARITY) * RANK_GRANULARITY)
    down = torch.zeros(len(merged), rank, n_in, device=device, dtype=dtype)
    up = torch.zeros(len(merged), n_out, rank, device=device, dtype=dtype)
    for i, (d, u) in enumerate(merged):
        down[i, : d.shape[0]] = d.to(device, dtype)
        up[i, :, : u.shape[1]] = u.to(device, dtype)
    return down, up


@contextlib.contextmanager
def _entered(adapters):
    before = _active.adapters, _active.task
    _active.adapters, _active.task = adapters, _task()
    try:
        yield
    finally:
        _active.adapters, _active.task = before


def lora_requests(adapters: torch.Tensor):
    """
    While active (in this thread), sample ``b`` of every layer's input uses adapter ``adapters[b]`` of the layer's stack;
    -1 (any value outside the stack): none.  ``adapters (B,)`` int32 on the model's device.  It may be changed in place
    between the replays of a graph that was captured while it was active.

    A function that is recomputed in a backward pass (``torch.utils.checkpoint``) runs on autograd's threads, after or
    beside other requests: give it through :func:`keep_lora_requests`.  Without, its layers refuse to be recomputed.
    """
    if adapters.dtype != torch.int32 or adapters.dim() != 1:
        raise ValueError(f"adapters must be a 1-D int32 tensor, got {tuple(adapters.shape)} {adapters.dtype}")
    return _entered(adapters)


def keep_lora_requests(fn):
    """
    ``fn``, run under the requests that are active now (or none) wherever and whenever it is called::

        with lora_requests(ids):
            y = checkpoint(keep_lora_requests(block), x, use_reentrant=False)
        y.sum().backward()  # recomputes block with the adapters of ids

    The adapters must not be changed in place in between.
    """
    adapters = _requests()
    version = None if adapters is None or adapters.is_inference() else adapters._version

    def run(*args, **kwargs):
        if version is not None and adapters._version != version:
            raise RuntimeError("the adapters of lora_requests were changed in place after keep_lora_requests")
        with _entered(adapters):
            return fn(*args, **kwargs)

    return run


def _requests():
    """The active requests' adapters, or ``None``; in a backward pass only those that were entered in it count."""
    return _active.adapters if _active.task == _task() else None


@functools.lru_cache(maxsize=256)
def _even_offsets(samples: int, rows: int, device: torch.device, stream: int) -> torch.Tensor:
    with torch.inference_mode(False):  # (a training step may save it)
        return torch.arange(0, samples * rows + 1, rows, dtype=torch.int32, device=device)


def _offsets(samples, rows, device):
    if device.type != "cuda":
        return _even_offsets(samples, rows, device, 0)
    if torch.cuda.is_current_stream_capturing():  # (a tensor made here belongs to the graph)
        return _even_offsets.__wrapped__(samples, rows, device, 0)
    # one per stream: another stream would not wait for the kernel that fills it
    return _even_offsets(samples, rows, device, torch.cuda.current_stream(device).cuda_stream)


def has_lora_batch(module: nn.Module) -> bool:
    """Whether ``module`` has a stack of adapters and requests are active that may use it."""
    if getattr(module, "_lora_stack", None) is None:
        return False
    if _active.task != _task() and (_active.adapters is not None or getattr(module, "_lora_stack_used", False)):
        raise RuntimeError("a layer with adapters of several requests is recomputed in a backward pass, which does not know its "
                           "requests: give the recomputed function through keep_lora_requests()")
    return _requests() is not None


def _stack_on(module: nn.Module, x: torch.Tensor):
    """
    The module's stack and scale where ``x`` is and in its dtype (the module may have moved after the attachment).  A stack
    that was given as tensors is converted anew in every call: its owner may change it, by ways that leave no trace (a graph's
    replay, ``.data``), and may train it.  One that was made at the attachment is nobody else's: its conversion takes its place,
    and further ones start from what was attached.
    """
    (down, up), scale = module._lora_stack, module._lora_stack_scale
    if down.device == x.device and down.dtype == x.dtype and (scale is None or scale.device == x.device):
        return down, up, scale
    made = getattr(module, "_lora_stack_made", None)
    if made is not None and made[1] is module._lora_stack:
        (down, up), scale = made[0], made[2]
    with torch.inference_mode(False):
        pair = tuple(t if t.device == x.device and t.dtype == x.dtype else t.to(x.device, x.dtype) for t in (down, up))
        scale = None if scale is None else scale.to(x.device)
    keep = made is not None and made[1] is module._lora_stack and not any(t.requires_grad for t in made[0])
    if keep and not (x.is_cuda and torch.cuda.is_current_stream_capturing()):
        if x.is_cuda:  # later calls may come on other streams, which would not wait for this one
            torch.cuda.current_stream(x.device).synchronize()
        module._lora_stack, module._lora_stack_scale, module._lora_stack_made = pair, scale, (made[0], pair, made[2])
    return *pair, scale


def add_lora_batch(module: nn.Module, x: torch.Tensor, out: torch.Tensor, samples: int | None = None,
                   fused: bool = False) -> torch.Tensor:
    """
    ``out`` plus the active requests' adapters of ``module`` on ``x``; ``x (B, ..., in)`` and ``out (B, ..., out)``, or
    2-D rows of ``samples`` equal samples.  In place unless a gradient is asked for or ``out`` is not laid out for it.
    A quantised layer has gradients of its adapters but none of its input (its weight has no backward pass), and a ``fused``
    path, whose next kernels have no backward pass either, has none at all: both refuse to be asked.
    """
    adapters = _requests()
    if "_lora_stack_used" not in module.__dict__:
        module._lora_stack_used = True
    samples = x.shape[0] if samples is None else samples
    if adapters.shape[0] != samples:
        raise ValueError(f"lora_requests has {adapters.shape[0]} samples, the layer's input {samples}")
    down, up, scale = _stack_on(module, x)
    rows = x.numel() // x.shape[-1]
    if rows == 0:
        return out
    offsets = _offsets(samples, rows // samples, x.device)
    graph = torch.is_grad_enabled() and any(t.requires_grad for t in (x, out, down, up))
    if graph and (fused or (x.requires_grad and _is_svdq(module))):
        raise NotImplementedError("no backward pass: " + ("a fused operator" if fused else "the input of a quantised layer"))
    in_place = not graph and out.is_contiguous() and out.data_ptr() % 16 == 0
    return lora_batched(x, down, up, offsets, adapters, base=out, scale=scale,
                        out=out if in_place else None)


def _hook(module, args, kwargs, output):
    return add_lora_batch(module, args[0] if args else next(iter(kwargs.values())), output) if has_lora_batch(module) else None


def attach_lora_batch(module: nn.Module, adapters, scale=None) -> None:
    """
    Give the layer a stack of adapters: ``adapters`` as in :func:`stack_loras`, or an already stacked ``(down, up)`` pair of
    3-D tensors, which every call reads as they are then (an adapter may be replaced in place, and they may require
    gradients); in the layer's 16-bit dtype and on its device, else every call converts them.  ``scale``: one float per adapter; a
    float32 tensor on the stack's device is read in every call too, anything else at the attachment.  Replaces an earlier
    stack; :func:`detach_lora_batch` removes it.  Ranks up to 128.
    """
    svdq = _is_svdq(module)
    ref = module.proj_down if svdq else next((p for p in module.parameters() if p.is_floating_point()), None)
    if ref is None:
        raise ValueError(f"{type(module).__name__} has no floating-point parameter to take the LoRA dtype from")
    given = len(adapters) == 2 and all(isinstance(t, torch.Tensor) and t.dim() == 3 for t in adapters)
    down, up = adapters if given else stack_loras(adapters, ref.device, ref.dtype)
    if down.dim() != 3 or up.dim() != 3 or down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2] or down.shape[1] % RANK_GRANULARITY:
        raise ValueError(f"stacked factors must be (A, R, in) and (A, out, R), R a multiple of {RANK_GRANULARITY}; got {tuple(down.shape)} and {tuple(up.shape)}")
    if down.shape[1] > L.LORA_MAX_RANK:
        raise NotImplementedError(f"rank {down.shape[1]}: stacks take ranks up to {L.LORA_MAX_RANK}")
    n_in, n_out = getattr(module, "in_features", None), getattr(module, "out_features", None)
    if (n_in, n_out) != (down.shape[2], up.shape[1]):
        raise ValueError(f"LoRA factors {tuple(down.shape)}, {tuple(up.shape)} do not fit a {n_in} -> {n_out} layer")
    if scale is not None:
        scale = torch.as_tensor(scale, dtype=torch.float32).to(down.device)
        if scale.shape != (down.shape[0],):
            raise ValueError(f"scale must have one value for each of {down.shape[0]} adapters, got {tuple(scale.shape)}")
    detach_lora_batch(module)
    module._lora_stack, module._lora_stack_scale = (down, up), scale
    if not given:  # (what was attached, what it was converted to)
        module._lora_stack_made = (module._lora_stack, module._lora_stack, scale)
    if not svdq:  # (SVDQW4A4Linear and the fused operators look for the stack themselves)
        module._lora_stack_hook = module.register_forward_hook(_hook, with_kwargs=True)


def detach_lora_batch(module: nn.Module) -> None:
    """Undo :func:`attach_lora_batch`; a layer without a stack is left alone."""
    if hasattr(module, "_lora_stack_hook"):
        module._lora_stack_hook.remove()
        del module._lora_stack_hook
    for name in ("_lora_stack", "_lora_stack_scale", "_lora_stack_made", "_lora_stack_used"):
        if hasattr(module, name):
            delattr(module, name)
