"""Runtime LoRA on the quantised layers (the per-layer half of the reference's ``nunchaku/lora/runtime.py``), one set for
all samples (:mod:`.runtime`) or one per sample (:mod:`.batched`)."""

from .batched import attach_lora_batch, detach_lora_batch, keep_lora_requests, lora_requests, stack_loras
from .runtime import attach_lora, attached_rank, detach_lora

__all__ = ["attach_lora", "attach_lora_batch", "attached_rank", "detach_lora", "detach_lora_batch", "keep_lora_requests",
           "lora_requests", "stack_loras"]
