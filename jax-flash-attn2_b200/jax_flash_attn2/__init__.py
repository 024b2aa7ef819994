"""B200-native FlashAttention-2 behind the jax_flash_attn2 API."""
from .flash_attention import (
    AttentionConfig,
    Backend,
    FlashAttention,
    Platform,
    create_flash_attention,
)
from ._flash_attention import flash_attention as triton_flash_attention
from ._kernel_calls import (
    bwd_attention_kernel_call,
    device_status,
    dropout_bits_buffer,
    fwd_attention_kernel_call,
)
from ._paged import PagedStepPlan, paged_attention, paged_cache_write, paged_step_plan
from ._scored_attention import (
    bwd_scored_attention_kernel_call,
    document_layout,
    fwd_scored_attention_kernel_call,
    scored_flash_attention,
)

__all__ = (
    "AttentionConfig",
    "Backend",
    "FlashAttention",
    "Platform",
    "create_flash_attention",
    "triton_flash_attention",
    "fwd_attention_kernel_call",
    "bwd_attention_kernel_call",
    "device_status",
    "dropout_bits_buffer",
    "scored_flash_attention",
    "PagedStepPlan",
    "paged_step_plan",
    "paged_cache_write",
    "paged_attention",
    "document_layout",
    "fwd_scored_attention_kernel_call",
    "bwd_scored_attention_kernel_call",
)
__version__ = "0.1.0"
