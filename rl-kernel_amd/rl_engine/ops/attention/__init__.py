"""What stands between the projections of an attention block: rotary positions, a paged cache of keys and values, attention."""

from rl_engine.backends.rocm.attention.paged import attention_contract_id, paged_append, paged_attention, qwen3_attention_block
from rl_engine.backends.rocm.attention.rotary import rotary_embedding, rotary_frequencies

__all__ = [
    "attention_contract_id",
    "paged_append",
    "paged_attention",
    "qwen3_attention_block",
    "rotary_embedding",
    "rotary_frequencies",
]
