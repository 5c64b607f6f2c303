"""Gated FFN operators (gfx950 build: ROCm only)."""

from rl_engine._C import mx8_decode, mx8_encode
from rl_engine.backends.rocm.ffn.ffn import (
    BACKEND_ID,
    Qwen3FFNOp,
    checkpointed_swiglu,
    qwen3_ffn,
    qwen3_ffn_block,
    qwen3_ffn_packed_inference,
)

__all__ = [
    "BACKEND_ID",
    "Qwen3FFNOp",
    "checkpointed_swiglu",
    "mx8_decode",
    "mx8_encode",
    "qwen3_ffn",
    "qwen3_ffn_block",
    "qwen3_ffn_packed_inference",
]
