"""Norms, gates and residual sums between the blocks of a transformer."""

from rl_engine.backends.rocm.norm.block_norm import gated_residual_norm, rms_norm

__all__ = ["gated_residual_norm", "rms_norm"]
