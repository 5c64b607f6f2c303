"""The native host side of the smallest calls (csrc/torch_host.cpp), bound to the loaded library on first use."""

from __future__ import annotations

import ctypes

import torch

from rl_engine import _lib

_ENTRIES = (
    "rlk_last_error", "rlk_det_gemm_bf16", "rlk_linear_bwd_bf16", "rlk_det_gemm_swiglu_workspace_bytes", "rlk_det_gemm_swiglu_bf16",
    "rlk_det_gemm_swiglu_training_bf16", "rlk_swiglu_bwd", "rlk_grpo_workspace_bytes", "rlk_grpo_ratio_kl_loss", "rlk_grpo_ratio_kl_loss_bwd",
    "rlk_logits_scores_workspace_bytes", "rlk_logits_scores", "rlk_logits_scores_backward", "rlk_block_norm_forward",
    "rlk_block_norm_workspace_bytes", "rlk_block_norm_backward", "rlk_linear_scores_workspace_bytes", "rlk_linear_scores_fwd",
    "rlk_linear_dlogits_row_stride", "rlk_linear_dlogits_bwd", "rlk_mx8_encode", "rlk_mx8_swiglu_forward", "rlk_mx8_swiglu_backward",
    "rlk_rotary_embedding", "rlk_paged_append", "rlk_paged_attention_workspace_bytes", "rlk_paged_attention",
)  # fmt: skip
_native = None


def native():
    """The module, whose functions answer ``None`` to arguments that are not everyday ones."""
    global _native
    if _native is None:
        lib = _lib.load()
        try:
            from rl_engine import _torch_host
        except ImportError as missing:
            raise _lib.RlkLibraryMissing(
                f"rl_engine/_torch_host.so could not be loaded ({missing}): build it with `python rl-kernel_amd/build.py`"
            ) from missing
        from rl_engine.backends.rocm.attention.rotary import rotary_gradients
        from rl_engine.backends.rocm.ffn.ffn import ffn_gradients, kept_swiglu_gradients
        from rl_engine.backends.rocm.gemm.det_gemm import linear_gradients
        from rl_engine.backends.rocm.logprob.token_scores import linear_scores_gradients, scores_gradient
        from rl_engine.backends.rocm.loss.grpo import _elementwise_gradient
        from rl_engine.backends.rocm.norm.block_norm import norm_gradients

        addresses = {name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _ENTRIES}
        _torch_host.bind(
            addresses, linear_gradients, ffn_gradients, _elementwise_gradient, scores_gradient, norm_gradients, kept_swiglu_gradients,
            linear_scores_gradients, rotary_gradients,
        )  # fmt: skip
        _native = _torch_host
    return _native


def recorded(*tensors) -> bool:
    """Whether something records or takes over the operations on ``tensors`` (``None`` among them is passed over): a compiler, a tracer, a
    mode, a profiler, a subclass. A launch on their addresses would escape it: the caller goes through a registered operator."""
    return torch.compiler.is_compiling() or not native().plain(*tensors)


def refuse_capture_into_another_graph() -> None:
    """For a backward in front of its first launch. A leaf keeps the node that gathers its gradient as long as any graph holds the leaf,
    and the engine orders that node's stream behind the gradient. Under graph capture a stream joins the capture by that, which the
    default stream cannot: the process would end over it."""
    from rl_engine import _torch_host

    if torch.cuda.is_current_stream_capturing() and _torch_host.reaches_default_stream():
        raise RuntimeError(
            "a backward cannot be captured into a graph while an autograd graph that was made on the default stream holds its inputs: "
            "drop the outputs of the earlier calls first"
        )
