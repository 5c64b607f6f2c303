"""Forward-mode tangents: token scores, norms and eight-bit copies refuse them, and their gradients those of what comes in, where they
would be lost otherwise."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

BF16 = torch.bfloat16


def _calls(device):
    """(name, call, its floating tensors) of every entry."""
    from rl_engine.ops.ffn import checkpointed_swiglu, qwen3_ffn, qwen3_ffn_block
    from rl_engine.ops.logprob import deterministic_linear_scores, deterministic_scores_from_logits
    from rl_engine.ops.norm import gated_residual_norm, rms_norm

    def t(*shape):
        return torch.randn(shape, device=device).to(BF16)

    ids = torch.zeros(4, dtype=torch.long, device=device)
    x, weights = t(4, 64), (t(128, 64), t(128, 64), t(64, 128))
    return [
        ("scores", lambda z: deterministic_scores_from_logits(z, ids), [t(4, 100)]),
        ("scores with alternatives", lambda z: deterministic_scores_from_logits(z[None], ids[None], top_k=3), [t(4, 100)]),
        ("linear scores", lambda h, w, b: deterministic_linear_scores(h, w, ids, b), [t(4, 64), t(100, 64), torch.randn(100, device=device)]),
        ("norm", lambda b, r, w, p, g: gated_residual_norm(b, r, w, post_weight=p, gate=g), [t(4, 64), t(4, 64), t(64), t(64), t(4, 1)]),
        ("rms_norm", lambda x, w: rms_norm(x, w), [t(4, 64), t(64)]),
        ("swiglu", checkpointed_swiglu, [t(4, 64), t(4, 64)]),
        ("ffn", lambda x, *w: qwen3_ffn(x, *w, checkpoint_bits=8), [x, *weights]),
        ("block", lambda r, x, *w: qwen3_ffn_block(r, x, *w, checkpoint_bits=8), [t(4, 64), x, *weights]),
    ]


NAMES = ["scores", "scores with alternatives", "linear scores", "norm", "rms_norm", "swiglu"]


def _refuses_every_tangent(call, tensors, differentiated):
    tensors = [x.clone().requires_grad_(x.dtype == BF16) if differentiated else x for x in tensors]
    for i, x in enumerate(tensors):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(y, torch.ones_like(y)) if j == i else y for j, y in enumerate(tensors)]
            with pytest.raises(NotImplementedError, match="forward"):
                call(*dual)


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused_in_front_of_everything_else(name):
    (call, tensors), = [(call, tensors) for n, call, tensors in _calls("cpu") if n == name]
    _refuses_every_tangent(call, tensors, False)


@pytest.mark.gpu
@pytest.mark.parametrize("name", [*NAMES, "ffn", "block"])
@pytest.mark.parametrize("differentiated", [False, True])
def test_tangents_are_refused(name, differentiated):
    (call, tensors), = [(call, tensors) for n, call, tensors in _calls("cuda") if n == name]
    _refuses_every_tangent(call, tensors, differentiated)
    with forward_ad.dual_level():  # a level by itself changes nothing
        call(*tensors)


@pytest.mark.gpu
@pytest.mark.parametrize("name", [*NAMES, "ffn", "block"])
@pytest.mark.parametrize("profiled", [False, True])
def test_tangents_of_incoming_gradients_are_refused(name, profiled):
    (call, tensors), = [(call, tensors) for n, call, tensors in _calls("cuda") if n == name]
    tensors = [x.clone().requires_grad_(True) if x.dtype == BF16 else x for x in tensors]
    if profiled:  # the general way of the forward
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]):
            out = call(*tensors)
    else:
        out = call(*tensors)
    out = out if isinstance(out, torch.Tensor) else out[0]
    leaves = [x for x in tensors if x.requires_grad]
    with forward_ad.dual_level():
        g = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward"):
            torch.autograd.grad(out, leaves, g, allow_unused=True)
