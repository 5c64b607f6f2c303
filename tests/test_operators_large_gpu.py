"""Token scores, norms and eight-bit SwiGLU at both ends of their ranges on a real MI355X: the widest vocabulary, buffers of more than
2^31 elements, whose ends equal the same rows computed alone, and the smallest vocabularies with as many alternatives."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _release_memory():
    yield
    torch.cuda.empty_cache()


def _normal(*shape, seed, dtype=BF16, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_the_widest_vocabulary(dtype):
    """2^28 columns of zeros and three others, by their closed form. A sum of V terms is a chain of V / 1024 in a lane, and 90 steps of
    merges: r = (V / 1024 + 90) 2^-24 relative, with exponentials off by 10 * 2^-24 (|x| up to 8) beside."""
    from rl_engine.ops.logprob import deterministic_scores_from_logits

    vocab = 1 << 28
    z = torch.zeros((2, vocab), dtype=dtype, device=DEV)
    places = {5: 8.0, vocab // 2 + 3: 7.5, vocab - 1: 7.75}
    for column, value in places.items():
        z[0, column] = value
    z.requires_grad_(True)
    target = torch.tensor([vocab - 1, vocab - 2], device=DEV)
    s = deterministic_scores_from_logits(z, target, top_k=5)
    total = (vocab - 3) + sum(math.exp(v) for v in places.values())
    lse = [math.log(total), math.log(vocab)]
    entropy = [lse[0] - sum(v * math.exp(v) for v in places.values()) / total, lse[1]]
    off = (vocab / 1024 + 100) * 2.0**-24
    for row in range(2):
        assert abs(float(s.lse[row]) - lse[row]) <= off + 2.0**-22 * 20
        assert abs(float(s.logp[row]) - ([7.75, 0.0][row] - lse[row])) <= off + 2.0**-22 * 40
        assert abs(float(s.entropy[row]) - entropy[row]) <= 2 * 21 * off
    assert s.top_ids.tolist() == [[5, vocab - 1, vocab // 2 + 3, 0, 1], [0, 1, 2, 3, 4]]
    (grad,) = torch.autograd.grad([s.logp, s.entropy], [z], [torch.tensor([1.0, 1.0], device=DEV), torch.tensor([3.0, 0.0], device=DEV)])
    half_step = torch.finfo(dtype).eps / 2
    for column, value in (*places.items(), (0, 0.0), (vocab - 2, 0.0), (vocab // 4 + 1, 0.0)):
        p = math.exp(value - lse[0])
        parts = [-p, -3 * p * (value - lse[0]), -3 * p * entropy[0], float(column == vocab - 1)]
        size = sum(abs(part) for part in parts)
        # p is off by its lse, the entropy's share by its own error, products by a few steps
        assert abs(float(grad[0, column]) - sum(parts)) <= half_step * abs(sum(parts)) + (off * (1 + 2 * 21) + 20 * 2.0**-22) * size, column
    assert abs(float(grad[1, vocab - 2]) - 1.0) <= half_step + 2.0**-20 and float(grad[1, 7]) < 0


@pytest.mark.parametrize("real", [1, 2, 63, 64])
@pytest.mark.parametrize("vocab", [64, 77, 4096])
def test_as_many_alternatives_as_columns(real, vocab):
    from rl_engine.ops.logprob import deterministic_linear_scores, deterministic_scores_from_logits

    z = _normal(70, vocab, seed=real, dtype=torch.float32)
    z[:, real:] = float("nan")
    target = torch.zeros(70, dtype=torch.long, device=DEV)
    s = deterministic_scores_from_logits(z, target, top_k=real, real_vocab_size=real)
    want = torch.sort(z[:, :real], dim=1, descending=True, stable=True)
    assert torch.equal(s.top_ids, want.indices)
    assert float((s.top_logp.double().exp().sum(1) - 1).abs().max()) <= 2.0**-18  # (all of the distribution)
    h, w = _normal(70, 64, seed=1), _normal(vocab, 64, seed=2)
    s = deterministic_linear_scores(h, w, target, top_k=real, real_vocab_size=real)
    assert torch.equal(s.top_ids.sort(1).values, torch.arange(real, device=DEV).expand(70, real))
    assert bool((s.top_logp[:, 1:] <= s.top_logp[:, :-1]).all())


def test_logits_of_hidden_states_beyond_two_to_the_31():
    """16500 x 131072: the logits in parts, d(logits) as a whole."""
    from rl_engine.ops.logprob import deterministic_linear_scores

    tokens, vocab, hidden = 16500, 131072, 128
    h, w = _normal(tokens, hidden, seed=1).requires_grad_(True), _normal(vocab, hidden, seed=2, scale=0.2)
    target = torch.arange(tokens, device=DEV) * 7 % vocab
    g = _normal(tokens, seed=3, dtype=torch.float32), _normal(tokens, seed=4, dtype=torch.float32)
    s = deterministic_linear_scores(h, w, target)
    (grad,) = torch.autograd.grad([s.logp, s.entropy], [h], g)
    for rows in (slice(0, 70), slice(tokens - 70, tokens)):
        some = h.detach()[rows].requires_grad_(True)
        alone = deterministic_linear_scores(some, w, target[rows])
        for a, b in zip(alone[:3], s[:3]):
            assert torch.equal(a, b[rows])
        (want,) = torch.autograd.grad([alone.logp, alone.entropy], [some], [t[rows] for t in g])
        assert torch.equal(grad[rows], want)


@pytest.mark.parametrize("width", [100, 4096])
def test_rows_of_a_norm_beyond_two_to_the_31(width):
    from rl_engine.ops.norm import gated_residual_norm

    rows = 2**31 // width + 500
    x = torch.zeros((rows, width), dtype=BF16, device=DEV)
    ends = _normal(140, width, seed=1)
    x[:70], x[-70:] = ends[:70], ends[70:]
    x.requires_grad_(True)
    w, gate = _normal(width, seed=2), _normal(width, seed=3)
    g = torch.zeros_like(x)
    g[:70], g[-70:] = ends[70:], ends[:70]
    total, normed = gated_residual_norm(x, x.detach(), w, post_weight=w, gate=gate)
    (grad,) = torch.autograd.grad([total, normed], [x], [g, g])
    some = ends.clone().requires_grad_(True)
    want = gated_residual_norm(some, ends, w, post_weight=w, gate=gate)
    g_some = torch.cat([ends[70:], ends[:70]])
    (want_grad,) = torch.autograd.grad(want, [some], [g_some, g_some])
    for got, alone in ((total, want[0]), (normed, want[1]), (grad, want_grad)):
        assert torch.equal(got[:70], alone[:70]) and torch.equal(got[-70:], alone[70:])


def test_eight_bit_swiglu_beyond_two_to_the_31():
    from rl_engine.ops.ffn import checkpointed_swiglu

    rows, cols = 180000, 12288
    gate = torch.zeros((rows, cols), dtype=BF16, device=DEV)
    ends = _normal(6, cols, seed=1)
    gate[:3], gate[-3:] = ends[:3], ends[3:]
    gate.requires_grad_(True)
    up = gate.detach()
    y = checkpointed_swiglu(gate, up)
    (grad,) = torch.autograd.grad(y, [gate], up)
    some = ends.clone().requires_grad_(True)
    alone = checkpointed_swiglu(some, ends)
    (want,) = torch.autograd.grad(alone, [some], ends)
    for got, w in ((y, alone), (grad, want)):
        assert torch.equal(got[:3], w[:3]) and torch.equal(got[-3:], w[3:])
