"""Seeded draws over the ranges of token scores, norms and eight-bit copies on a real MI355X: sizes, types, strides, masks and what is
asked for, each against its definition in 64 bits with the tolerances of its own file."""

from __future__ import annotations

import math
import random

import pytest
import test_block_norm_gpu as norms
import test_mx8_gpu as copies
import test_token_scores_gpu as scores
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _inside(rng, t, fill=float("nan")):
    """The same values as a part of wider rows that start anywhere, `fill` around them."""
    rows, cols = t.shape
    before, behind = rng.choice([0, 0, 1, 3, 8]), rng.choice([0, 0, 1, 5, 64])
    wide = torch.full((rows, cols + before + behind), fill, dtype=t.dtype, device=DEV)
    wide[:, before : before + cols] = t
    return wide[:, before : before + cols]


@pytest.mark.parametrize("seed", range(24))
def test_scores_of_logits(seed):
    from rl_engine.ops.logprob import deterministic_scores_from_logits

    rng = random.Random(seed)
    rows, vocab, dtype = _log_int(rng, 1, 400), _log_int(rng, 1, 60000), rng.choice(DTYPES)
    real = vocab if rng.random() < 0.5 else rng.randint(max(1, vocab - 300), vocab)
    k = min(real, 64, rng.choice([0, 1, 2, 5, 20, 40, 64]))
    gen = scores._gen(seed)
    z = scores._logits(rows, vocab, seed, dtype, scale=rng.choice([0.01, 1.0, 4.0]))
    if rng.random() < 0.4:
        z[torch.rand(z.shape, generator=gen, device=DEV) < rng.choice([0.1, 0.9, 0.999])] = scores.NEG
        z[:, rng.randrange(real)] = 0.5
    if rng.random() < 0.3:
        z[:, : vocab // 2] = z[:, :1]
    # the likeliest column, or any that is not masked (rows of which nothing is left take their first)
    target = (z[:, :real].float() if rng.random() < 0.5 else torch.rand((rows, real), generator=gen, device=DEV) * (z[:, :real] > scores.NEG)).argmax(1)
    temp = 0.3 + 2 * torch.rand(rows, generator=gen, device=DEV) if rng.random() < 0.5 else None
    z[:, real:] = float("nan")
    z = _inside(rng, z).requires_grad_(True)
    s = deterministic_scores_from_logits(z, target, top_k=k, temperature=temp, real_vocab_size=real)
    g = [torch.randn(rows, generator=gen, device=DEV) for _ in range(3)]
    g_top = torch.randn((rows, k), generator=gen, device=DEV) if k else None
    (grad,) = torch.autograd.grad([s.logp, s.lse, s.entropy] + ([s.top_logp] if k else []), [z], g + ([g_top] if k else []))
    with torch.no_grad():
        scores._check(s, z[:, :real], target, k, temp, vocab)
        finite = torch.isfinite(s.lse)
        if k:
            finite &= torch.isfinite(s.top_logp).all(1)
        want, size = scores._gradient(z[:, :real], target, temp, s.top_ids, *g, g_top)
        off = (grad[:, :real].double() - want).abs()
        # the exponential's results below 2^-126 are 0; what they are multiplied with is at most 3.4 (1 / temperature) times the sum of
        # up to 67 gradients of deviation 1 and of one more times |log p| + entropy, 100: below 2^11
        tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-115
        assert bool((off <= scores.HALF_STEP[dtype] * want.abs() + size + tiny)[finite].all()) and not bool(grad[:, real:].any())


@pytest.mark.parametrize("seed", range(16))
def test_scores_of_hidden_states(seed):
    from rl_engine.ops.logprob import deterministic_linear_logp, deterministic_linear_scores, recompute_logits

    rng = random.Random(100 + seed)
    tokens, vocab, hidden = _log_int(rng, 1, 1500), _log_int(rng, 1, 40000), rng.choice([8, 24, 64, 100, 128, 256, 512])
    real = rng.randint(max(1, vocab - 200), vocab)
    k = min(real, 64, rng.choice([0, 0, 1, 7, 64]))
    h, w, target = scores._head(tokens, vocab, hidden, 7 * seed)
    target.clamp_(max=real - 1)
    temp = 0.3 + 2 * torch.rand(tokens, generator=scores._gen(seed), device=DEV) if rng.random() < 0.5 else None
    s = deterministic_linear_scores(h, w, target, top_k=k, temperature=temp, real_vocab_size=real)
    scores._check(s, (h.double() @ w.double().t())[:, :real], target, k, temp, 16 * vocab)
    logp, lse = deterministic_linear_logp(h, w, target, temperature=temp, real_vocab_size=real)
    assert torch.equal(s.logp.view(torch.int32), logp.view(torch.int32)) and torch.equal(s.lse.view(torch.int32), lse.view(torch.int32))
    some = slice(rng.randrange(tokens), None)
    alone = deterministic_linear_scores(h[some], w, target[some], top_k=k, temperature=None if temp is None else temp[some], real_vocab_size=real)
    for a, b in zip(alone, s):
        assert a is None or torch.equal(a, b[some])
    h.requires_grad_(True), w.requires_grad_(True)

    def grads():
        t = deterministic_linear_scores(h, w, target, top_k=k, temperature=temp, real_vocab_size=real)
        return [*(o for o in t if o is not None), *torch.autograd.grad(t.logp.sum() + t.entropy.sum(), [h, w])]

    kept = grads()
    with recompute_logits():
        again = grads()
    for a, b in zip(kept, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("seed", range(40))
def test_norms(seed):
    from rl_engine.ops import norm

    rng = random.Random(200 + seed)
    tokens, width = _log_int(rng, 1, 3000), _log_int(rng, 1, 16384)
    tokens = min(tokens, max(1, 4_000_000 // width))
    dtype = rng.choice(DTYPES)
    wide = rng.choice([dtype, torch.float32])
    kind, post, pre, weights = rng.choice(["none", "channel", "token", "full"]), rng.random() < 0.6, rng.random() < 0.8, rng.choice([dtype, torch.float32])
    t, g_total, g_normed = norms._case(tokens, width, dtype, wide, kind, post, pre, seed=seed, weights=weights)
    if not pre or rng.random() < 0.5:
        g_total = g_total if g_total is not None else norms._normal(tokens, width, seed=5, dtype=wide)
    want = norms._definition(*(t[k] for k in ("block", "residual", "gate", "post", "pre")), g_total, g_normed)
    t = {k: _inside(rng, v) if v is not None and v.dim() == 2 and v.size(1) == width and width > 1 else v for k, v in t.items()}
    norms._compare(norms._run(norm, t, g_total, g_normed), want, t, tokens)


@pytest.mark.parametrize("seed", range(24))
def test_copies(seed):
    from rl_engine import _C
    from rl_engine.ops.ffn import checkpointed_swiglu

    rng = random.Random(300 + seed)
    rows, cols, dtype = _log_int(rng, 1, 2000), _log_int(rng, 1, 3000), rng.choice(DTYPES)
    gate = _inside(rng, copies._normal(rows, cols, seed=seed, dtype=dtype, scale=rng.choice([1e-3, 1.0, 50.0])))
    up = _inside(rng, copies._normal(rows, cols, seed=seed + 1, dtype=dtype))
    codes, scale_bytes = _C.mx8_encode(gate)
    want_codes, want_bytes, values = copies._definition(gate)
    assert torch.equal(codes, want_codes) and torch.equal(scale_bytes, want_bytes)
    assert torch.equal(_C.mx8_decode(codes, scale_bytes, torch.float32).double(), values)
    dy = _inside(rng, copies._normal(rows, cols, seed=seed + 2, dtype=dtype))
    kept = [_C.mx8_decode(*_C.mx8_encode(t), torch.float32 if dtype == torch.float16 else dtype) for t in (gate, up)]
    f = kept[0].dtype
    want = _C.swiglu_backward(dy.to(f).contiguous(), *kept)
    gate.requires_grad_(True), up.requires_grad_(True)
    y = checkpointed_swiglu(gate, up)
    grads = torch.autograd.grad(y, [gate, up], dy)
    assert torch.equal(y, _C.swiglu_forward(gate.detach().to(f).contiguous(), up.detach().to(f).contiguous()).to(dtype))
    for g, w in zip(grads, want):
        assert torch.equal(copies._bits(g), copies._bits(w.to(dtype)))
