"""A policy update as it is run: blocks of norm, FFN on eight-bit copies, gate and residual scale, token scores from the last norm, and
a GRPO loss with an entropy bonus, on a real MI355X.

Against the same steps one by one the gradients are equal to the bit. Against plain autograd in 64 bits they are near, by norms: a
tensor that is stored in bf16 is off by at most 2^-8 of itself (2^-9.8 in the mean square: a third of the square of half a step of up to
2^-8), an eight-bit copy of normal values by a step's 12th root of a 64th of a run's largest, which is 2.1 deviations: 2^-6.7. On the way
of a gradient through two blocks lie 2 * 8 tensors in bf16 forward and 2 * 9 backward and 2 * 2 copies, whose errors are independent:
sqrt(34 * 2^-19.6 + 4 * 2^-13.4) = 0.021 of the norm. Each is carried on with a factor of at most 2 (the second derivative of SwiGLU and the
norm's share in its own direction), and a quotient of two norms over some thousand elements spreads by less than half: 0.021 * 2 * 1.5 =
0.063 for the gradients. Log-probabilities and entropies: logits have deviation 1 and are off by sqrt(16 * 2^-19.6 + 2^-16) = 0.0061 in
the mean square; the largest of 2000 errors is below 5 of them, and the log-sum-exp moves by less than one logit: 0.0061 * 2 * 5 = 0.061."""

from __future__ import annotations

import gc

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32
ROLLOUTS, TOKENS, HIDDEN, INTER, VOCAB, REAL = 6, 37, 256, 384, 1030, 1001
SCALE, EPS, BETA, BONUS = 0.7, 1e-5, 0.04, 0.02


def _normal(*shape, seed, dtype=BF16, scale=1.0, mean=0.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=DEV) * scale + mean).to(dtype)


def _parameters():
    block = lambda i: {
        "gate_weight": _normal(INTER, HIDDEN, seed=10 * i, scale=HIDDEN**-0.5),
        "up_weight": _normal(INTER, HIDDEN, seed=10 * i + 1, scale=HIDDEN**-0.5),
        "down_weight": _normal(HIDDEN, INTER, seed=10 * i + 2, scale=2 * INTER**-0.5),
        "next_norm_weight": _normal(HIDDEN, seed=10 * i + 3, scale=0.1, mean=1.0),
        "post_norm_weight": _normal(HIDDEN, seed=10 * i + 4, scale=0.1, mean=1.0, dtype=FP32),
        "gate": _normal(HIDDEN, seed=10 * i + 5, scale=0.2, mean=0.8),
    }
    names = {"first_norm": _normal(HIDDEN, seed=1, scale=0.1, mean=1.0), "head": _normal(VOCAB, HIDDEN, seed=2, scale=HIDDEN**-0.5)}
    for i in (1, 2):
        names.update({f"{name}_{i}": t for name, t in block(i).items()})
    return {name: t.requires_grad_(True) for name, t in names.items()}


def _batch(wide):
    gen = torch.Generator(device=DEV).manual_seed(99)
    mask = torch.rand(ROLLOUTS, TOKENS, generator=gen, device=DEV) < 0.8
    mask[2] = False  # a rollout without a token that counts
    return {
        "stream": _normal(ROLLOUTS, TOKENS, HIDDEN, seed=5, dtype=wide),
        "ids": torch.randint(0, REAL, (ROLLOUTS, TOKENS), generator=gen, device=DEV),
        "advantages": _normal(ROLLOUTS, seed=6, dtype=FP32),
        "mask": mask,
    }


def _update(p, stream, ids, advantages, mask, old, ref, bits):
    """Scores and the loss through the entry points."""
    from rl_engine.ops.ffn import qwen3_ffn_block
    from rl_engine.ops.logprob import deterministic_linear_scores
    from rl_engine.ops.loss import grpo_ratio_kl_loss
    from rl_engine.ops.norm import rms_norm

    x = rms_norm(stream, p["first_norm"], eps=EPS, dtype=BF16)
    for i in (1, 2):
        stream, x = qwen3_ffn_block(
            stream, x, p[f"gate_weight_{i}"], p[f"up_weight_{i}"], p[f"down_weight_{i}"], p[f"next_norm_weight_{i}"],
            post_norm_weight=p[f"post_norm_weight_{i}"], gate=p[f"gate_{i}"], residual_scale=SCALE, eps=EPS, checkpoint_bits=bits,
        )  # fmt: skip
    scores = deterministic_linear_scores(x, p["head"], ids, top_k=3, real_vocab_size=REAL)
    loss = grpo_ratio_kl_loss(scores.logp, old, ref, advantages, mask, beta=BETA).loss
    bonus = (scores.entropy * mask).sum() / mask.sum()
    return scores, loss - BONUS * bonus


def _plain(p, stream, ids, advantages, mask, old=None, ref=None):
    """The definitions in the type of what it is given; log-probabilities and entropies alone without ``old``."""
    norm = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w  # noqa: E731
    x = norm(stream, p["first_norm"])
    for i in (1, 2):
        y = torch.nn.functional.silu(x @ p[f"gate_weight_{i}"].t()) * (x @ p[f"up_weight_{i}"].t()) @ p[f"down_weight_{i}"].t()
        stream = stream + SCALE * p[f"gate_{i}"] * norm(y, p[f"post_norm_weight_{i}"])
        x = norm(stream, p[f"next_norm_weight_{i}"])
    logits = (x @ p["head"].t())[..., :REAL]
    every = torch.log_softmax(logits, -1)
    logp, entropy = every.gather(-1, ids[..., None])[..., 0], -(every.exp() * every).sum(-1)
    if old is None:
        return logp.detach(), entropy.detach(), every.detach()
    ratio, a = torch.exp(logp - old), advantages[:, None]
    policy = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a)
    k3 = torch.exp(ref - logp) - (ref - logp) - 1
    count = mask.sum()
    return ((policy + BETA * k3 - BONUS * entropy) * mask).sum() / count


def _with_past(batch, p):
    """The log-probabilities of the policy that drew the tokens: ratios of e^+-0.08 and of e^+-0.5, away from where they are clipped."""
    wide = {name: t.double() if t.is_floating_point() else t for name, t in batch.items()}
    logp, entropy, every = _plain({n: t.detach().double() for n, t in p.items()}, **wide)
    steps = torch.tensor([0.08, -0.5, -0.08, 0.5], device=DEV).repeat(ROLLOUTS * TOKENS)[: ROLLOUTS * TOKENS].view(ROLLOUTS, TOKENS)
    past = {"old": (logp + steps).float(), "ref": (logp + 0.3 * steps.roll(1, 1)).float()}
    return past, (logp, entropy, every)


@pytest.mark.parametrize("wide", [BF16, FP32])
@pytest.mark.parametrize("bits", [None, 8])
def test_a_policy_update(wide, bits):
    p, batch = _parameters(), _batch(wide)
    past, (logp, entropy, every) = _with_past(batch, p)
    scores, loss = _update(p, **batch, **past, bits=bits)
    assert float((scores.logp.double() - logp).abs().max()) < 0.061
    assert float((scores.entropy.double() - entropy).abs().max()) < 0.061
    assert float((scores.top_logp.double() - every.topk(3, -1).values).abs().max()) < 0.061
    grads = torch.autograd.grad(loss, list(p.values()))
    p64 = {n: t.detach().double().requires_grad_(True) for n, t in p.items()}
    wide_batch = {n: t.double() if t.is_floating_point() else t for n, t in {**batch, **past}.items()}
    want = torch.autograd.grad(_plain(p64, **wide_batch), list(p64.values()))
    off = {n: float((g.double() - w).norm() / w.norm()) for n, g, w in zip(p, grads, want)}
    assert all(g.dtype == t.dtype for g, t in zip(grads, p.values()))
    assert max(off.values()) < 0.063, off
    # a rollout that is masked out has no share in anything
    other = {**batch, "ids": batch["ids"].clone()}
    other["ids"][2] = 0
    again = torch.autograd.grad(_update(p, **other, **past, bits=bits)[1], list(p.values()))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_the_steps_one_by_one():
    """The gradients of the whole are those of its operators handed on by hand, to the bit."""
    from rl_engine.ops.ffn import qwen3_ffn
    from rl_engine.ops.logprob import deterministic_linear_scores
    from rl_engine.ops.loss import grpo_ratio_kl_loss
    from rl_engine.ops.norm import gated_residual_norm, rms_norm

    p, batch = _parameters(), _batch(BF16)
    past, _ = _with_past(batch, p)
    want = dict(zip(p, torch.autograd.grad(_update(p, **batch, **past, bits=8)[1], list(p.values()))))

    leaf = lambda t: t.detach().requires_grad_(True)  # noqa: E731
    mask, got = batch["mask"], {}
    stream = batch["stream"]
    first = rms_norm(stream, p["first_norm"], eps=EPS, dtype=BF16)
    steps, x = [], leaf(first)
    for i in (1, 2):
        weights = [p[f"{n}_{i}"] for n in ("gate_weight", "up_weight", "down_weight")]
        y = qwen3_ffn(x, *weights, checkpoint_bits=8)
        block, residual = leaf(y), leaf(stream)
        around = [p[f"{n}_{i}"] for n in ("next_norm_weight", "post_norm_weight", "gate")]
        total, normed = gated_residual_norm(block, residual, around[0], post_weight=around[1], gate=around[2], residual_scale=SCALE, eps=EPS)
        steps.append((x, y, weights, block, residual, around, total, normed))
        stream, x = total, leaf(normed)
    scores = deterministic_linear_scores(x, p["head"], batch["ids"], top_k=3, real_vocab_size=REAL)
    logp, entropy = leaf(scores.logp), leaf(scores.entropy)
    loss = grpo_ratio_kl_loss(logp, past["old"], past["ref"], batch["advantages"], mask, beta=BETA).loss - BONUS * ((entropy * mask).sum() / mask.sum())
    g_scores = torch.autograd.grad(loss, [logp, entropy])
    g_x, got["head"] = torch.autograd.grad([scores.logp, scores.entropy], [x, p["head"]], g_scores)
    g_total = None
    for i in (2, 1):
        x, y, weights, block, residual, around, total, normed = steps[i - 1]
        outputs, g = ([total, normed], [g_total, g_x]) if g_total is not None else ([normed], [g_x])
        g_block, g_total, *rest = torch.autograd.grad(outputs, [block, residual, *around], g)
        got.update(zip((f"next_norm_weight_{i}", f"post_norm_weight_{i}", f"gate_{i}"), rest))
        g_x, *rest = torch.autograd.grad(y, [x, *weights], g_block)
        got.update(zip((f"gate_weight_{i}", f"up_weight_{i}", f"down_weight_{i}"), rest))
    got["first_norm"] = torch.autograd.grad(first, [p["first_norm"]], g_x)[0]
    for name in p:
        assert torch.equal(got[name], want[name]), name


def test_a_captured_update_replays():
    p, batch = _parameters(), _batch(BF16)
    past, _ = _with_past(batch, p)

    def step():
        scores, loss = _update(p, **batch, **past, bits=8)
        return [*(t.detach() for t in scores), loss.detach(), *torch.autograd.grad(loss, list(p.values()))]

    step()
    gc.collect()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            batch["stream"].copy_(_normal(ROLLOUTS, TOKENS, HIDDEN, seed=50 + seed))
            p["head"].mul_(1.25)
            p["gate_1"].copy_(_normal(HIDDEN, seed=60 + seed))
        eager = step()
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


def test_a_rollout_scores_its_tokens():
    """Serving: single tokens, with the packed projections and without gradients, give a token the bits that it has in the batch."""
    from rl_engine.ops.ffn import qwen3_ffn_block
    from rl_engine.ops.logprob import deterministic_linear_scores
    from rl_engine.ops.norm import rms_norm

    p, batch = _parameters(), _batch(BF16)
    packed = {i: torch.cat([p[f"gate_weight_{i}"], p[f"up_weight_{i}"]]).detach() for i in (1, 2)}

    def score(stream, ids):
        with torch.no_grad():
            x = rms_norm(stream, p["first_norm"], eps=EPS)
            for i in (1, 2):
                stream, x = qwen3_ffn_block(
                    stream, x, p[f"gate_weight_{i}"], p[f"up_weight_{i}"], p[f"down_weight_{i}"], p[f"next_norm_weight_{i}"],
                    post_norm_weight=p[f"post_norm_weight_{i}"], gate=p[f"gate_{i}"], residual_scale=SCALE, eps=EPS, fused_gate_up_weight=packed[i],
                )  # fmt: skip
            return deterministic_linear_scores(x, p["head"], ids, top_k=5, real_vocab_size=REAL)

    whole = score(batch["stream"], batch["ids"])
    past, _ = _with_past(batch, p)
    trained, _ = _update(p, **batch, **past, bits=8)
    for a, b in ((whole.logp, trained.logp), (whole.entropy, trained.entropy), (whole.top_ids[..., :3], trained.top_ids), (whole.top_logp[..., :3], trained.top_logp)):
        assert torch.equal(a, b)
    for r, t in ((0, 0), (3, 17), (5, 36)):
        for rows in (slice(t, t + 1), slice(max(t - 2, 0), t + 1)):
            one = score(batch["stream"][r, rows], batch["ids"][r, rows])
            for a, b in zip(one, whole):
                assert torch.equal(a[-1], b[r, t])


def test_graphed_callables():
    """A module whose forward and backward are captured one by one, after warm-up on a stream of its own, and replayed by autograd."""
    from rl_engine.ops.ffn import qwen3_ffn_block
    from rl_engine.ops.logprob import deterministic_linear_scores
    from rl_engine.ops.norm import rms_norm

    batch = _batch(BF16)
    ids = batch["ids"].reshape(-1)

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            for name, t in _parameters().items():
                if not name.endswith("_2"):
                    self.register_parameter(name, torch.nn.Parameter(t.detach()))

        def forward(self, stream):
            p = dict(self.named_parameters())
            x = rms_norm(stream, p["first_norm"], eps=EPS)
            _, x = qwen3_ffn_block(
                stream, x, p["gate_weight_1"], p["up_weight_1"], p["down_weight_1"], p["next_norm_weight_1"],
                post_norm_weight=p["post_norm_weight_1"], gate=p["gate_1"], residual_scale=SCALE, eps=EPS, checkpoint_bits=8,
            )  # fmt: skip
            scores = deterministic_linear_scores(x, p["head"], ids, real_vocab_size=REAL)
            return scores.logp, scores.entropy

    eager, net = Net(), Net()
    first = batch["stream"].reshape(-1, HIDDEN).clone().requires_grad_(True)
    graphed = torch.cuda.make_graphed_callables(net, (first,))
    g = _normal(ids.numel(), seed=7, dtype=FP32), _normal(ids.numel(), seed=8, dtype=FP32)
    for seed in range(3):
        stream = _normal(ids.numel(), HIDDEN, seed=70 + seed).requires_grad_(True)
        results = []
        for module in (graphed, eager):
            module.zero_grad()
            out = module(stream)
            torch.autograd.backward(out, [t.clone() for t in g])
            results.append([*(t.detach().clone() for t in out), stream.grad.clone(), *(q.grad.clone() for q in module.parameters())])
            stream.grad = None
            torch.cuda.synchronize()
        for a, b in zip(*results):
            assert torch.equal(a, b)
