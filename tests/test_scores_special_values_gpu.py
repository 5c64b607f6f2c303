"""Token scores of rows that hold what a mask or a diverged model leaves in them, on a real MI355X against the definitions in 64 bits
(tolerances: test_token_scores_gpu.py)."""

from __future__ import annotations

import math
import random
from contextlib import nullcontext

import pytest
import test_operators_random_gpu as draws
import test_token_scores_gpu as plain
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
NEG = plain.NEG
BF16_LOWEST, FP32_LOWEST = torch.finfo(torch.bfloat16).min, torch.finfo(torch.float32).min


@pytest.fixture(scope="module")
def ops():
    from rl_engine.ops import logprob

    return logprob


# ---------------------------------------------------------------------------
# Masks of a finite lowest value: their probability is 0 in 64 bits too, so the definitions are those of a mask of -inf
# ---------------------------------------------------------------------------

MASKS = ["all but one", "all but some", "half", "whole vectors", "whole tiles", "the end"]


def _left(kind, vocab):
    """Which columns a mask leaves."""
    column = torch.arange(vocab, device=DEV)
    return {
        "all but one": column == vocab // 3,
        "all but some": column % 401 == 17,
        "half": torch.rand(vocab, generator=plain._gen(4), device=DEV) < 0.5,
        "whole vectors": (column // 8) % 16 < 5,
        "whole tiles": (column // -(-vocab // 64)) % 3 == 1,
        "the end": column < vocab - vocab // 4,
    }[kind]


@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("dtype,value", [(torch.bfloat16, BF16_LOWEST), (torch.bfloat16, -1e38), (torch.float32, FP32_LOWEST), (torch.float32, -1e38), (torch.float16, -65504.0)])
@pytest.mark.parametrize("rows,vocab,tempered", [(3, 1000, False), (2, 50257, True), (40, 4096, True)])
def test_masks_of_a_finite_lowest_value(ops, kind, dtype, value, rows, vocab, tempered):
    left = _left(kind, vocab)
    z = plain._logits(rows, vocab, vocab, dtype).masked_fill(~left, NEG)
    masked = z.masked_fill(~left, value).requires_grad_(True)
    columns = left.nonzero()[:, 0]
    target = columns[torch.randint(0, columns.numel(), (rows,), generator=plain._gen(5), device=DEV)]
    temp = 0.5 + torch.rand(rows, generator=plain._gen(6), device=DEV) if tempered else None
    g = [torch.randn(rows, generator=plain._gen(20 + i), device=DEV) for i in range(3)]
    for k in (0, min(8, columns.numel())):
        scores = ops.deterministic_scores_from_logits(masked, target, top_k=k, temperature=temp)
        plain._check(scores, z, target, k, temp, vocab)
        g_top = torch.randn((rows, k), generator=plain._gen(30), device=DEV) if k else None
        (grad,) = torch.autograd.grad([scores.logp, scores.lse, scores.entropy] + ([scores.top_logp] if k else []), [masked], g + ([g_top] if k else []))
        want, size = plain._gradient(z, target, temp, scores.top_ids, *g, g_top)
        tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-115
        assert bool(((grad.double() - want).abs() <= plain.HALF_STEP[dtype] * want.abs() + size + tiny).all())


def _linear_case(kind, tokens, vocab, value, by):
    """Hidden states and a head whose masked logits are `value`, by a bias or by a column of the weight, and the logits with -inf in
    their place. A sum of products of some hundreds at most changes nothing in a `value` of 10^38."""
    hidden = 64
    h, w, _ = plain._head(tokens, vocab, hidden, tokens + vocab)
    left = _left(kind, vocab)
    bias = None
    if by == "bias":
        bias = torch.where(left, 0.0, value)
    else:
        h[:, hidden - 1] = 1.0
        w[:, hidden - 1] = torch.where(left, 0.0, value).bfloat16()
    with torch.no_grad():
        z = (h[:, : hidden - 1].double() @ w[:, : hidden - 1].double().t()) if by == "weight" else h.double() @ w.double().t()
    columns = left.nonzero()[:, 0]
    target = columns[torch.randint(0, columns.numel(), (tokens,), generator=plain._gen(5), device=DEV)]
    return h, w, bias, z.masked_fill(~left, NEG), target, columns.numel()


@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("by,value", [("bias", FP32_LOWEST), ("bias", -1e38), ("weight", BF16_LOWEST)])
@pytest.mark.parametrize("tokens,tempered", [(5, False), (300, True), (1100, True), (1281, False)])
def test_masked_scores_of_hidden_states(ops, kind, by, value, tokens, tempered):
    """One token tile, the stream groups, and the entropy in the product's fold."""
    vocab = 5000
    h, w, bias, z, target, left = _linear_case(kind, tokens, vocab, value, by)
    temp = 0.5 + torch.rand(tokens, generator=plain._gen(6), device=DEV) if tempered else None
    h.requires_grad_(True), w.requires_grad_(True)
    g = [torch.randn(tokens, generator=plain._gen(20 + i), device=DEV) for i in range(3)]
    for k in (0, min(3, left)):
        scores = ops.deterministic_linear_scores(h, w, target, bias, top_k=k, temperature=temp)
        plain._check(scores, z, target, k, temp, 16 * vocab)
        dh, dw = torch.autograd.grad([scores.logp, scores.lse, scores.entropy], [h, w], g)
        with torch.no_grad():
            dz, size = plain._gradient(z, target, temp, None, *g, None)
            slack = 2.0**-8 * dz.abs() + 1.01 * size
            for got, want, room in ((dh, dz @ w.double(), slack @ w.double().abs()), (dw, dz.t() @ h.double(), slack.t() @ h.double().abs())):
                assert bool(((got.double() - want).abs() <= 2.0**-8 * want.abs() + 1.01 * room + 2.0**-115).all())


@pytest.mark.parametrize("seed", range(16))
def test_draws_with_masks_of_any_value(ops, seed):
    rng = random.Random(500 + seed)
    rows, vocab, dtype = draws._log_int(rng, 1, 300), draws._log_int(rng, 1, 60000), rng.choice(draws.DTYPES)
    real, gen = rng.randint(max(1, vocab - 100), vocab), plain._gen(seed)
    value = rng.choice([torch.finfo(dtype).min, torch.finfo(dtype).min / 2, -30000.0])
    mask = torch.rand((rows, vocab), generator=gen, device=DEV) < rng.choice([0.1, 0.9, 0.999])
    mask[:, rng.randrange(real)] = False
    if rng.random() < 0.5:
        mask[:, : vocab // 2] = mask[:, :1]
        mask[:, real - 1] = False
    z = plain._logits(rows, vocab, seed, dtype, scale=rng.choice([0.01, 1.0, 4.0])).masked_fill(mask, NEG)
    k = min(int((~mask[:, :real]).sum(1).min()), rng.choice([0, 1, 8, 64]))
    target = (torch.rand((rows, real), generator=gen, device=DEV) * ~mask[:, :real]).argmax(1)
    temp = 0.3 + 2 * torch.rand(rows, generator=gen, device=DEV) if rng.random() < 0.5 else None
    given = z.masked_fill(mask, value)
    given[:, real:] = rng.choice([float("nan"), float("inf"), value])
    given = draws._inside(rng, given).requires_grad_(True)
    s = ops.deterministic_scores_from_logits(given, target, top_k=k, temperature=temp, real_vocab_size=real)
    plain._check(s, z[:, :real], target, k, temp, vocab)
    g = [torch.randn(rows, generator=gen, device=DEV) for _ in range(3)]
    (grad,) = torch.autograd.grad([s.logp, s.lse, s.entropy], [given], g)
    with torch.no_grad():
        want, size = plain._gradient(z[:, :real], target, temp, None, *g, None)
        off = (grad[:, :real].double() - want).abs()
        tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-115
        assert bool((off <= plain.HALF_STEP[dtype] * want.abs() + size + tiny).all()) and not bool(grad[:, real:].any())


# ---------------------------------------------------------------------------
# Rows that have no distribution
# ---------------------------------------------------------------------------


def _nan(t):
    return torch.isnan(t).reshape(t.size(0), -1).all(1)


@pytest.mark.parametrize("tokens", [6, 300, 1100])
@pytest.mark.parametrize("k", [0, 4])
def test_diverged_hidden_states(ops, tokens, k):
    vocab, hidden = 3000, 64
    h, w, target = plain._head(tokens, vocab, hidden, 9)
    w[:, hidden - 1] = 0.0
    w[9, hidden - 1] = 4.0
    h[:, hidden - 1] = 0.0
    clean = ops.deterministic_linear_scores(h, w, target, top_k=k)
    h[1] = float("nan")
    h[2, 5] = float("nan")
    h[3, hidden - 1] = 3e38  # its logit 9 is +inf
    s = ops.deterministic_linear_scores(h, w, target, top_k=k)
    logp, _ = ops.deterministic_linear_logp(h, w, target)
    for t in [s.logp, s.entropy, logp] + ([s.top_logp] if k else []):
        assert _nan(t)[:6].tolist() == [False, True, True, True, False, False]
    assert k == 0 or (s.top_ids[3, 0] == 9 and bool(((s.top_ids >= 0) & (s.top_ids < vocab)).all()))
    for a, b in zip(s, clean):
        assert a is None or (torch.equal(a[0], b[0]) and torch.equal(a[4:], b[4:]))


@pytest.mark.parametrize("tokens", [6, 300, 1100])
@pytest.mark.parametrize("k", [0, 4])
def test_a_bias_that_masks_everything(ops, tokens, k):
    h, w, target = plain._head(tokens, 3000, 64, 9)
    bias = torch.full((3000,), NEG, device=DEV)
    s = ops.deterministic_linear_scores(h, w, target, bias, top_k=k)
    logp, lse = ops.deterministic_linear_logp(h, w, target, bias)
    assert bool((s.lse == NEG).all()) and torch.equal(lse, s.lse)
    for t in (s.logp, s.entropy, s.top_logp, logp):
        assert t is None or bool(torch.isnan(t).all())
    assert k == 0 or s.top_ids[0].tolist() == [0, 1, 2, 3]


def _answers(s):
    return [t for t in (s.logp, s.lse, s.entropy, s.top_logp) if t is not None]


def _rows_with_nan(vocab, dtype, mask):
    """Rows in which a NaN has nothing but NaN and masked logits around it, or before it, and two that have none."""
    nan = float("nan")
    z = plain._logits(9, vocab, 3, dtype)
    z[0, :8] = nan  # a whole vector
    z[1, :8], z[1, 3] = mask, nan
    z[2] = nan
    z[3, : -(-vocab // 64)] = nan  # a whole tile
    z[4], z[4, vocab // 2] = mask, nan
    z[5, vocab - 1] = nan
    z[6, 8:16], z[6, 16:24] = mask, nan
    z[7, : vocab // 2] = mask
    return z


@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("vocab", [100, 5000, 151936])
@pytest.mark.parametrize("k,tempered", [(0, False), (5, True)])
def test_nan_in_any_place_of_a_row(ops, dtype, vocab, k, tempered):
    target = torch.full((9,), vocab - 2, device=DEV)
    temp = torch.full((9,), 0.75, device=DEV) if tempered else None
    for mask in (NEG, torch.finfo(dtype).min):
        z = _rows_with_nan(vocab, dtype, mask)
        s = ops.deterministic_scores_from_logits(z, target, top_k=k, temperature=temp)
        for t in _answers(s):
            assert _nan(t).tolist() == [True] * 7 + [False] * 2
        alone = ops.deterministic_scores_from_logits(z[7:], target[7:], top_k=k, temperature=None if temp is None else temp[7:])
        for a, b in zip(s, alone):
            assert a is None or torch.equal(a[7:], b)
        if k:
            want = torch.sort(z.masked_fill(torch.isnan(z), NEG), dim=1, descending=True, stable=True).indices[:, :k]
            assert torch.equal(s.top_ids, want)


@pytest.mark.parametrize("tokens", [3, 300, 1100])
@pytest.mark.parametrize("by", ["weight", "bias"])
@pytest.mark.parametrize("k", [0, 4])
def test_nan_in_any_place_of_a_head(ops, tokens, by, k):
    """Sixteen columns are what a lane folds at a time, 1024 a split."""
    vocab = 3000
    for first, end, masked in ((0, 16, None), (16, 32, (0, 16)), (1024, 2048, None), (5, 6, (0, 16)), (0, vocab, None)):
        h, w, target = plain._head(tokens, vocab, 64, 9)
        bias = torch.zeros(vocab, device=DEV) if by == "bias" or masked else None
        if masked:
            bias[slice(*masked)] = NEG
        if by == "bias":
            bias[first:end] = float("nan")
        else:
            w[first:end] = float("nan")
        s = ops.deterministic_linear_scores(h, w, target.clamp(min=2500), bias, top_k=k)
        for t in _answers(s):
            assert bool(torch.isnan(t).all()), (first, end, masked)


@pytest.mark.parametrize("tokens", [6, 300, 1100])
def test_lse_of_diverged_hidden_states(ops, tokens):
    h, w, target = plain._head(tokens, 3000, 64, 9)
    h[1], h[2, 5] = float("nan"), float("nan")
    for k in (0, 4):
        assert _nan(ops.deterministic_linear_scores(h, w, target, top_k=k).lse)[:6].tolist() == [False, True, True, False, False, False]


# ---------------------------------------------------------------------------
# Their gradients
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("k", [0, 3])
def test_rows_that_no_gradient_reaches(ops, dtype, k):
    """Zeros, and zeros behind the real columns of every row, temperatures of nothing among them."""
    rows, vocab, real = 6, 9000, 8990
    z = plain._logits(rows, vocab, 3, dtype)
    z[:, real:] = float("nan")
    z[3, 5] = float("nan")
    temp = torch.tensor([1.0, 0.0, -1.0, 1.0, 0.0, 0.7], device=DEV)
    z.requires_grad_(True)
    s = ops.deterministic_scores_from_logits(z, torch.arange(rows, device=DEV), top_k=k, temperature=temp, real_vocab_size=real)
    outputs = [s.logp, s.lse, s.entropy] + ([s.top_logp] if k else [])
    g = [torch.ones_like(o) for o in outputs]
    for t in g:
        t[1:4] = 0.0
    (grad,) = torch.autograd.grad(outputs, [z], g)
    assert not bool(grad[1:4].any()) and not bool(grad[:, real:].any()) and bool(grad[[0, 5]].any(1).all())


@pytest.mark.parametrize("tokens", [7, 300, 1100])
@pytest.mark.parametrize("k", [0, 3])
@pytest.mark.parametrize("kept", [True, False])
def test_tokens_that_a_loss_leaves_out(ops, tokens, k, kept):
    h, w, target = plain._head(tokens, 3001, 64, 9)
    temp = torch.ones(tokens, device=DEV)
    quiet = [2, 5]
    h.requires_grad_(True), w.requires_grad_(True)

    def grads():
        with nullcontext() if kept else ops.recompute_logits():
            s = ops.deterministic_linear_scores(h, w, target, top_k=k, temperature=temp)
            outputs = [s.logp, s.entropy] + ([s.top_logp] if k else [])
            g = [torch.randn(o.shape, generator=plain._gen(20 + i), device=DEV) for i, o in enumerate(outputs)]
            for t in g:
                t[quiet] = 0.0
            return torch.autograd.grad(outputs, [h, w], g)

    clean = grads()
    temp[quiet] = 0.0
    for a, b in zip(grads(), clean):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("asked", ["logp", "lse", "entropy", "top_logp", "all"])
def test_gradients_of_rows_without_a_distribution(ops, dtype, asked):
    """NaN on the real columns where a row is NaN and a gradient reaches it, zeros where a mask has left nothing or where none does."""
    rows, vocab, real, k = 9, 9000, 8999, 3
    z = plain._logits(rows, vocab, 3, dtype)
    z[1, 77] = float("nan")
    z[2, 8500] = float("inf")
    z[3] = NEG
    z[6, 77] = float("nan")
    z[8] = float("nan")
    z[:, real:] = float("nan")
    temp = torch.ones(rows, device=DEV)
    temp[4], temp[7] = 0.0, -1.0
    target = torch.arange(rows, device=DEV) * 900
    g = [torch.randn(rows, generator=plain._gen(20 + i), device=DEV) for i in range(3)] + [torch.randn((rows, k), generator=plain._gen(30), device=DEV)]
    for t in g:
        t[5:8] = 0.0
    z.requires_grad_(True)
    s = ops.deterministic_scores_from_logits(z, target, top_k=k, temperature=temp, real_vocab_size=real)
    outputs = dict(zip(("logp", "lse", "entropy", "top_logp"), zip((s.logp, s.lse, s.entropy, s.top_logp), g)))
    picked = list(outputs.values()) if asked == "all" else [outputs[asked]]
    (grad,) = torch.autograd.grad([o for o, _ in picked], [z], [g for _, g in picked])
    assert _nan(grad[:, :real]).tolist() == [False, True, True, False, True, False, False, False, True]
    assert not bool(grad[:, real:].any()) and not bool(grad[[3, 5, 6, 7]].any())
    with torch.no_grad():
        zero = [t if asked == "all" or name == asked else torch.zeros_like(t) for name, t in zip(outputs, g)]
        want, size = plain._gradient(z[:1, :real], target[:1], None, s.top_ids[:1], *(t[:1] for t in zero))
        tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-115
        assert bool(((grad[:1, :real].double() - want).abs() <= plain.HALF_STEP[dtype] * want.abs() + size + tiny).all())


@pytest.mark.parametrize("tokens", [7, 300, 1100])
@pytest.mark.parametrize("k", [0, 3])
@pytest.mark.parametrize("kept", [True, False])
def test_gradients_of_diverged_hidden_states(ops, tokens, k, kept):
    h, w, target = plain._head(tokens, 3001, 64, 9)
    h.requires_grad_(True), w.requires_grad_(True)

    def grads():
        with nullcontext() if kept else ops.recompute_logits():
            s = ops.deterministic_linear_scores(h, w, target, top_k=k)
            outputs = [s.logp, s.entropy] + ([s.top_logp] if k else [])
            return torch.autograd.grad(outputs, [h, w], [torch.randn(o.shape, generator=plain._gen(20 + i), device=DEV) for i, o in enumerate(outputs)])

    clean, _ = grads()
    with torch.no_grad():
        h[4, 3] = float("nan")
    dh, dw = grads()
    assert _nan(dh)[:7].tolist() == [False] * 4 + [True] + [False] * 2 and bool(torch.isnan(dw).all())
    rest = torch.arange(tokens, device=DEV) != 4
    assert torch.equal(dh[rest], clean[rest])


@pytest.mark.parametrize("tokens", [5, 1100])
def test_gradients_under_a_bias_that_masks_everything(ops, tokens):
    h, w, target = plain._head(tokens, 1000, 64, 9)
    h.requires_grad_(True), w.requires_grad_(True)
    s = ops.deterministic_linear_scores(h, w, target, torch.full((1000,), NEG, device=DEV), top_k=2)
    one = torch.ones(tokens, device=DEV)
    dh, dw = torch.autograd.grad([s.logp, s.entropy, s.top_logp], [h, w], [one, one, torch.ones((tokens, 2), device=DEV)])
    assert not bool(dh.any()) and not bool(dw.any())


# ---------------------------------------------------------------------------
# Masked columns that are asked for
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("vocab,left", [(50, 3), (9000, 20), (9000, 1)])
def test_masked_targets_and_alternatives(ops, dtype, vocab, left):
    """logp and top_logp of a masked column are -inf; its gradient is that of any other column, with p = 0."""
    rows, k = 6, 8 if left < 8 else 40
    z = plain._logits(rows, vocab, 3, dtype)
    keep = torch.rand((rows, vocab), generator=plain._gen(4), device=DEV).topk(left, dim=1).indices
    mask = torch.ones_like(z, dtype=torch.bool).scatter_(1, keep, False)
    z = z.masked_fill(mask, NEG).requires_grad_(True)
    target = keep[:, 0].clone()
    target[:3] = mask[:3].int().argmax(1)
    s = ops.deterministic_scores_from_logits(z, target, top_k=k)
    plain._check(s, z.detach(), target, k, None, vocab)
    assert bool((s.logp[:3] == NEG).all()) and bool((s.top_logp[:, left:] == NEG).all())
    g = [torch.randn(rows, generator=plain._gen(20 + i), device=DEV) for i in range(3)]
    g_top = torch.randn((rows, k), generator=plain._gen(30), device=DEV)
    (grad,) = torch.autograd.grad([s.logp, s.lse, s.entropy, s.top_logp], [z], [*g, g_top])
    with torch.no_grad():
        want, size = plain._gradient(z, target, None, s.top_ids, *g, g_top)
        tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-115
        assert bool(((grad.double() - want).abs() <= plain.HALF_STEP[dtype] * want.abs() + size + tiny).all())


@pytest.mark.parametrize("tokens", [6, 1100])
def test_masked_targets_and_alternatives_of_hidden_states(ops, tokens):
    h, w, target = plain._head(tokens, 3000, 64, 9)
    left = torch.zeros(3000, dtype=torch.bool, device=DEV)
    left[[7, 1500, 2999]] = True
    target[:5] = torch.tensor([7, 8, 1500, 0, 2999], device=DEV)
    bias = torch.where(left, 0.0, NEG)
    h.requires_grad_(True), w.requires_grad_(True)
    s = ops.deterministic_linear_scores(h, w, target, bias, top_k=5)
    with torch.no_grad():
        z = h.double() @ w.double().t() + bias.double()
    plain._check(s, z, target, 5, None, 16 * 3000)
    g, g_top = torch.randn(tokens, generator=plain._gen(20), device=DEV), torch.randn((tokens, 5), generator=plain._gen(30), device=DEV)
    dh, dw = torch.autograd.grad([s.logp, s.top_logp], [h, w], [g, g_top])
    with torch.no_grad():
        zero = torch.zeros_like(g)
        dz, size = plain._gradient(z, target, None, s.top_ids, g, zero, zero, g_top)
        slack = 2.0**-8 * dz.abs() + 1.01 * size
        for got, want, room in ((dh, dz @ w.double(), slack @ w.double().abs()), (dw, dz.t() @ h.double(), slack.t() @ h.double().abs())):
            assert bool(((got.double() - want).abs() <= 2.0**-8 * want.abs() + 1.01 * room + 2.0**-115).all())


# ---------------------------------------------------------------------------
# Logits so far out that lse does not hold the logarithm of the sum: a row that is masked throughout with a finite value, or an offset
# ---------------------------------------------------------------------------


def _far_out(rows, vocab, dtype):
    z = plain._logits(rows, vocab, 3)
    z[0], z[1], z[2] = torch.finfo(dtype).min if dtype != torch.float32 else FP32_LOWEST, -30000.0 if dtype == torch.float16 else -1e9, 60000.0
    if dtype != torch.float16:
        z[3] += 1e6
        z[4] -= 3e6
        z[5, : vocab // 2], z[5, vocab // 2 :] = -1e30, FP32_LOWEST if dtype == torch.float32 else BF16_LOWEST
    return z.to(dtype)


def _shifted(z):
    """The logits from the row's largest on, those without a probability in 64 bits masked."""
    d = z.double() - z.double().amax(1, keepdim=True)
    return d.masked_fill(d < -1500.0, NEG)


@pytest.mark.parametrize("dtype", plain.DTYPES)
@pytest.mark.parametrize("vocab", [70, 5000, 20000])
@pytest.mark.parametrize("tempered", [False, True])
def test_logits_far_out(ops, dtype, vocab, tempered):
    """The steps of the tolerances are those of rows around 0: a temperature of 2 scales without rounding, and the distances from the
    largest logit are what is rounded."""
    rows, k = 8, 5
    z = _far_out(rows, vocab, dtype).requires_grad_(True)
    target = z.argmax(1)
    temp = torch.full((rows,), 2.0, device=DEV) if tempered else None
    s = ops.deterministic_scores_from_logits(z, target, top_k=k, temperature=temp)
    g = [torch.randn(rows, generator=plain._gen(20 + i), device=DEV) for i in range(3)]
    g_top = torch.randn((rows, k), generator=plain._gen(30), device=DEV)
    (grad,) = torch.autograd.grad([s.logp, s.lse, s.entropy, s.top_logp], [z], [*g, g_top])
    with torch.no_grad():
        d = _shifted(z)
        want, bound = plain._reference(d, target, k, temp), plain._bound(d, vocab, temp)
        top = z.double().amax(1) / (2.0 if tempered else 1.0)
        plain._close(s.lse, want["lse"] + top, bound + 2.0**-23 * top.abs())
        # (below 65536, in fp16 and of ordinary rows, log p is a difference with the rounded lse)
        rounded = torch.where(s.lse.abs() < 65536, 2.0**-23 * s.lse.double().abs(), 0.0)
        plain._close(s.logp, want["logp"], bound + rounded)
        plain._close(s.entropy, want["entropy"], 2 * (math.log(vocab) + 1) * bound)
        assert torch.equal(s.top_ids, want["top_ids"])
        plain._close(s.top_logp, want["top_logp"], (bound + rounded)[:, None])
        dz, size = plain._gradient(d, target, temp, s.top_ids, *g, g_top)
        tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-115
        room = size * (1 + rounded[:, None] * 2.0**24 / (vocab / 1024 + 90))
        assert bool(((grad.double() - dz).abs() <= plain.HALF_STEP[dtype] * dz.abs() + room + tiny).all())


@pytest.mark.parametrize("tokens", [5, 300, 1100])
@pytest.mark.parametrize("kept", [True, False])
def test_logits_of_hidden_states_far_out(ops, tokens, kept):
    """A bias of -10^9 on every column leaves nothing of logits around 0: all tokens are the same, and none is certain."""
    vocab, k = 3000, 4
    h, w, target = plain._head(tokens, vocab, 64, 9)
    h.requires_grad_(True), w.requires_grad_(True)
    g, g_entropy, g_top = (torch.randn(shape, generator=plain._gen(20 + i), device=DEV) for i, shape in enumerate([(tokens,), (tokens,), (tokens, k)]))
    with nullcontext() if kept else ops.recompute_logits():
        s = ops.deterministic_linear_scores(h, w, target, torch.full((vocab,), -1e9, device=DEV), top_k=k)
        dh, dw = torch.autograd.grad([s.logp, s.entropy, s.top_logp], [h, w], [g, g_entropy, g_top])
    with torch.no_grad():
        z = torch.zeros((tokens, vocab), dtype=torch.float64, device=DEV)
        want, bound = plain._reference(z, target, k), plain._bound(z, 16 * vocab)
        plain._close(s.logp, want["logp"], bound)
        plain._close(s.entropy, want["entropy"], 2 * (math.log(vocab) + 1) * bound)
        plain._close(s.top_logp, want["top_logp"], bound[:, None])
        assert torch.equal(s.top_ids, want["top_ids"])
        dz, size = plain._gradient(z, target, None, s.top_ids, g, torch.zeros_like(g), g_entropy, g_top)
        slack = 2.0**-8 * dz.abs() + 1.01 * size
        for got, exact, room in ((dh, dz @ w.double(), slack @ w.double().abs()), (dw, dz.t() @ h.double(), slack.t() @ h.double().abs())):
            assert bool(((got.double() - exact).abs() <= 2.0**-8 * exact.abs() + 1.01 * room + 2.0**-115).all())


@pytest.mark.parametrize("dtype", plain.DTYPES)
def test_logits_far_out_that_no_gradient_reaches(ops, dtype):
    z = _far_out(8, 9000, dtype).requires_grad_(True)
    s = ops.deterministic_scores_from_logits(z, z.argmax(1), top_k=2)
    outputs = [s.logp, s.lse, s.entropy, s.top_logp]
    g = [torch.zeros_like(o) for o in outputs]
    for t in g:
        t[6] = 1.0
    (grad,) = torch.autograd.grad(outputs, [z], g)
    assert not bool(grad[:6].any()) and not bool(grad[7].any()) and bool(grad[6].any())


@pytest.mark.parametrize("vocab", [4096, 5000])
@pytest.mark.parametrize("k", [0, 3])
def test_temperatures_without_a_reciprocal(ops, vocab, k):
    """NaN throughout, whatever masked lanes a row's geometry leaves, and zeros or NaN for the gradient by whether one reaches the row."""
    temp = torch.tensor([1.0, math.inf, 1e-40, 2.0**126, 2.0**-126], device=DEV)
    z = plain._logits(5, vocab, 3)
    z[4] *= 2.0**-126
    z.requires_grad_(True)
    s = ops.deterministic_scores_from_logits(z, torch.arange(5, device=DEV), top_k=k, temperature=temp)
    for t in (s.logp, s.lse, s.entropy, s.top_logp):
        assert t is None or _nan(t).tolist() == [False, True, True, False, False]
    (grad,) = torch.autograd.grad(s.logp.sum(), [z])
    assert _nan(grad)[1:4].tolist() == [True, True, False]
    for tokens in (5, 300, 1100):
        h, w, target = plain._head(tokens, vocab, 64, 9)
        temps = torch.ones(tokens, device=DEV)
        temps[1], temps[2] = math.inf, 1e-40
        for t in ops.deterministic_linear_scores(h, w, target, top_k=k, temperature=temps)[:4]:
            assert t is None or _nan(t)[:5].tolist() == [False, True, True, False, False]
