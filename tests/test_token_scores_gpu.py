"""Token scores (log-probability, log-sum-exp, entropy, alternatives) on a real MI355X against their definitions in 64 bits.

Tolerances. A row's sums are chains of about V / 1024 additions in a lane and 80 in the merges, each off by half a step of
2^-24 relative; an exponential e(x) = exp2(x log2 e) is off by |x| 2^-24 (the product's rounding) and 2^-23 (the instruction),
and weighted with itself |x| e(x) <= 1/e; a temperature rounds twice, 2^-23 of the logit. So S is off by
r = (V / 1024 + 90) 2^-24 relative, lse and logp by r + 2^-22 (largest scaled logit and lse), the entropy, whose terms are
weighted with up to |log p|, by 2 (log V + 1) times that. Ids are exact."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
NEG = float("-inf")
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    from rl_engine.ops import logprob

    return logprob


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(rows, vocab, seed, dtype=torch.float32, scale=3.0):
    return (torch.randn((rows, vocab), generator=_gen(seed), device=DEV) * scale).to(dtype)


def _reference(z, target, k=0, temp=None):
    """The definitions in 64 bits, z [rows, real]."""
    z = z.double()
    y = z if temp is None else z / temp.double()[:, None]
    lse = torch.logsumexp(y, 1)
    logq = y - lse[:, None]
    p = logq.exp()
    out = {"lse": lse, "logp": logq.gather(1, target[:, None])[:, 0], "entropy": -torch.special.xlogy(p, p).sum(1)}
    if k:
        out["top_ids"] = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
        out["top_logp"] = logq.gather(1, out["top_ids"])
    return out


def _bound(z, vocab, temp=None):
    y = z.double().masked_fill(torch.isinf(z), 0.0).abs().amax(1)
    y = y if temp is None else y / temp.double()
    return (vocab / 1024 + 90) * 2.0**-24 + 2.0**-22 * (2 * y + math.log(vocab) + 1)


def _close(got, want, bound):
    got = got.double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    near = (got - want).abs() <= bound + 2.0**-23 * want.abs()
    assert bool((same | near).all()), float((got - want).abs().nan_to_num(0.0, 0.0, 0.0).max())


def _check(scores, z, target, k, temp, vocab):
    want = _reference(z, target, k, temp)
    bound = _bound(z, vocab, temp)
    _close(scores.lse, want["lse"], bound)
    _close(scores.logp, want["logp"], bound)
    _close(scores.entropy, want["entropy"], 2 * (math.log(vocab) + 1) * bound)
    if k:
        assert scores.top_ids.dtype == torch.int64 and torch.equal(scores.top_ids, want["top_ids"])
        _close(scores.top_logp, want["top_logp"], bound[:, None])
    else:
        assert scores.top_ids is None and scores.top_logp is None


SHAPES = [
    (1, 1, 1, 1, False), (3, 7, 5, 5, True), (5, 64, 64, 64, False), (2, 300, 257, 33, True), (3, 513, 513, 0, True), (37, 4096, 4000, 8, False),
    (9, 50257, 50257, 20, True), (70, 32768, 32768, 1, True), (4, 151936, 151669, 64, False), (3, 151936, 2375, 64, True),
]  # fmt: skip


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,real,k,tempered", SHAPES)
def test_scores_match_the_definitions(ops, rows, vocab, real, k, tempered, dtype):
    z = _logits(rows, vocab, rows + vocab, dtype)
    z[:, real:] = float("nan")
    if vocab > 100:
        z[:, 1:real:3] = NEG  # tokens that cannot be drawn
    target = torch.randint(0, max(real // 3, 1), (rows,), generator=_gen(5), device=DEV) * 3
    temp = 0.5 + torch.rand(rows, generator=_gen(6), device=DEV) if tempered else None
    scores = ops.deterministic_scores_from_logits(z, target, top_k=k, temperature=temp, real_vocab_size=real)
    _check(scores, z[:, :real], target, k, temp, vocab)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,real", [(4096, 4096), (151936, 151669), (64, 60)])
def test_logp_and_lse_are_the_bits_of_the_logits_entry(ops, dtype, vocab, real):
    rows = 33
    z = _logits(rows, vocab, 77, dtype)
    z[3, : real // 2] = NEG
    target = torch.randint(0, real, (rows,), generator=_gen(1), device=DEV)
    for temp in (None, 0.5 + torch.rand(rows, generator=_gen(2), device=DEV)):
        logp, lse = ops.deterministic_logp_from_logits(z, target, real_vocab_size=real, temperature=temp)
        for k in (0, 7):
            scores = ops.deterministic_scores_from_logits(z, target, real_vocab_size=real, temperature=temp, top_k=k)
            assert torch.equal(scores.logp.view(torch.int32), logp.view(torch.int32))
            assert torch.equal(scores.lse.view(torch.int32), lse.view(torch.int32))


def _spread(kind, vocab):
    """Rows whose largest logits lie where they are hardest to pick out."""
    column = torch.arange(vocab, device=DEV, dtype=torch.float32)
    if kind == "constant":
        return torch.full((vocab,), 1.5, device=DEV)
    if kind == "ascending":
        return column / vocab
    if kind == "descending":
        return -column / vocab
    if kind == "two values":
        return (column % 5 == 3).float()
    if kind == "signed zeros":
        return torch.where(column % 2 == 0, -0.0, 0.0)
    if kind == "one tile":  # the largest thousands lie side by side
        return torch.where((column >= 5000) & (column < 7000), 2.0 + column / vocab, -column / vocab)
    if kind == "every sixteenth vector":  # in one slice of each tile
        return torch.where((column // 8) % 16 == 7, 3.0 + (column * 37 % vocab) / vocab, 0.0)
    if kind == "all but a few masked":
        return torch.where(column % 4001 == 17, column / vocab, NEG)
    if kind == "one":
        return torch.where(column == vocab - 1, -40.0, NEG)
    raise AssertionError(kind)


KINDS = ["constant", "ascending", "descending", "two values", "signed zeros", "one tile", "every sixteenth vector", "all but a few masked", "one"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", [1000, 50257, 151936])
def test_alternatives_wherever_they_lie(ops, kind, vocab):
    z = _spread(kind, vocab)[None].repeat(3, 1)
    z[1] = z[1].flip(0)
    z[2] = z[2].roll(12345)
    target = torch.full((3,), vocab - 1, device=DEV)
    for k in (1, 20, 64):
        for dtype in (torch.float32, torch.bfloat16):
            got = ops.deterministic_scores_from_logits(z.to(dtype), target, top_k=k)
            want = torch.sort(z.to(dtype), dim=1, descending=True, stable=True).indices[:, :k]
            assert torch.equal(got.top_ids, want), (kind, vocab, k, dtype)


def test_rows_without_a_distribution(ops):
    z = _logits(6, 5000, 3)
    z[0] = NEG
    z[1, 77] = float("inf")
    z[2, 99] = float("nan")
    target = torch.tensor([4, 4, 4, -1, 5000, 4], device=DEV)
    temp = torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 0.0], device=DEV)
    scores = ops.deterministic_scores_from_logits(z, target, top_k=5, temperature=temp)
    nan = torch.isnan
    assert scores.lse[0] == NEG and bool(nan(scores.lse[[1, 2, 5]]).all()) and not bool(nan(scores.lse[[3, 4]]).any())
    assert bool(nan(scores.logp).all())
    assert nan(scores.entropy).tolist() == [True, True, True, False, False, True]
    assert scores.top_ids[0].tolist() == [0, 1, 2, 3, 4]
    assert scores.top_ids[1, 0] == 77 and 99 not in scores.top_ids[2].tolist()
    want = torch.sort(z[3:5], dim=1, descending=True, stable=True).indices[:, :5]
    assert torch.equal(scores.top_ids[3:5], want)
    assert bool(((scores.top_ids >= 0) & (scores.top_ids < 5000)).all())


@pytest.mark.parametrize("layout", ["padded rows", "odd start", "columns apart", "batch of two axes", "one row repeated", "transposed batch"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts(ops, layout, dtype):
    rows, vocab, k = 6, 3001, 9
    plain = _logits(rows, vocab, 4, dtype)
    target = torch.randint(0, vocab, (rows,), generator=_gen(8), device=DEV)
    z, ids = plain, target
    if layout == "padded rows":
        z = torch.full((rows, vocab + 13), float("nan"), dtype=dtype, device=DEV)[:, :vocab].copy_(plain)
    elif layout == "odd start":
        z = torch.empty(rows * vocab + 3, dtype=dtype, device=DEV)[3:].view(rows, vocab).copy_(plain)
    elif layout == "columns apart":
        z = torch.empty((rows, vocab, 2), dtype=dtype, device=DEV)[:, :, 1].copy_(plain)
    elif layout == "batch of two axes":
        z, ids = plain.view(2, 3, vocab), target.view(2, 3)
    elif layout == "one row repeated":
        z = plain[:1].expand(rows, vocab)
        plain = z.contiguous()
    else:
        z, ids = plain.view(2, 3, vocab).transpose(0, 1), target.view(2, 3).t()
        plain, target = z.reshape(rows, vocab), ids.reshape(rows)
    got = ops.deterministic_scores_from_logits(z, ids, top_k=k)
    assert got.logp.shape == ids.shape and got.top_ids.shape == (*ids.shape, k)
    want = ops.deterministic_scores_from_logits(plain, target, top_k=k)
    for g, w in zip(got, want):
        assert torch.equal(g.reshape(w.shape), w)
    _check(want, plain, target, k, None, vocab)


def test_a_row_does_not_depend_on_its_batch(ops):
    z = _logits(2100, 1536, 9, torch.bfloat16)
    target = torch.randint(0, 1536, (2100,), generator=_gen(9), device=DEV)
    whole = ops.deterministic_scores_from_logits(z, target, top_k=6)
    for rows in ([0], [2099], list(range(700, 765))):
        some = ops.deterministic_scores_from_logits(z[rows], target[rows], top_k=6)
        for s, w in zip(some, whole):
            assert torch.equal(s, w[rows])


# ---------------------------------------------------------------------------
# Gradients
# ---------------------------------------------------------------------------


def _gradient(z, target, temp, ids, g_logp, g_lse, g_entropy, g_top):
    """The definition's gradient in 64 bits and, per element, by how much it may be off before the last rounding: the sizes of
    its factors times p's relative error. With y the scaled logit and d = y - lse, in units of 2^-24: 2 |y| for the reciprocal
    temperature and the product with it, |lse| for the rounding of lse beside the V / 1024 + 90 of its sum, |d| for the
    difference, |d| for its product with log2 e, and 8 for the exponential and the products behind it. The gradients that are summed
    to p's factor may cancel: the sum of g_top takes 6 steps over a wave and 2 more with the others, 8 of the sizes of what is summed."""
    z = z.double()
    rows = torch.arange(z.size(0), device=DEV)
    inv = torch.ones(z.size(0), dtype=torch.float64, device=DEV) if temp is None else 1 / temp.double()
    y = z * inv[:, None]
    logq = y - torch.logsumexp(y, 1)[:, None]
    p = logq.exp()
    entropy = -torch.special.xlogy(p, p).sum(1)
    slope = g_lse.double() - g_logp.double() - (g_top.double().sum(1) if g_top is not None else 0.0)
    dz = p * slope[:, None] - g_entropy.double()[:, None] * (torch.special.xlogy(p, p) + p * entropy[:, None])
    size = p * (slope.abs()[:, None] + g_entropy.double().abs()[:, None] * (torch.where(p > 0, -logq, 0.0) + entropy[:, None] + 1))
    dz[rows, target] += g_logp.double()
    size[rows, target] += g_logp.double().abs()
    if g_top is not None:
        dz.scatter_add_(1, ids, g_top.double())
        size.scatter_add_(1, ids, g_top.double().abs())
    d = torch.where(p > 0, y - torch.logsumexp(y, 1)[:, None], 0.0).abs()
    y = torch.where(p > 0, y, 0.0).abs()
    steps = 2 * y + torch.logsumexp(y, 1)[:, None].abs() + 2 * d + 8 + z.size(1) / 1024 + 90
    summed = g_lse.double().abs() + g_logp.double().abs() + (g_top.double().abs().sum(1) if g_top is not None else 0.0)
    return dz * inv[:, None], 2.0**-24 * (steps * size + 8 * p * summed[:, None]) * inv[:, None]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,real,k,tempered", [(1, 9, 9, 3, False), (5, 300, 257, 0, True), (11, 8192, 8192, 64, True), (6, 50257, 50001, 20, False), (130, 8200, 8200, 5, True)])
def test_gradients_match_the_definition(ops, rows, vocab, real, k, tempered, dtype):
    z = _logits(rows, vocab, 2 * rows + vocab, dtype, scale=2.0)
    z[:, real:] = float("nan")
    if vocab > 100:
        z[:, 2:real:7] = NEG
    z.requires_grad_(True)
    target = torch.randint(0, real // 7 + 1, (rows,), generator=_gen(5), device=DEV) * 7
    target.clamp_(max=real - 1)
    temp = 0.5 + torch.rand(rows, generator=_gen(6), device=DEV) if tempered else None
    scores = ops.deterministic_scores_from_logits(z, target, top_k=k, temperature=temp, real_vocab_size=real)
    g = [torch.randn(rows, generator=_gen(20 + i), device=DEV) for i in range(3)]
    g_top = torch.randn((rows, k), generator=_gen(30), device=DEV) if k else None
    outputs = [scores.logp, scores.lse, scores.entropy] + ([scores.top_logp] if k else [])
    (grad,) = torch.autograd.grad(outputs, [z], g + ([g_top] if k else []))
    assert grad.dtype == dtype and grad.shape == z.shape
    assert not bool(grad[:, real:].any())
    with torch.no_grad():
        want, size = _gradient(z[:, :real], target, temp, scores.top_ids, *g, g_top)
        off = (grad[:, :real].double() - want).abs()
        tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-130
        assert bool((off <= HALF_STEP[dtype] * want.abs() + size + tiny).all()), float((off / (size + tiny)).max())


def test_gradient_against_differences(ops):
    """Central differences of the forward itself: h = 2^-5, so the third derivative (at most a few) leaves h^2, and the forward's
    rounding, 2^-21 of its values up to 10, leaves 2^-21 10 / h."""
    rows, vocab, k, h = 4, 40, 3, 2.0**-5
    z = _logits(rows, vocab, 12, scale=1.0)
    target = torch.tensor([0, 5, 39, 20], device=DEV)
    temp = torch.tensor([1.0, 0.75, 2.0, 1.5], device=DEV)
    weights = [torch.randn(rows, generator=_gen(40 + i), device=DEV) for i in range(3)] + [torch.randn((rows, k), generator=_gen(44), device=DEV)]
    ids = ops.deterministic_scores_from_logits(z, target, top_k=k, temperature=temp).top_ids

    def loss(z):
        s = ops.deterministic_scores_from_logits(z, target, top_k=k, temperature=temp)
        return s, [s.logp, s.lse, s.entropy, s.top_logp]

    zg = z.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(loss(zg)[1], [zg], weights)
    for column in (0, 5, 20, 39, int(ids[0, 0]), int(ids[2, 1])):
        ends = []
        for sign in (1.0, -1.0):
            moved = z.clone()
            moved[:, column] += sign * h
            s, outputs = loss(moved)
            assert s.top_ids.sort(1).values.shape == ids.shape
            at = {int(r): [s.top_ids[r].tolist().index(i) if i in s.top_ids[r].tolist() else None for i in ids[r].tolist()] for r in range(rows)}
            total = sum((w * o).double() for w, o in zip(weights[:3], outputs[:3]))
            for r in range(rows):
                y = moved[r].double() / temp[r].double()
                logq = y - torch.logsumexp(y, 0)
                for j, place in enumerate(at[r]):
                    value = s.top_logp[r, place].double() if place is not None else logq[ids[r, j]]
                    total[r] += weights[3][r, j].double() * value
            ends.append(total)
        slope = (ends[0] - ends[1]) / (2 * h)
        assert bool(((slope - grad[:, column].double()).abs() <= 8 * h * h + 2.0**-21 * 40 / h).all())


def test_only_what_is_differentiated_is_asked_for(ops):
    z = _logits(7, 900, 15)
    target = torch.arange(7, device=DEV)
    for pick in ("logp", "lse", "entropy", "top_logp"):
        zg = z.clone().requires_grad_(True)
        scores = ops.deterministic_scores_from_logits(zg, target, top_k=4)
        out = getattr(scores, pick)
        assert out.requires_grad and not scores.top_ids.requires_grad
        (grad,) = torch.autograd.grad(out.sum(), [zg])
        zero, one = torch.zeros(7, device=DEV), torch.ones(7, device=DEV)
        g = {"logp": (one, zero, zero, None), "lse": (zero, one, zero, None), "entropy": (zero, zero, one, None),
             "top_logp": (zero, zero, zero, torch.ones((7, 4), device=DEV))}[pick]  # fmt: skip
        want, size = _gradient(z, target, None, scores.top_ids, *g)
        assert bool(((grad.double() - want).abs() <= size + 2.0**-24 * want.abs() + 2.0**-130).all())
    with pytest.raises(RuntimeError):  # a gradient of the gradient is not served
        zg = z.clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(ops.deterministic_scores_from_logits(zg, target).entropy.sum(), [zg], create_graph=True)
        grad.sum().backward()


# ---------------------------------------------------------------------------
# From hidden states. Hidden states and weights on grids of 1/16 and 1/512: every product's sum is exact in fp32.
# ---------------------------------------------------------------------------


def _head(tokens, vocab, hidden, seed):
    h = (torch.randn((tokens, hidden), generator=_gen(seed), device=DEV) * 16).round().clamp(-64, 64).div(16).bfloat16()
    w = (torch.randn((vocab, hidden), generator=_gen(seed + 1), device=DEV) * (1024 / math.sqrt(hidden))).round().clamp(-64, 64).div(512).bfloat16()
    return h, w, torch.randint(0, vocab, (tokens,), generator=_gen(seed + 2), device=DEV)


@pytest.mark.parametrize("tokens,vocab,hidden,real,k,tempered", [(1, 1000, 64, 1000, 5, False), (17, 1030, 256, 1000, 64, True), (300, 4096, 128, 4096, 20, True), (64, 18992, 512, 18992, 0, False), (3, 77, 24, 70, 3, True)])
def test_linear_scores_match_the_definitions(ops, tokens, vocab, hidden, real, k, tempered):
    h, w, target = _head(tokens, vocab, hidden, tokens + vocab)
    target.clamp_(max=real - 1)
    temp = 0.5 + torch.rand(tokens, generator=_gen(6), device=DEV) if tempered else None
    scores = ops.deterministic_linear_scores(h, w, target, top_k=k, temperature=temp, real_vocab_size=real)
    z = (h.double() @ w.double().t())[:, :real]
    _check(scores, z, target, k, temp, 16 * vocab)  # (the fused pass has chains of up to 64 in a stream and one over splits)
    logp, lse = ops.deterministic_linear_logp(h, w, target, temperature=temp, real_vocab_size=real)
    assert torch.equal(scores.logp.view(torch.int32), logp.view(torch.int32))
    assert torch.equal(scores.lse.view(torch.int32), lse.view(torch.int32))


@pytest.mark.parametrize("tokens,k", [(5, 64), (5, 0), (1030, 0)])
def test_linear_scores_of_more_splits_than_a_wave_holds(ops, tokens, k):
    h, w, target = _head(tokens, 600011, 64, 77)
    s = ops.deterministic_linear_scores(h, w, target, top_k=k)
    logp, lse = ops.deterministic_linear_logp(h, w, target)
    assert torch.equal(s.logp.view(torch.int32), logp.view(torch.int32)) and torch.equal(s.lse.view(torch.int32), lse.view(torch.int32))
    rows = slice(tokens - 5, tokens)
    some = type(s)(*(None if t is None else t[rows] for t in s))
    _check(some, h[rows].double() @ w.double().t(), target[rows], k, None, 16 * 600011)


@pytest.mark.parametrize("tokens", [40, 1100])
@pytest.mark.parametrize("k", [0, 3])
def test_linear_scores_of_ids_and_temperatures_that_name_nothing(ops, tokens, k):
    h, w, target = _head(tokens, 3000, 64, 5)
    temp = 0.5 + torch.rand(tokens, generator=_gen(6), device=DEV)
    clean = ops.deterministic_linear_scores(h, w, target.clamp(max=2899), top_k=k, temperature=temp, real_vocab_size=2900)
    target = target.clamp(max=2899)
    for row, value in ((1, -1), (4, 2900), (7, 2999), (9, 3000), (30, 1 << 40)):
        target[row] = value
    for row, value in ((4, 0.0), (12, -1.0), (13, float("nan"))):
        temp[row] = value
    s = ops.deterministic_linear_scores(h, w, target, top_k=k, temperature=temp, real_vocab_size=2900)
    logp, lse = ops.deterministic_linear_logp(h, w, target, temperature=temp, real_vocab_size=2900)
    assert torch.equal(s.logp.view(torch.int32), logp.view(torch.int32)) and torch.equal(s.lse.view(torch.int32), lse.view(torch.int32))
    no_id, no_temperature = torch.tensor([1, 4, 7, 9, 30], device=DEV), torch.tensor([4, 12, 13], device=DEV)
    assert bool(torch.isnan(s.logp[no_id]).all()) and all(bool(torch.isnan(t[no_temperature]).all()) for t in s[:3])
    rest = torch.ones(tokens, dtype=torch.bool, device=DEV)
    rest[no_id], rest[no_temperature] = False, False
    for a, b in zip(s, clean):
        assert a is None or torch.equal(a[rest], b[rest])


@pytest.mark.parametrize("kind", ["five rows", "one row", "rising", "falling", "a block at the end", "all but some masked"])
@pytest.mark.parametrize("vocab,real", [(1030, 1001), (70000, 70000), (151936, 151669)])
def test_alternatives_of_hidden_states_wherever_they_lie(ops, kind, vocab, real):
    """Columns of one logit in many splits of the vocabulary, and the largest ones side by side."""
    h = torch.ones((3, 64), dtype=torch.bfloat16, device=DEV)
    h[1] *= -1
    column = torch.arange(vocab, device=DEV)
    bias = None
    if kind == "five rows":
        value = torch.randn(5, generator=_gen(1), device=DEV)[torch.randint(0, 5, (vocab,), generator=_gen(2), device=DEV)]
    elif kind == "one row":
        value = torch.ones(vocab, device=DEV)
    elif kind == "a block at the end":
        value = torch.where(column >= real - 70, 2.0, 1.0) + torch.randn(vocab, generator=_gen(3), device=DEV) * 0.01
    else:
        value = column / vocab * (-1 if kind == "falling" else 1)
    if kind == "all but some masked":
        bias = torch.full((vocab,), NEG, device=DEV)
        bias[[3, 1000, real - 1]] = 0.0
    w = value.to(torch.bfloat16)[:, None].expand(vocab, 64).contiguous()
    z = h.double() @ w.double().t()
    z = (z if bias is None else z + bias.double())[:, :real]
    for k in (1, 20, 64):
        s = ops.deterministic_linear_scores(h, w, torch.zeros(3, dtype=torch.long, device=DEV), bias, top_k=k, real_vocab_size=real)
        want = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(s.top_ids, want), (k, s.top_ids, want)


def test_linear_scores_with_a_bias(ops):
    h, w, target = _head(9, 640, 64, 31)
    bias = torch.randn(640, generator=_gen(33), device=DEV).mul(64).round().div(64)
    scores = ops.deterministic_linear_scores(h.view(3, 3, 64), w, target.view(3, 3), bias, top_k=4)
    assert scores.logp.shape == (3, 3) and scores.top_ids.shape == (3, 3, 4)
    flat = type(scores)(*(t.reshape(9, *t.shape[2:]) for t in scores))
    _check(flat, h.double() @ w.double().t() + bias.double(), target, 4, None, 16 * 640)
    with pytest.raises(RuntimeError, match="bias"):
        ops.deterministic_linear_scores(h, w, target, bias.requires_grad_(True))


@pytest.mark.parametrize("tokens,vocab,hidden,k,tempered", [(1, 1000, 64, 5, False), (33, 1030, 256, 7, True), (520, 4096, 128, 0, True), (40, 2050, 1536, 3, False)])
def test_linear_gradients(ops, tokens, vocab, hidden, k, tempered):
    """d(logits) is rounded to bf16 (2^-8 of each at most), then a product over the vocabulary or the tokens, rounded again."""
    h, w, target = _head(tokens, vocab, hidden, 3 * tokens + vocab)
    temp = 0.5 + torch.rand(tokens, generator=_gen(6), device=DEV) if tempered else None
    h.requires_grad_(True), w.requires_grad_(True)
    g = [torch.randn(tokens, generator=_gen(20 + i), device=DEV) for i in range(3)]
    g_top = torch.randn((tokens, k), generator=_gen(30), device=DEV) if k else None

    def grads():
        s = ops.deterministic_linear_scores(h, w, target, top_k=k, temperature=temp)
        outputs = [s.logp, s.lse, s.entropy] + ([s.top_logp] if k else [])
        return s, torch.autograd.grad(outputs, [h, w], g + ([g_top] if k else []))

    scores, (dh, dw) = grads()
    with torch.no_grad():
        z = h.double() @ w.double().t()
        dz, size = _gradient(z, target, temp, scores.top_ids, *g, g_top)
        slack = 2.0**-8 * dz.abs() + 1.01 * size
        for got, want, room in ((dh, dz @ w.double(), slack @ w.double().abs()), (dw, dz.t() @ h.double(), slack.t() @ h.double().abs())):
            assert got.dtype == torch.bfloat16
            assert bool(((got.double() - want).abs() <= 2.0**-8 * want.abs() + 1.01 * room + 2.0**-130).all())
    with ops.recompute_logits():
        again = grads()
    for a, b in zip([*scores[:3], dh, dw], [*again[0][:3], *again[1]]):
        assert torch.equal(a, b)
    (only,) = torch.autograd.grad(ops.deterministic_linear_scores(h.detach(), w, target, temperature=temp).entropy.sum(), [w])
    assert only.shape == w.shape


@pytest.mark.parametrize("rows,parts_of_it", [(256, 3), (100, 7)])
def test_a_buffer_of_some_tokens_gives_the_same_bits(ops, monkeypatch, rows, parts_of_it):
    from rl_engine import _C
    from rl_engine.backends.rocm.logprob import token_scores

    h, w, target = _head(700, 1030, 256, 55)
    temp = 0.5 + torch.rand(700, generator=_gen(6), device=DEV)
    whole = ops.deterministic_linear_scores(h, w, target, top_k=5, temperature=temp)
    h.requires_grad_(True), w.requires_grad_(True)
    with ops.recompute_logits():
        first = torch.autograd.grad([ops.deterministic_linear_scores(h, w, target, top_k=5, temperature=temp).entropy.sum()], [h, w])
        monkeypatch.setattr(token_scores, "_LOGITS_BUFFER_BYTES", rows * 4 * _C.linear_logp_logits_row_stride(1030))
        assert len(token_scores._token_chunks(700, 1030)) == parts_of_it
        parts = ops.deterministic_linear_scores(h, w, target, top_k=5, temperature=temp)
        second = torch.autograd.grad([parts.entropy.sum()], [h, w])
    for a, b in zip([*whole, *first], [*parts, *second]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("tokens,vocab,hidden,real,tempered", [(1056, 4096, 128, 4096, False), (1100, 1030, 64, 1001, True), (1280, 18992, 64, 18992, True), (1400, 300, 256, 300, False)])
def test_a_token_has_the_same_bits_with_and_without_logits(ops, tokens, vocab, hidden, real, tempered):
    """Above 1024 tokens the entropy comes out of the product's fold; with alternatives, in smaller batches and where the logits are
    kept for a backward it comes from logits that were stored."""
    from rl_engine import _C

    h, w, target = _head(tokens, vocab, hidden, tokens)
    target.clamp_(max=real - 1)
    temp = 0.5 + torch.rand(tokens, generator=_gen(6), device=DEV) if tempered else None
    assert not _C.linear_scores_needs_logits(h, w, None, 0) and _C.linear_scores_needs_logits(h, w, None, 1)
    assert _C.linear_scores_needs_logits(h[:1024], w, None, 0)
    call = ops.deterministic_linear_scores
    whole = call(h, w, target, temperature=temp, real_vocab_size=real)
    want = _reference((h.double() @ w.double().t())[:, :real], target, 0, temp)
    bound = _bound((h.double() @ w.double().t())[:, :real], 16 * vocab, temp)
    _close(whole.entropy, want["entropy"], 2 * (math.log(vocab) + 1) * bound)
    top = call(h, w, target, top_k=3, temperature=temp, real_vocab_size=real)
    grad_h = h.clone().requires_grad_(True)
    trained = call(grad_h, w, target, temperature=temp, real_vocab_size=real)
    stored = torch.empty((tokens, _C.linear_logp_logits_row_stride(vocab)), dtype=torch.float32, device=DEV)
    kept = _C.linear_scores(h, w, target, None, temp, real, 0, stored)
    for other in (top, trained, kept):
        for a, b in zip(whole[:3], other[:3]):
            assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    for rows in (slice(0, 1), slice(300, 420), slice(tokens - 70, tokens), slice(0, 1024)):
        part = call(h[rows], w, target[rows], temperature=None if temp is None else temp[rows], real_vocab_size=real)
        for a, b in zip(part[:3], whole[:3]):
            assert torch.equal(a.view(torch.int32), b[rows].view(torch.int32))
    grads = [torch.autograd.grad(trained.entropy.sum(), [grad_h])[0]]
    with ops.recompute_logits():
        grads.append(torch.autograd.grad(call(grad_h, w, target, temperature=temp, real_vocab_size=real).entropy.sum(), [grad_h])[0])
    assert torch.equal(*grads)


# ---------------------------------------------------------------------------
# Streams, graphs, sizes
# ---------------------------------------------------------------------------


def test_on_another_stream_and_in_a_graph(ops):
    z = _logits(65, 5000, 21, torch.bfloat16).requires_grad_(True)
    target = torch.randint(0, 5000, (65,), generator=_gen(9), device=DEV)
    g = [torch.randn(65, generator=_gen(50), device=DEV), torch.randn(65, generator=_gen(51), device=DEV)]

    def step():
        s = ops.deterministic_scores_from_logits(z, target, top_k=9, temperature=0.8)
        return [*(t.detach() for t in s), *torch.autograd.grad([s.logp, s.entropy], [z], g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    eager = step()
    for a, b in zip(other, eager):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            z.copy_(_logits(65, 5000, 60 + seed, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_no_rows(ops):
    z = torch.empty((0, 100), device=DEV, requires_grad=True)
    scores = ops.deterministic_scores_from_logits(z, torch.empty(0, dtype=torch.long, device=DEV), top_k=3)
    assert scores.logp.shape == (0,) and scores.top_ids.shape == (0, 3)
    (grad,) = torch.autograd.grad(scores.entropy.sum() + scores.top_logp.sum(), [z])
    assert grad.shape == (0, 100)
    h, w = torch.empty((0, 64), dtype=torch.bfloat16, device=DEV), torch.ones((100, 64), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    scores = ops.deterministic_linear_scores(h, w, torch.empty(0, dtype=torch.long, device=DEV), top_k=3)
    (grad,) = torch.autograd.grad(scores.entropy.sum(), [w])
    assert not bool(grad.any())


def test_rows_beyond_four_gigabytes(ops):
    """A row behind 2^32 bytes of logits answers as it does alone."""
    rows, vocab = 16500, 131072
    z = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=DEV)
    last = _logits(2, vocab, 3, torch.bfloat16)
    z[-2:] = last
    target = torch.full((rows,), 7, device=DEV)
    scores = ops.deterministic_scores_from_logits(z, target, top_k=2)
    alone = ops.deterministic_scores_from_logits(last, target[:2], top_k=2)
    for s, a in zip(scores, alone):
        assert torch.equal(s[-2:], a)
    assert scores.top_ids[100].tolist() == [0, 1]


def test_refused_calls(ops):
    z, target = _logits(4, 100, 1), torch.zeros(4, dtype=torch.long, device=DEV)
    call = ops.deterministic_scores_from_logits
    for kwargs in ({"top_k": 65}, {"top_k": -1}, {"real_vocab_size": 0}, {"real_vocab_size": 101}, {"real_vocab_size": 5, "top_k": 6},
                   {"temperature": torch.ones(3, device=DEV)}):  # fmt: skip
        with pytest.raises(ValueError):
            call(z, target, **kwargs)
    for top_k in (2.0, True):
        with pytest.raises(TypeError):
            call(z, target, top_k=top_k)
    for bad in (target[:3], target.view(2, 2), target.cpu()):
        with pytest.raises(ValueError):
            call(z, bad)
    with pytest.raises(TypeError):
        call(z.double(), target)
    with pytest.raises(RuntimeError):
        call(z.cpu(), target.cpu())
    with pytest.raises(ValueError, match="real vocabulary"):
        call(z, target + 100, validate=True)
    with pytest.raises(ValueError, match="temperature"):
        call(z, target, temperature=0.0, validate=True)
    h, w = torch.ones((4, 64), dtype=torch.bfloat16, device=DEV), torch.ones((100, 64), dtype=torch.bfloat16, device=DEV)
    linear = ops.deterministic_linear_scores
    with pytest.raises(ValueError):
        linear(h, w, target[:3])
    with pytest.raises(ValueError):
        linear(h, w, target, top_k=65)
    with pytest.raises(ValueError):
        linear(h, w[:, :32], target)
    with pytest.raises(TypeError):
        linear(h.float(), w, target)
