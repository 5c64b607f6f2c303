"""The attention block as it is used, on a real MI355X: a prompt in one piece, in chunks and token by token, next to other
sequences, through projection, norms of the heads, rotation, cache, attention and output projection."""

from __future__ import annotations

import pytest
import torch

from attention_cases import DEV, same_bits

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HEADS, KEY_HEADS, WIDTH, HIDDEN, PAGE = 8, 2, 64, 256, 16


def _normal(*shape, seed=0, scale=1.0, mean=0.0):
    return (torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * scale + mean).to(BF16)


class Layer:
    def __init__(self):
        from rl_engine.ops import attention

        self.attention = attention
        self.qkv = _normal((HEADS + 2 * KEY_HEADS) * WIDTH, HIDDEN, seed=1, scale=0.06)
        self.o = _normal(HIDDEN, HEADS * WIDTH, seed=2, scale=0.05)
        self.q_norm, self.k_norm = _normal(WIDTH, seed=3, scale=0.1, mean=1.0), _normal(WIDTH, seed=4, scale=0.1, mean=1.0)
        self.next = _normal(HIDDEN, seed=5, scale=0.1, mean=1.0)
        self.f = attention.rotary_frequencies(WIDTH, 1e6, device=DEV)

    def caches(self, pages):
        return tuple(torch.full((pages, PAGE, KEY_HEADS, WIDTH), float("nan"), device=DEV, dtype=BF16) for _ in range(2))

    def __call__(self, residual, normed, caches, table, lengths, starts, **how):
        return self.attention.qwen3_attention_block(
            residual, normed, self.qkv, self.o, *caches, table, lengths, starts, self.f, self.next, q_norm_weight=self.q_norm, k_norm_weight=self.k_norm, **how
        )


def _ints(*values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def _table(pages, first, columns):
    return (torch.randperm(pages, generator=torch.Generator(device=DEV).manual_seed(first), device=DEV, dtype=torch.int32))[:columns]


@pytest.mark.parametrize("window", (None, 50))
def test_a_prompt_in_one_piece_in_chunks_and_token_by_token(window):
    layer, length = Layer(), 300
    residual, normed = _normal(length, HIDDEN, seed=6), _normal(length, HIDDEN, seed=7)
    table = _table(25, 1, 20).view(1, -1)
    caches = layer.caches(25)
    want = layer(residual, normed, caches, table, _ints(length), _ints(0, length), window=window)
    for sizes in ([100, 1, 199], [256, 44], [290] + [1] * 10):
        mine, at, parts = layer.caches(25), 0, []
        for n in sizes:
            rows = slice(at, at + n)
            parts.append(layer(residual[rows], normed[rows], mine, table, _ints(at + n), _ints(0, n), window=window))
            at += n
        for i in range(2):
            assert same_bits(torch.cat([p[i] for p in parts]), want[i]), (sizes, i)
            used = table[0, : -(-length // PAGE)].long()
            flat = lambda c: c[used].flatten(0, 1)[:length]  # noqa: E731
            assert same_bits(flat(mine[i]), flat(caches[i]))


def test_a_batch_has_the_bits_of_its_sequences():
    layer = Layer()
    lengths = [(40, 40), (1, 200), (0, 7), (17, 90)]
    pages, columns = 60, 14
    perm = torch.randperm(pages, generator=torch.Generator(device=DEV).manual_seed(8), device=DEV, dtype=torch.int32)
    table = perm[: 4 * columns].view(4, columns)
    caches = layer.caches(pages)
    inputs = [(_normal(c, HIDDEN, seed=10 + i), _normal(c, HIDDEN, seed=20 + i)) for i, (_, c) in enumerate(lengths)]
    for i, ((n, c), (residual, normed)) in enumerate(zip(lengths, inputs)):  # the contexts, each on its own
        if c > n:
            layer(residual[: c - n], normed[: c - n], caches, table[i : i + 1], _ints(c - n), _ints(0, c - n))
    alone = []
    for i, ((n, c), (residual, normed)) in enumerate(zip(lengths, inputs)):
        mine = tuple(t.clone() for t in caches)
        alone.append(layer(residual[c - n :], normed[c - n :], mine, table[i : i + 1], _ints(c), _ints(0, n)) if n else None)
    starts = [0, 40, 41, 41, 58]
    new = [torch.cat([pair[j][c - n :] for (n, c), pair in zip(lengths, inputs)]) for j in range(2)]
    got = layer(*new, caches, table, _ints(*(c for _, c in lengths)), _ints(*starts))
    for i, want in enumerate(alone):
        if want is not None:
            for j in range(2):
                assert same_bits(got[j][starts[i] : starts[i + 1]], want[j])


def test_against_the_plain_formulas():
    """Every step is rounded to bf16 on the way (7 of them, half a step of 2^-8 each), and products of rounded operands add the roundings
    of their terms at random: 4 half steps of an output's deviation at most, taken over all of them."""
    layer, length = Layer(), 130
    residual, normed = _normal(length, HIDDEN, seed=30), _normal(length, HIDDEN, seed=31)
    total, after = layer(residual, normed, layer.caches(25), _table(25, 2, 20).view(1, -1), _ints(length), _ints(0, length))
    d = lambda t: t.double()  # noqa: E731
    qkv = d(normed) @ d(layer.qkv).t()
    q, k, v = (t.unflatten(1, (-1, WIDTH)) for t in qkv.split([HEADS * WIDTH, KEY_HEADS * WIDTH, KEY_HEADS * WIDTH], 1))
    norm = lambda t, w: t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * d(w)  # noqa: E731
    angle = torch.arange(length, device=DEV).double()[:, None, None] * layer.f

    def turned(t):
        a, b = t.chunk(2, -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

    q, k = turned(norm(q, layer.q_norm)), turned(norm(k, layer.k_norm))
    k, v = (t.repeat_interleave(HEADS // KEY_HEADS, 1) for t in (k, v))
    s = (q.transpose(0, 1) @ k.permute(1, 2, 0)) * WIDTH**-0.5
    s = s.masked_fill(torch.ones(length, length, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
    y = (s.softmax(-1) @ v.transpose(0, 1)).transpose(0, 1).flatten(1) @ d(layer.o).t()
    want = d(residual) + y
    assert float((total.double() - want).square().mean().sqrt()) <= 4 * 2.0**-8 * float(want.square().mean().sqrt())
    want = norm(want, layer.next)
    assert float((after.double() - want).square().mean().sqrt()) <= 4 * 2.0**-8 * float(want.square().mean().sqrt())


def test_decoding_in_a_graph():
    layer, steps, context = Layer(), 20, 55
    table = torch.stack([_table(40, 3, 8), _table(40, 3, 16)[8:]])
    residual, normed = _normal(2 * (context + steps), HIDDEN, seed=40), _normal(2 * (context + steps), HIDDEN, seed=41)
    starts = _ints(0, context, 2 * context)
    eager, captured = layer.caches(40), layer.caches(40)
    for caches in (eager, captured):
        layer(residual[: 2 * context], normed[: 2 * context], caches, table, _ints(context, context), starts)
    lengths, one = _ints(context, context), _ints(0, 1, 2)
    r, n = residual[:2].clone(), normed[:2].clone()
    lengths += 1
    layer(r, n, layer.caches(40), table, lengths, one)  # (the first call of a shape is not captured)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(r, n, captured, table, lengths, one)
    for step in range(steps):
        rows = slice(2 * context + 2 * step, 2 * context + 2 * step + 2)
        r.copy_(residual[rows])
        n.copy_(normed[rows])
        lengths.fill_(context + 1 + step)
        want = layer(r, n, eager, table, lengths.clone(), one)
        graph.replay()
        torch.cuda.synchronize()
        assert same_bits(got[0], want[0]) and same_bits(got[1], want[1]), step
    assert all(same_bits(a, b) for a, b in zip(eager, captured))


def test_refusals_of_the_block():
    layer = Layer()
    x = _normal(3, HIDDEN, seed=50)
    args = (layer.caches(4), _table(4, 1, 2).view(1, -1), _ints(3), _ints(0, 3))
    with pytest.raises(RuntimeError, match="no gradient"):
        layer(x.clone().requires_grad_(), x, *args)
    whole = layer.qkv
    for qkv in (whole[: 4 * WIDTH], whole[:-1]):
        layer.qkv = qkv
        with pytest.raises(ValueError, match="rows"):
            layer(x, x, *args)
