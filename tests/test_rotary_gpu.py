"""Rotary positions and appending to a paged cache on a real MI355X against the definition in 64 bits.

Tolerance of an element: sine and cosine are correct to 2 ulp of 2^-24 of 1 for an angle that is rounded to 2^-25 of a turn's half (pi times that,
2^-23), and the two products and their sum take 3 roundings of 2^-24: 8 steps of 2^-23 of the pair's magnitudes, then half a step of the type."""

from __future__ import annotations

import pytest
import torch

from attention_cases import DEV, HALF_STEP, Batch, same_bits

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def attention():
    from rl_engine.ops import attention

    return attention


def _normal(*shape, seed=0, dtype=BF16):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def _definition(x, positions, frequencies, interleaved, magnitude=1.0, inverse=False):
    """(value, the sum of the magnitudes that it is made of), in 64 bits."""
    x = x.double()
    pairs = frequencies.numel()
    angle = positions.double().unsqueeze(-1) * frequencies * (-1 if inverse else 1)
    cos, sin = angle.cos().unsqueeze(-2) * magnitude, angle.sin().unsqueeze(-2) * magnitude
    first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
    out, size = x.clone(), x.abs()
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(magnitude)
    return out, size


def _near(got, want, size, copied_from=None):
    bound = HALF_STEP[got.dtype] * want.abs() + 8 * 2.0**-23 * size + (2.0**-25 if got.dtype == FP16 else 2.0**-126)
    off = (got.double() - want).abs()
    assert got.shape == want.shape and bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("tokens", (1, 3, 1030))
@pytest.mark.parametrize("heads, key_heads, width, part", [(8, 2, 128, 128), (3, 1, 64, 32), (5, 5, 80, 20), (2, 1, 33, 6), (1, 3, 256, 64), (2, 2, 10, 10), (2, 1, 1024, 1024), (4, 1, 24, 0)])
def test_definition(attention, dtype, interleaved, tokens, heads, key_heads, width, part):
    q, k = _normal(tokens, heads, width, seed=1, dtype=dtype), _normal(tokens, key_heads, width, seed=2, dtype=dtype)
    positions = torch.arange(tokens, device=DEV) * 7 % 5003
    f = attention.rotary_frequencies(part, device=DEV) if part else torch.empty(0, dtype=torch.float64, device=DEV)
    got = attention.rotary_embedding(q, k, positions, f, interleaved=interleaved)
    for x, y in zip((q, k), got):
        _near(y, *_definition(x, positions, f, interleaved))
        assert same_bits(y[..., part:], x[..., part:]) and y.is_contiguous()
    alone, none = attention.rotary_embedding(q, None, positions.int(), f, interleaved=interleaved)
    assert none is None and same_bits(alone, got[0])


@pytest.mark.parametrize("start", (0, 10**6, 2**31 - 2000, 2**40, -5000))
def test_far_positions(attention, start):
    q = _normal(1000, 2, 64, seed=3, dtype=FP32)
    positions = start + torch.arange(1000, device=DEV)
    f = attention.rotary_frequencies(64, 1e6, device=DEV)
    # an angle in 64 bits is off by 2^-52 of itself, in the definition as well
    got, want = attention.rotary_embedding(q, None, positions, f)[0].double(), _definition(q, positions, f, False)
    bound = 2.0**-24 * want[0].abs() + (8 * 2.0**-23 + 4 * 2.0**-52 * abs(start)) * want[1]
    assert bool(((got - want[0]).abs() <= bound).all())


def test_layouts_and_magnitude(attention):
    f = attention.rotary_frequencies(32, device=DEV)
    x = _normal(2, 6, 50, 48, seed=4)  # batch, heads, tokens, width
    positions = torch.randint(0, 10000, (2, 50), generator=torch.Generator(device=DEV).manual_seed(5), device=DEV)
    q = x.transpose(1, 2)
    k = _normal(2, 50, 9, 48, seed=6)[:, :, 3:5]
    got = attention.rotary_embedding(q, k, positions, f, magnitude=1.25)
    for t, y in zip((q, k), got):
        _near(y, *_definition(t, positions, f, False, 1.25))
    plain = attention.rotary_embedding(q.contiguous(), k.contiguous(), positions, f, magnitude=1.25)
    assert same_bits(plain[0], got[0]) and same_bits(plain[1], got[1])
    five = attention.rotary_embedding(q.unsqueeze(0).expand(3, 2, 50, 6, 48), None, positions.expand(3, 2, 50), f, magnitude=1.25)[0]
    assert all(same_bits(part, got[0]) for part in five)
    odd = torch.zeros(2 * 50 * 6 * 48 + 1, device=DEV, dtype=BF16)[1:].view(2, 50, 6, 48)
    odd.copy_(q)
    assert same_bits(attention.rotary_embedding(odd, None, positions, f, magnitude=1.25)[0], got[0])
    last = q.transpose(-1, -2).contiguous().transpose(-1, -2)  # elements apart
    assert same_bits(attention.rotary_embedding(last, None, positions, f, magnitude=1.25)[0], got[0])
    none = attention.rotary_embedding(q[:, :0], k[:, :0], positions[:, :0], f)
    assert none[0].shape == (2, 0, 6, 48) and none[1].shape == (2, 0, 2, 48)


@pytest.mark.parametrize("dtype", (BF16, FP32))
@pytest.mark.parametrize("interleaved", (False, True))
def test_gradients(attention, dtype, interleaved):
    q, k = _normal(70, 4, 40, seed=7, dtype=dtype).requires_grad_(), _normal(70, 2, 40, seed=8, dtype=dtype).requires_grad_()
    positions, f = torch.arange(70, device=DEV) + 90000, attention.rotary_frequencies(16, device=DEV)
    y = attention.rotary_embedding(q, k, positions, f, interleaved=interleaved, magnitude=0.8)
    g = [_normal(*t.shape, seed=9, dtype=dtype) for t in y]
    grads = torch.autograd.grad(y, [q, k], g, retain_graph=True)
    for got, given in zip(grads, g):
        _near(got, *_definition(given, positions, f, interleaved, 0.8, inverse=True))
    only = torch.autograd.grad(y[1], [k], g[1], retain_graph=True)[0]
    assert same_bits(only, grads[1])
    one = torch.autograd.grad(y[0].sum(), [q, k], allow_unused=True)  # a gradient that is one number, repeated
    assert one[1] is None
    _near(one[0], *_definition(torch.ones_like(q), positions, f, interleaved, 0.8, inverse=True))


def test_gradients_against_differences_and_of_gradients(attention):
    q = _normal(5, 2, 12, seed=10, dtype=FP32).requires_grad_()
    positions, f = torch.arange(5, device=DEV) * 3, attention.rotary_frequencies(8, device=DEV)
    w = _normal(5, 2, 12, seed=11, dtype=FP32)

    def loss(x):
        return (attention.rotary_embedding(x, None, positions, f, magnitude=1.5)[0].double().pow(2) * w).sum()

    (grad,) = torch.autograd.grad(loss(q), q, create_graph=True)
    step = 2.0**-6  # a quadratic: central differences are exact but for rounding, 2^-24 of sums of about 100 over a step
    for at in ((0, 0, 0), (2, 1, 5), (4, 0, 7), (3, 1, 11)):
        d = torch.zeros_like(q)
        d[at] = step
        with torch.no_grad():
            slope = (loss(q + d) - loss(q - d)) / (2 * step)
        assert abs(float(slope.detach() - grad.detach()[at])) <= 100 * 8 * 2.0**-23 / step
    (second,) = torch.autograd.grad(grad.sum(), q)  # 2 R^T diag(w) R 1
    ones = torch.ones_like(q)
    turned = attention.rotary_embedding(ones, None, positions, f, magnitude=1.5)[0].double()
    want, size = _definition(2 * w * turned, positions, f, False, 1.5, inverse=True)
    assert bool(((second.double() - want).abs() <= 32 * 2.0**-23 * (size + 1)).all())


def test_frequencies(attention):
    f = attention.rotary_frequencies
    plain = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    assert torch.allclose(f(64, device="cpu"), plain, rtol=1e-14)
    assert torch.allclose(f(64, factor=4.0, device="cpu"), plain / 4, rtol=1e-14)
    scaled = f(64, factor=4.0, scaling="base", device="cpu")
    assert float(scaled[0]) == 1.0 and abs(float(scaled[-1] * 4 / plain[-1]) - 1) < 1e-12
    for kind in ("bands", "wavelengths"):
        both = f(64, factor=4.0, scaling=kind, original_length=4096, device="cpu")
        turns = 4096 * plain / (2 * torch.pi)
        assert torch.equal(both[turns > 40], plain[turns > 40]) and torch.allclose(both[turns < 0.7], plain[turns < 0.7] / 4, rtol=1e-14)
        assert bool((both <= plain).all()) and bool((both >= plain / 4 * (1 - 1e-12)).all())


# ---------------------------------------------------------------------------
# Appending
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("lengths", ([(1, 1), (1, 40), (0, 12), (1, 17)], [(30, 30), (5, 100), (0, 0), (300, 1100), (2, 2)]), ids=("single", "chunks"))
@pytest.mark.parametrize("heads, key_heads, width, part, page, interleaved", [(4, 2, 128, 128, 16, False), (3, 1, 80, 20, 7, True), (2, 2, 33, 6, 1, False), (0, 2, 64, 0, 64, False)])
@pytest.mark.parametrize("order", ("rows", "heads", "pairs"))
def test_append(attention, dtype, lengths, heads, key_heads, width, part, page, interleaved, order):
    b = Batch(lengths, max(heads, 1), key_heads, width, page, dtype, seed=20, order=order, behind=3)
    tokens = b.tokens + 3
    rows = _normal(tokens, 2 * key_heads + heads, width, seed=21, dtype=dtype)
    q, k, v = rows.split([heads, key_heads, key_heads], dim=1)
    f = attention.rotary_frequencies(part, device=DEV) if part else None
    keys, values = b.keys.clone(), b.values.clone()
    turned = attention.paged_append(k, v, *b.where, f, q=q if heads else None, interleaved=interleaved)
    positions = torch.cat([torch.arange(c - n, c, device=DEV) for n, c in lengths])
    sequence = torch.cat([torch.full((n,), i, device=DEV) for i, (n, _) in enumerate(lengths)])
    page_of, row = b.table.long()[sequence, positions // page], positions % page
    padded = torch.nn.functional.pad(positions, (0, 3))
    if f is None:
        want_k, want_q = k, None
        assert turned is None
    else:
        want_q, want_k = attention.rotary_embedding(q, k, padded, f, interleaved=interleaved)
        assert same_bits(turned[: b.tokens], want_q[: b.tokens]) and not bool(turned[b.tokens :].any())
    keys[page_of, row], values[page_of, row] = want_k[: b.tokens], v[: b.tokens]
    assert same_bits(b.keys, keys) and same_bits(b.values, values)


def test_append_positions_of_ones_own(attention):
    b = Batch([(4, 9), (6, 6)], 2, 2, 64, 16, BF16, seed=22)
    k, v = _normal(10, 2, 64, seed=23), _normal(10, 2, 64, seed=24)
    f = attention.rotary_frequencies(64, device=DEV)
    for positions in (torch.arange(10, device=DEV) * 1000, torch.arange(10, device=DEV, dtype=torch.int32) + 5):
        q = attention.paged_append(k, v, *b.where, f, q=b.q, positions=positions, magnitude=1.1)
        want_q, want_k = attention.rotary_embedding(b.q, k, positions, f, magnitude=1.1)
        assert same_bits(q, want_q)
        place = torch.tensor([5, 6, 7, 8], device=DEV)
        assert same_bits(b.keys[b.table[0, 0].long(), place], want_k[:4]) and same_bits(b.values[b.table[1, 0].long(), place - 5], v[4:8])


def test_append_to_places_that_are_missing(attention):
    b = Batch([(5, 3), (20, 40), (3, 40), (2, 90)], 2, 1, 64, 16, BF16, seed=25)
    b.table[1, 1], b.table[2, 2] = b.keys.size(0), -1
    keys = b.keys.clone()
    k, v = _normal(30, 1, 64, seed=26), _normal(30, 1, 64, seed=27)
    attention.paged_append(k, v, b.keys, b.values, b.table[:, :5], b.contexts, b.starts)
    keys[b.table[0, 0].long(), :3] = k[2:5]  # of the five, two lie before the start
    keys[b.table[1, 2].long(), :8] = k[17:25]  # positions 32 ... 39; 20 ... 31 have no page
    assert same_bits(b.keys, keys)  # nor has the third sequence, and the fourth's lies behind the table


def test_append_of_nothing(attention):
    b = Batch([(0, 5), (0, 0)], 2, 1, 64, 16, BF16, seed=28)
    keys = b.keys.clone()
    q = attention.paged_append(b.q[:, :1], b.q[:, :1], *b.where, attention.rotary_frequencies(64, device=DEV), q=b.q)
    assert q.shape == (0, 2, 64) and same_bits(b.keys, keys)
    k = _normal(3, 1, 64, seed=29)
    empty = torch.empty((0, 3), device=DEV, dtype=torch.int32)
    q = attention.paged_append(k, k, b.keys, b.values, empty, b.contexts[:0], b.starts[:1], q=_normal(3, 2, 64, seed=30))
    assert not bool(q.any()) and same_bits(b.keys, keys)


def test_append_captured(attention):
    b = Batch([(1, 20), (1, 33)], 4, 2, 128, 16, BF16, seed=31)
    k, v = _normal(2, 2, 128, seed=32), _normal(2, 2, 128, seed=33)
    f = attention.rotary_frequencies(128, device=DEV)
    attention.paged_append(k, v, *b.where, f, q=b.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = attention.paged_append(k, v, *b.where, f, q=b.q)
        out = attention.paged_attention(q, *b.where)
    for step in range(3):
        b.contexts.copy_(torch.tensor((20 - step, 33 - 2 * step), dtype=torch.int32))
        k.copy_(_normal(2, 2, 128, seed=40 + step))
        want_q = attention.paged_append(k, v, *b.where, f, q=b.q)
        want = attention.paged_attention(want_q, *b.where)
        keys = b.keys.clone()
        b.keys[b.table[0, 1].long()] = 0
        graph.replay()
        torch.cuda.synchronize()
        assert same_bits(q, want_q) and same_bits(out[1], want[1])
        assert same_bits(b.keys[b.table[1, 1].long()], keys[b.table[1, 1].long()])


def test_a_backward_in_a_graph(attention):
    positions, f = torch.arange(6, device=DEV), attention.rotary_frequencies(64, device=DEV)
    q, g = _normal(6, 2, 64, seed=34).requires_grad_(), _normal(6, 2, 64, seed=35)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        (warm,) = torch.autograd.grad(attention.rotary_embedding(q, None, positions, f)[0], q, g)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        (grad,) = torch.autograd.grad(attention.rotary_embedding(q, None, positions, f)[0], q, g)
    for seed in (36, 37):
        g.copy_(_normal(6, 2, 64, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        want, size = _definition(g, positions, f, False, inverse=True)
        _near(grad, want, size)
    assert warm.shape == grad.shape


def test_more_tokens_than_a_launch_has_workgroups(attention):
    tokens, f = 2**24 + 5, attention.rotary_frequencies(8, device=DEV)
    q = torch.randn((1024, 1, 8), device=DEV).to(BF16).repeat(tokens // 1024 + 1, 1, 1)[:tokens]
    positions = torch.arange(tokens, device=DEV)
    turned = attention.rotary_embedding(q, None, positions, f)[0]
    for first in (0, 2**20 - 3, 2**23, tokens - 7):
        rows = slice(first, first + 7)
        assert same_bits(turned[rows], attention.rotary_embedding(q[rows].clone(), None, positions[rows].clone(), f)[0])
