"""Paged attention and appending at the edges of what they are given: starts out of order, rows behind the page table, the largest
positions, memory that autograd watches."""

from __future__ import annotations

import pytest
import torch

from attention_cases import DEV, Batch, same_bits
from rl_engine import _lib

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
CONFIGS = tuple(name for name in _lib.ATTENTION_CONFIGS if name != "auto")


@pytest.fixture(scope="module")
def attention():
    from rl_engine.ops import attention

    return attention


def _ints(*values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def _normal(*shape, seed=0, dtype=BF16):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


OUT_OF_ORDER = [(0, 1000, 10, 1010), (1010, 500, 0, 3), (700, 0, 1010, 20), (-5, 2000, -7, 900), (3, 3, 1, 1), (1010, 0, 0, 0), (0, 5, 900, 1)]


@pytest.mark.parametrize("starts", OUT_OF_ORDER)
def test_starts_that_do_not_ascend_stay_within_the_tensors(attention, starts):
    b = Batch([(1, 700), (1, 900), (1, 1010)], 8, 2, 64, 16, BF16, seed=1)
    tokens, guard = 1010, 64
    room = torch.full((tokens + 2 * guard, 8, 64), 7.0, device=DEV, dtype=BF16)
    q = torch.zeros_like(room)[guard:-guard]
    for config in ("auto", *CONFIGS):
        for out in (None, room[guard:-guard]):
            attention.paged_attention(q, b.keys, b.values, b.table, b.contexts, _ints(*starts), out=out, return_lse=True, config=config)
        assert bool((room[:guard] == 7).all()) and bool((room[-guard:] == 7).all())


@pytest.mark.parametrize("starts", OUT_OF_ORDER)
def test_appending_with_starts_that_do_not_ascend_writes_new_places_alone(attention, starts):
    contexts = (700, 900, 1010)
    b = Batch([(1, c) for c in contexts], 8, 2, 64, 16, BF16, seed=1)
    k = _normal(1010, 2, 64, seed=2)
    keys = b.keys.clone()
    attention.paged_append(k, k, b.keys, b.values, b.table, b.contexts, _ints(*starts), q=k)
    for s, c in enumerate(contexts):
        new = min(max(0, starts[s + 1] - starts[s]), c)
        place = torch.arange(c - new, device=DEV)
        page, row = b.table[s].long()[place // 16], place % 16
        assert same_bits(b.keys[page, row], keys[page, row]), s
    used = torch.cat([b.table[s, : -(-c // 16)] for s, c in enumerate(contexts)]).long()
    rest = torch.ones(b.keys.size(0), dtype=torch.bool, device=DEV)
    rest[used] = False
    assert same_bits(b.keys[rest], keys[rest])


def test_a_token_that_no_ascending_search_finds_is_not_written(attention):
    """Token 3 of starts 0, 5, 6, 1: two of them are at most 3, and the second sequence starts behind it."""
    b = Batch([(1, 40), (1, 40), (1, 40)], 2, 1, 64, 16, BF16, seed=3)
    keys = b.keys.clone()
    k = _normal(6, 1, 64, seed=4)
    attention.paged_append(k, k, b.keys, b.values, b.table, b.contexts, _ints(0, 5, 6, 1))
    place = torch.arange(39, device=DEV)
    page, row = b.table[1].long()[place // 16], place % 16
    assert same_bits(b.keys[page, row], keys[page, row])


@pytest.mark.parametrize("config", ("auto", *CONFIGS))
@pytest.mark.parametrize("columns, window, new, context", [(4, 8, 1, 100), (4, 8, 1, 400), (4, 8, 40, 100), (4, 8, 1, 67), (4, 70, 30, 100), (8, 40, 300, 700), (20, 300, 5, 4000), (0, 8, 3, 100)])
@pytest.mark.parametrize("width, page", [(64, 16), (128, 16), (96, 17)])
def test_windowed_rows_behind_the_table(attention, config, columns, window, new, context, width, page):
    """Missing, whether the window reaches back into the table or not: NaN and a NaN logarithm. The rows in front keep their bits."""
    b = Batch([(new, context)], 4, 2, width, page, BF16, seed=7)
    want, want_lse = attention.paged_attention(b.q, *b.where, window=window, return_lse=True)
    table = b.table[:, :columns].contiguous()
    out, lse = attention.paged_attention(b.q, b.keys, b.values, table, b.contexts, b.starts, window=window, return_lse=True, config=config)
    inside = max(0, min(new, columns * page - (context - new)))  # rows at positions that the table has room for
    assert same_bits(out[:inside], want[:inside]) and same_bits(lse[:inside], want_lse[:inside])
    assert bool(out[inside:].isnan().all()) and bool(lse[inside:].isnan().all())


@pytest.mark.parametrize("config", ("auto", *CONFIGS))
def test_the_last_positions(attention, config):
    """Positions from 2^31 - 256 on have no place, whatever the table holds; the one in front of them is as any other."""
    page = 2**24
    keys, values = (torch.zeros((1, page, 1, 8), device=DEV, dtype=BF16) for _ in range(2))
    keys[0, -320:, 0], values[0, -320:, 0] = _normal(320, 8, seed=1), _normal(320, 8, seed=2)
    table, q = torch.zeros((1, 128), device=DEV, dtype=torch.int32), _normal(2, 2, 8, seed=3)
    run = lambda q, k, v, t, c: attention.paged_attention(q, k, v, t, _ints(c), _ints(0, q.size(0)), window=8, return_lse=True, config=config)  # noqa: E731
    near = keys[:, -320:-256].contiguous(), values[:, -320:-256].contiguous()
    want, want_lse = run(q[:1], *near, table[:, :1], 64)  # position 63 there, 2^31 - 257 here
    out, lse = run(q, keys, values, table, 2**31 - 255)
    assert same_bits(out[:1], want) and same_bits(lse[:1], want_lse)
    assert bool(out[1].isnan().all()) and bool(lse[1].isnan().all())
    out, lse = run(q, keys, values, table, 2**31 - 1)
    assert bool(out.isnan().all()) and bool(lse.isnan().all())


class _Nothing:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture(params=("native", "general"))
def way(request, monkeypatch):
    if request.param == "general":
        from rl_engine import _host

        monkeypatch.setattr(_host, "_native", _Nothing())
    return request.param


def test_autograd_sees_what_is_written(attention, way):
    b = Batch([(2, 40), (1, 33)], 4, 2, 64, 16, BF16, seed=5)
    k, f = _normal(3, 2, 64, seed=6), attention.rotary_frequencies(64, device=DEV)
    for which in ("keys", "values"):
        w = torch.ones((), device=DEV, dtype=BF16, requires_grad=True)
        kept = getattr(b, which) * w  # its backward reads the cache
        attention.paged_append(k, k, *b.where, f, q=b.q)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.sum().backward()
    whole = torch.zeros((3, 6, 64), device=DEV, dtype=BF16)
    w = torch.ones((), device=DEV, dtype=BF16, requires_grad=True)
    kept = whole * w
    before = [t._version for t in (*b.where, b.q)]
    attention.paged_attention(b.q, *b.where, out=whole[:, 1:5])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()
    assert before == [t._version for t in (*b.where, b.q)]  # it reads the others
    with pytest.raises(ValueError):
        attention.paged_append(k, k[:2], *b.where, f)
    assert before == [t._version for t in (*b.where, b.q)]


def test_caches_of_inference_mode(attention, way):
    b = Batch([(2, 40), (1, 33)], 4, 2, 64, 16, BF16, seed=5)
    k = _normal(3, 2, 64, seed=6)
    with torch.inference_mode():
        keys, values, out = b.keys.clone(), b.values.clone(), torch.zeros_like(b.q)
    attention.paged_append(k, k, *b.where)
    attention.paged_append(k, k, keys, values, *b.where[2:])  # (outside of the mode, they have no versions)
    assert same_bits(keys, b.keys) and same_bits(values, b.values)
    attention.paged_attention(b.q, keys, values, *b.where[2:], out=out)
    assert same_bits(out, attention.paged_attention(b.q, *b.where))
    with torch.inference_mode():
        attention.paged_append(k, k, *b.where)
