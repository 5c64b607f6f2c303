"""Attention over a paged cache on a real MI355X against its definition in 64 bits (bounds: attention_cases.Batch.bounds), and what its bits
may not depend on."""

from __future__ import annotations

import threading

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


SINGLE = [(1, 1), (1, 63), (1, 64), (1, 65), (1, 256), (1, 257), (1, 1000), (1, 4160)]
MIXED = [(5, 5), (0, 7), (3, 300), (1, 90), (7, 4), (0, 0), (40, 129)]
PROMPTS = [(70, 70), (33, 1000), (129, 129)]


@pytest.mark.parametrize("config", ("auto", *CONFIGS))
@pytest.mark.parametrize("lengths", (SINGLE, MIXED, PROMPTS), ids=("single", "mixed", "prompts"))
@pytest.mark.parametrize("heads, key_heads, width, page, dtype", [(8, 2, 128, 16, BF16), (6, 2, 96, 7, FP16), (3, 3, 64, 64, BF16), (5, 1, 256, 1, FP16)])
def test_definition(attention, config, lengths, heads, key_heads, width, page, dtype):
    b = Batch(lengths, heads, key_heads, width, page, dtype, seed=len(lengths))
    out, lse = attention.paged_attention(b.q, *b.where, return_lse=True, config=config)
    b.check(out, lse)
    assert same_bits(out, attention.paged_attention(b.q, *b.where, config=config))  # (without lse the kernels take other branches)


@pytest.mark.parametrize("heads, key_heads, width, page", [(32, 1, 128, 100), (2, 2, 8, 5), (20, 4, 80, 16), (7, 1, 136, 24), (9, 3, 40, 33), (4, 4, 200, 48), (17, 1, 64, 16)])
@pytest.mark.parametrize("dtype", (BF16, FP16))
def test_head_layouts(attention, heads, key_heads, width, page, dtype):
    b = Batch([(3, 200), (1, 1), (18, 18), (1, 333)], heads, key_heads, width, page, dtype, seed=width)
    for config in CONFIGS:
        out, lse = attention.paged_attention(b.q, *b.where, return_lse=True, config=config)
        b.check(out, lse)


@pytest.mark.parametrize("causal, window", [(False, None), (True, 1), (True, 2), (True, 63), (True, 64), (True, 300), (True, 10**6)])
@pytest.mark.parametrize("width", (128, 64))
def test_masks(attention, causal, window, width):
    b = Batch([(1, 700), (50, 400), (200, 200), (3, 2), (1, 5000)], 6, 3, width, 16, BF16, seed=3)
    first = None
    for config in ("auto", *CONFIGS):
        out, lse = attention.paged_attention(b.q, *b.where, causal=causal, window=window, return_lse=True, config=config)
        b.check(out, lse, causal=causal, window=window)
        first = (out, lse) if first is None else first
        assert same_bits(out, first[0]) and same_bits(lse, first[1])


def test_long_contexts_of_every_run_length(attention):
    b = Batch([(1, 140001), (2, 70000), (3, 20000)], 4, 1, 64, 256, BF16, seed=9)
    first = None
    for config in ("auto", *CONFIGS):
        out, lse = attention.paged_attention(b.q, *b.where, return_lse=True, config=config)
        if first is None:
            b.check(out, lse)
            first = (out, lse)
        assert same_bits(out, first[0]) and same_bits(lse, first[1])


@pytest.mark.parametrize("heads, key_heads, width, dtype", [(8, 2, 128, BF16), (3, 1, 64, FP16), (2, 2, 256, BF16)])
@pytest.mark.parametrize("window", (None, 100))
def test_a_rows_bits_do_not_depend_on_its_chunk_or_batch(attention, heads, key_heads, width, dtype, window):
    length = 900
    whole = Batch([(length, length)], heads, key_heads, width, 16, dtype, seed=4)
    want, want_lse = attention.paged_attention(whole.q, *whole.where, window=window, return_lse=True, config="rows256")
    for config in CONFIGS:
        out, lse = attention.paged_attention(whole.q, *whole.where, window=window, return_lse=True, config=config)
        assert same_bits(out, want) and same_bits(lse, want_lse), config

    def contexts(n, c):
        return torch.tensor([c], device=DEV, dtype=torch.int32), torch.tensor([0, n], device=DEV, dtype=torch.int32)

    for chunk in (1, 37, 256):  # the cache holds what comes later, which a chunk does not see
        at = 0
        while at < length:
            n = min(chunk, length - at)
            out = attention.paged_attention(whole.q[at : at + n], whole.keys, whole.values, whole.table, *contexts(n, at + n), window=window)
            assert same_bits(out, want[at : at + n]), (chunk, at)
            at += n if chunk > 1 else 13
    # the same sequence next to others, in pages of another size
    other = Batch([(3, 77), (length, length), (0, 9), (64, 500)], heads, key_heads, width, 33, dtype, seed=5)
    place = torch.arange(length, device=DEV)
    pages = other.table[1].long()[place // 33]
    other.keys[pages, place % 33], other.values[pages, place % 33] = whole.k[0], whole.v[0]
    other.q[3 : 3 + length] = whole.q
    out = attention.paged_attention(other.q, *other.where, window=window)
    assert same_bits(out[3 : 3 + length], want)


@pytest.mark.parametrize("config", ("auto", *CONFIGS))
@pytest.mark.parametrize("dtype, width, page_size", [(BF16, 128, 16), (FP16, 64, 16), (BF16, 256, 16), (FP16, 128, 7), (BF16, 96, 1)])
def test_what_a_row_does_not_see_does_not_reach_it(attention, config, dtype, width, page_size):
    lengths = [(40, 100), (1, 50), (130, 300)]
    inf, nan = float("inf"), float("nan")
    for window in (None, 20):
        clean = Batch(lengths, 4, 2, width, page_size, dtype, seed=6)
        want, want_lse = attention.paged_attention(clean.q, *clean.where, window=window, return_lse=True, config=config)
        b = Batch(lengths, 4, 2, width, page_size, dtype, seed=6)
        # keys and values at the places of some of the new tokens, and of the context
        for i, p, key, value in ((0, 80, nan, nan), (0, 85, 1.0, inf), (0, 95, inf, -inf), (2, 170, nan, 1.0), (2, 201, 1.0, -inf), (2, 260, 1.0, nan), (2, 262, 1.0, inf)):
            page, row = int(b.table[i, p // page_size]), p % page_size
            if key != 1.0:
                b.keys[page, row, :, 3] = key
            if value != 1.0:
                b.values[page, row, :, 5] = value
        out, lse = attention.paged_attention(b.q, *b.where, window=window, return_lse=True, config=config)
        for i, first, start, affected in ((0, 0, 60, (80, 85, 95)), (2, 41, 170, (170, 201, 260, 262))):
            for t in range(lengths[i][0]):
                p = start + t
                seen = [x for x in affected if x <= p and (window is None or x > p - window)]
                row = first + t
                if not seen:
                    assert same_bits(out[row], want[row]) and same_bits(lse[row], want_lse[row]), (window, i, p)
                    continue
                values_only = all(x in (85, 201, 260, 262) for x in seen)
                if values_only:  # one element of the output takes it, the others and the logarithm are as they were
                    keep = [e for e in range(width) if e != 5]
                    assert same_bits(out[row][:, keep], want[row][:, keep]) and same_bits(lse[row], want_lse[row]), (window, i, p)
                    special = {85: inf, 201: -inf, 260: nan, 262: inf}
                    total = sum(special[x] for x in seen)
                    element = out[row][:, 5].float()
                    assert bool((element.isnan() if total != total else element == total).all()), (window, i, p, element)
                else:
                    assert bool(out[row][:, 5].isnan().all())


def test_missing_pages(attention):
    for config in ("auto", *CONFIGS):
        b = Batch([(1, 100), (90, 200), (1, 300)], 4, 2, 128, 16, BF16, seed=7)
        want = attention.paged_attention(b.q, *b.where, config=config)
        b.table[1, 9] = b.keys.size(0)  # positions 144 ... 159
        b.table[2, 0] = -1
        out, lse = attention.paged_attention(b.q, *b.where, return_lse=True, config=config)
        assert same_bits(out[:1], want[:1]) and same_bits(out[1 : 1 + 34], want[1 : 1 + 34])  # positions 110 ... 143
        assert bool(out[35:].isnan().all()) and bool(lse[35:].isnan().all())
        # a context that is longer than the table
        b = Batch([(70, 160)], 4, 2, 128, 16, BF16, seed=7)
        want = attention.paged_attention(b.q, *b.where, config=config)
        out = attention.paged_attention(b.q, b.keys, b.values, b.table[:, :8], b.contexts, b.starts, config=config)
        assert same_bits(out[:38], want[:38]) and bool(out[38:].isnan().all())  # positions 90 ... 127, and those behind
        b.contexts.fill_(2**31 - 1)
        assert bool(attention.paged_attention(b.q, *b.where, config=config).isnan().all())
        b.contexts.fill_(-5)
        out, lse = attention.paged_attention(b.q, *b.where, return_lse=True, config=config)
        assert not bool(out.any()) and bool((lse == float("-inf")).all())


@pytest.mark.parametrize("order", ("heads", "pairs"))
def test_orders_in_memory(attention, order):
    lengths = [(1, 77), (20, 200)]
    a, b = (Batch(lengths, 4, 2, 64, 16, BF16, seed=8, order=o) for o in ("rows", order))
    want = attention.paged_attention(a.q, *a.where)
    assert same_bits(attention.paged_attention(b.q, *b.where), want)
    # queries as parts of a packed projection, unaligned, by head, and repeated; a table with a stride; an output inside of another
    wide = torch.zeros((21, 9, 64), device=DEV, dtype=BF16)
    wide[:, 3:7] = a.q
    assert same_bits(attention.paged_attention(wide[:, 3:7], *a.where), want)
    odd = torch.zeros(21 * 4 * 64 + 1, device=DEV, dtype=BF16)[1:].view(21, 4, 64)
    odd.copy_(a.q)
    assert same_bits(attention.paged_attention(odd, *a.where), want)
    assert same_bits(attention.paged_attention(a.q.transpose(0, 1).contiguous().transpose(0, 1), *a.where), want)
    one = a.q[:1, :1].expand(21, 4, 64)
    assert same_bits(attention.paged_attention(one, *a.where), attention.paged_attention(one.contiguous(), *a.where))
    table = torch.full((2, 2 * a.table.size(1)), 10**6, device=DEV, dtype=torch.int32)
    table[:, ::2] = a.table
    assert same_bits(attention.paged_attention(a.q, a.keys, a.values, table[:, ::2], a.contexts, a.starts), want)
    big = torch.full((21, 10, 64), 5.0, device=DEV, dtype=BF16)
    got = attention.paged_attention(a.q, *a.where, out=big[:, 2:6])
    assert got.data_ptr() == big[:, 2:6].data_ptr() and same_bits(big[:, 2:6], want)
    assert bool((big[:, :2] == 5).all()) and bool((big[:, 6:] == 5).all())


@pytest.mark.parametrize("config", ("auto", *CONFIGS))
def test_rows_behind_the_last_sequence(attention, config):
    b = Batch([(3, 40), (60, 80)], 4, 2, 128, 16, BF16, seed=10, behind=300)
    out, lse = attention.paged_attention(b.q, *b.where, return_lse=True, config=config)
    b.check(out, lse)
    assert not bool(out[63:].any()) and bool((lse[63:] == float("-inf")).all())
    kept = torch.full_like(out, 7.0)
    attention.paged_attention(b.q, *b.where, out=kept, config=config)
    assert same_bits(kept[:63], out[:63]) and bool((kept[63:] == 7).all())
    b.starts += 5  # nor are there sequences for the first five
    out = attention.paged_attention(b.q, *b.where, config=config)
    assert not bool(out[:5].any()) and not bool(out[68:].any()) and bool(out[5:68].any(-1).all())


def test_no_tokens_and_no_sequences(attention):
    b = Batch([(0, 40), (0, 0)], 4, 2, 128, 16, BF16)
    assert attention.paged_attention(b.q, *b.where).shape == (0, 4, 128)
    empty = torch.empty((0, 3), device=DEV, dtype=torch.int32)
    q = torch.ones((3, 4, 128), device=DEV, dtype=BF16)
    out, lse = attention.paged_attention(q, b.keys, b.values, empty, b.contexts[:0], b.starts[:1], return_lse=True)
    assert not bool(out.any()) and bool((lse == float("-inf")).all())
    none = torch.empty((2, 0), device=DEV, dtype=torch.int32)  # contexts without a page
    out = attention.paged_attention(q, b.keys, b.values, none, b.contexts, torch.tensor([0, 2, 3], device=DEV, dtype=torch.int32))
    assert bool(out[:2].isnan().all()) and not bool(out[2].any())


def test_scores_at_the_ends_of_their_range(attention):
    b = Batch([(1, 300), (60, 60)], 4, 2, 128, 16, BF16, seed=11, q_scale=200.0)  # one key takes nearly all
    out, lse = attention.paged_attention(b.q, *b.where, return_lse=True)
    b.check(out, lse)
    for scale in (1e-6, 0.5, 3.0):
        small = Batch([(1, 300), (60, 60)], 4, 2, 128, 16, BF16, seed=11, q_scale=0.5)
        out, lse = attention.paged_attention(small.q, *small.where, scale=scale, return_lse=True)
        small.check(out, lse, scale=scale)
    b.q.fill_(float("-inf"))
    assert bool(attention.paged_attention(b.q, *b.where).isnan().all())


def test_captured_and_replayed_with_other_lengths(attention):
    b = Batch([(1, 700), (1, 33), (1, 260)], 8, 2, 128, 16, BF16, seed=12)
    out = torch.empty_like(b.q)
    attention.paged_attention(b.q, *b.where, out=out)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        attention.paged_attention(b.q, *b.where, out=out)
    for lengths in ((700, 33, 260), (699, 1, 64), (512, 20, 257)):
        b.contexts.copy_(torch.tensor(lengths, dtype=torch.int32))
        want = attention.paged_attention(b.q, *b.where)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same_bits(out, want)


def test_another_stream_and_two_at_once(attention):
    b, c = (Batch([(1, 3000), (1, 2000)], 8, 2, 128, 16, BF16, seed=s) for s in (13, 14))
    want = [attention.paged_attention(x.q, *x.where) for x in (b, c)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, (x, s) in enumerate(zip((b, c), streams)):
            with torch.cuda.stream(s):
                got[i] = attention.paged_attention(x.q, *x.where)
    torch.cuda.synchronize()
    assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])


def test_a_cache_behind_2_31_elements(attention):
    pages, page, key_heads, width = 1100000, 16, 1, 128  # 2.25e9 elements, 4.5 GB
    keys = torch.empty((pages, page, key_heads, width), device=DEV, dtype=BF16)
    values = torch.empty_like(keys)
    small = Batch([(2, 100), (30, 30)], 4, key_heads, width, page, BF16, seed=15)
    far = pages - small.keys.size(0)
    keys[far:], values[far:] = small.keys, small.values
    for config in CONFIGS:
        want = attention.paged_attention(small.q, *small.where, config=config)
        got = attention.paged_attention(small.q, keys, values, small.table + far, small.contexts, small.starts, config=config)
        assert same_bits(got, want)


def test_many_sequences(attention):
    lengths = [(1 + i % 3, 3 + i % 70) for i in range(1500)] + [(0, 5)] * 40 + [(2, 9)]
    b = Batch(lengths, 2, 1, 64, 16, BF16, seed=16)
    want = None
    for config in ("auto", *CONFIGS):
        out = attention.paged_attention(b.q, *b.where, config=config)
        want = out if want is None else want
        assert same_bits(out, want)
    b.check(want)


def test_from_several_threads(attention):
    batches = [Batch([(1, 3000 + 100 * s), (5, 2000), (300, 900)], 8, 2, 128, 16, BF16, seed=s) for s in range(4)]
    want = [attention.paged_attention(b.q, *b.where) for b in batches]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            wrong.extend(i for _ in range(20) if not same_bits(attention.paged_attention(batches[i].q, *batches[i].where), want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_two_graphs_of_one_pool(attention):
    batches = [Batch([(1, 3000), (5, 2000 + 300 * s)], 8, 2, 128, 16, BF16, seed=s) for s in range(2)]
    want = [attention.paged_attention(b.q, *b.where) for b in batches]
    graphs, outs, pool = [torch.cuda.CUDAGraph() for _ in range(2)], [], torch.cuda.graph_pool_handle()
    for b, graph in zip(batches, graphs):
        with torch.cuda.graph(graph, pool=pool):
            outs.append(attention.paged_attention(b.q, *b.where))
    for _ in range(3):
        for i, graph in enumerate(graphs):
            graph.replay()
            torch.cuda.synchronize()
            assert same_bits(outs[i], want[i])
            assert same_bits(attention.paged_attention(batches[i].q, *batches[i].where), want[i])


def test_views_and_repeated_memory(attention):
    b = Batch([(1, 3000), (5, 2000)], 8, 2, 128, 16, BF16, seed=3)
    want = attention.paged_attention(b.q, *b.where)
    repeated = b.q[:1].expand(6, 8, 128)
    assert same_bits(attention.paged_attention(repeated, *b.where), attention.paged_attention(repeated.contiguous(), *b.where))
    wide = torch.zeros((6, 8, 160), device=DEV, dtype=BF16)
    wide[..., 16:144] = b.q
    assert same_bits(attention.paged_attention(wide[..., 16:144], *b.where), want)
    wide[..., 1:129] = b.q  # rows that do not start on 16 bytes
    assert same_bits(attention.paged_attention(wide[..., 1:129], *b.where), want)
    with torch.inference_mode():
        assert same_bits(attention.paged_attention(b.q * 1, *b.where), want)
    with pytest.raises(ValueError, match="memory of its own"):
        attention.paged_attention(b.q, *b.where, out=torch.empty((1, 8, 128), device=DEV, dtype=BF16).expand(6, 8, 128))
    b.table[0, 1] = b.table[0, 0]  # a page twice
    assert same_bits(attention.paged_attention(b.q, *b.where), attention.paged_attention(b.q, *b.where, config="rows128"))


def test_windows_beyond_32_bits(attention):
    b = Batch([(3, 300), (40, 129)], 4, 2, 64, 16, BF16, seed=5)
    want = attention.paged_attention(b.q, *b.where)
    for window in (2**31 - 1, 2**31, 2**32 + 5):
        assert same_bits(attention.paged_attention(b.q, *b.where, window=window), want)
