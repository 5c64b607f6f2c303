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


@pytest.mark.parametrize("heads, key_heads, width", [(32, 8, 64), (24, 3, 72), (32, 1, 64)])
@pytest.mark.parametrize("window", (None, 900))
def test_a_table_so_wide_that_the_parts_do_not_fit_at_once(attention, heads, key_heads, width, window):
    """Without a window the key heads take several launches, or, where one of them has too many parts, all runs go one after the other."""
    b = Batch([(700, 5000)], heads, key_heads, width, 16, BF16, seed=8)
    table = torch.full((1, 2**16), -1, device=DEV, dtype=torch.int32)
    table[:, : b.table.size(1)] = b.table
    want, want_lse = attention.paged_attention(b.q, *b.where, window=window, return_lse=True, config="rows128")
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    out, lse = attention.paged_attention(b.q, b.keys, b.values, table, b.contexts, b.starts, window=window, return_lse=True)
    assert same_bits(out, want) and same_bits(lse, want_lse)
    assert torch.cuda.max_memory_allocated() - held <= 2**30 + 2**26
    given = torch.zeros((700, heads + 2, width), device=DEV, dtype=BF16)
    attention.paged_attention(b.q, b.keys, b.values, table, b.contexts, b.starts, window=window, out=given[:, 1:-1])
    assert same_bits(given[:, 1:-1], want) and not bool(given[:, 0].any()) and not bool(given[:, -1].any())


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


# ---------------------------------------------------------------------------
# Tracers and compilers: what they record computes on other inputs what the call does
# ---------------------------------------------------------------------------


def _fx(f, *args):
    from torch.fx.experimental.proxy_tensor import make_fx

    return make_fx(f)(*args)


def _fx_of_shapes(f, *args):
    from torch.fx.experimental.proxy_tensor import make_fx

    return make_fx(f, tracing_mode="fake")(*args)


def _jit(f, *args):
    return torch.jit.trace(f, args, check_trace=False)


def _compiled(f, *args):
    return torch.compile(f, backend="aot_eager", fullgraph=True)


RECORDERS = pytest.mark.parametrize("record", (_fx, _fx_of_shapes, _jit, _compiled))


@RECORDERS
def test_a_recorded_rotation(attention, record):
    f, positions = attention.rotary_frequencies(32, device=DEV), torch.arange(9, device=DEV)
    run = lambda q, k, p, f: attention.rotary_embedding(q, k, p, f)  # noqa: E731
    recorded = record(run, _normal(9, 4, 48, seed=1), _normal(9, 2, 48, seed=2), positions, f)
    q, k = _normal(9, 4, 48, seed=3), _normal(9, 2, 48, seed=4)
    for got, want in zip(recorded(q, k, positions + 5, f), run(q, k, positions + 5, f)):
        assert same_bits(got, want)


@pytest.mark.parametrize("record", (_fx, _fx_of_shapes, _compiled))
def test_a_recorded_gradient_of_a_rotation(attention, record):
    f, positions = attention.rotary_frequencies(32, device=DEV), torch.arange(9, device=DEV)

    def run(q, g, positions, f):
        q = q.detach().requires_grad_()
        return torch.autograd.grad(attention.rotary_embedding(q, None, positions, f, interleaved=True)[0], q, g)[0]

    if record is _compiled:  # (a compiler takes the forward, its backward comes with it)
        rotate = torch.compile(lambda q: attention.rotary_embedding(q, None, positions, f, interleaved=True)[0], backend="aot_eager", fullgraph=True)
        q, g = _normal(9, 4, 48, seed=3).requires_grad_(), _normal(9, 4, 48, seed=4)
        assert same_bits(torch.autograd.grad(rotate(q), q, g)[0], run(q, g, positions, f))
        return
    recorded = record(run, _normal(9, 4, 48, seed=1), _normal(9, 4, 48, seed=2), positions, f)
    q, g = _normal(9, 4, 48, seed=3), _normal(9, 4, 48, seed=4)
    assert same_bits(recorded(q, g, positions, f), run(q, g, positions, f))


@RECORDERS
def test_a_recorded_append_and_attention(attention, record):
    f = attention.rotary_frequencies(64, device=DEV)

    def run(f, q, k, v, keys, values, table, contexts, starts):
        where = (keys, values, table, contexts, starts)
        q = attention.paged_append(k, v, *where, f, q=q)
        attention.paged_append(v, k, *where)  # (returns nothing: what it writes must not be dropped)
        out = torch.zeros_like(q)
        attention.paged_attention(q, *where, out=out)
        return out, *attention.paged_attention(q, *where, return_lse=True, window=20)

    def inputs(seed):
        b = Batch([(3, 20), (1, 33)], 4, 2, 64, 16, BF16, seed=seed)
        return b, (f, b.q, _normal(4, 2, 64, seed=seed + 1), _normal(4, 2, 64, seed=seed + 2), *b.where)

    recorded = record(run, *inputs(1)[1])
    b, args = inputs(10)
    got = recorded(*args)
    eager, args = inputs(10)
    for g, w in zip(got, run(*args)):
        assert same_bits(g, w)
    assert same_bits(b.keys, eager.keys) and same_bits(b.values, eager.values)


@RECORDERS
def test_a_recorded_block(attention, record):
    hidden = 128
    weights = _normal(8 * 64, hidden, seed=1), _normal(hidden, 4 * 64, seed=2)
    f, one, norm = attention.rotary_frequencies(64, device=DEV), torch.ones(64, device=DEV, dtype=BF16), torch.ones(hidden, device=DEV, dtype=BF16)

    def run(residual, normed, qkv, o, f, one, norm, *where):
        total, after = attention.qwen3_attention_block(residual, normed, qkv, o, *where, f, norm, q_norm_weight=one, window=16)
        total, none = attention.qwen3_attention_block(total, after, qkv, o, *where, None)
        assert none is None
        return total, after

    def inputs(seed):
        b = Batch([(3, 20), (1, 33)], 4, 2, 64, 16, BF16, seed=seed)
        return b, (_normal(4, hidden, seed=seed + 1), _normal(4, hidden, seed=seed + 2), *weights, f, one, norm, *b.where)

    recorded = record(run, *inputs(1)[1])
    b, args = inputs(10)
    got = recorded(*args)
    eager, args = inputs(10)
    for g, w in zip(got, run(*args)):
        assert same_bits(g, w)
    assert same_bits(b.keys, eager.keys) and same_bits(b.values, eager.values)


def test_a_profiler_and_a_mode_see_the_operators(attention):
    b, f, k = Batch([(3, 20), (1, 33)], 4, 2, 64, 16, BF16), attention.rotary_frequencies(64, device=DEV), _normal(4, 2, 64, seed=1)

    def run():
        attention.rotary_embedding(b.q, None, torch.arange(4, device=DEV), f)
        attention.paged_append(k, k, *b.where, f)
        return attention.paged_attention(b.q, *b.where)

    seen = []

    class Mode(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    want = run()
    with Mode():
        assert same_bits(run(), want)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as profile:
        run()
    names = " ".join(seen), " ".join(e.key for e in profile.key_averages())
    assert all(f"rl_kernel.{name}" in names[0] and f"rl_kernel::{name}" in names[1] for name in ("rotary_embedding", "paged_append", "paged_attention"))
    for tensors in ((b.q.as_subclass(type("Sub", (torch.Tensor,), {})), *b.where), (torch.nn.Parameter(b.q, requires_grad=False), *b.where)):
        assert same_bits(attention.paged_attention(*tensors).as_subclass(torch.Tensor), want)


def test_frequencies_that_want_a_gradient_are_refused(attention, way):
    b = Batch([(2, 40), (1, 33)], 4, 2, 64, 16, BF16, seed=5)
    k, positions = _normal(3, 2, 64, seed=6), torch.arange(3, device=DEV)
    f = attention.rotary_frequencies(64, device=DEV)
    asks = f.clone().requires_grad_()
    weights = _normal(8 * 64, 128, seed=1), _normal(128, 4 * 64, seed=2)
    x = _normal(3, 128, seed=7)
    keys = b.keys.clone()
    calls = (
        lambda f: attention.rotary_embedding(b.q, k, positions, f)[0], lambda f: attention.paged_append(k, k, *b.where, f, q=b.q),
        lambda f: attention.rotary_embedding(b.q.clone().requires_grad_(), None, positions, f)[0].detach(),
        lambda f: attention.qwen3_attention_block(x, x, *weights, *b.where, f)[0],
    )  # fmt: skip
    for call in calls:
        with pytest.raises(RuntimeError, match="gradient"):
            call(asks)
        assert same_bits(b.keys, keys)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(f, torch.ones_like(f))
        for call in calls[:2]:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual)
    with torch.no_grad():
        for call in calls:
            assert same_bits(call(asks), call(f))


def test_a_block_that_is_refused_leaves_the_caches_as_they_were(attention):
    b = Batch([(2, 40), (1, 33)], 4, 2, 64, 16, BF16, seed=5)
    keys, values = b.keys.clone(), b.values.clone()
    given = {"residual": _normal(3, 128, seed=6), "normed": _normal(3, 128, seed=7), "qkv_weight": _normal(8 * 64, 128, seed=1), "o_weight": _normal(128, 4 * 64, seed=2)}
    names = ("key_cache", "value_cache", "page_table", "context_lengths", "query_starts")
    given |= {**dict(zip(names, b.where)), "frequencies": attention.rotary_frequencies(64, device=DEV), "next_norm_weight": _normal(128, seed=3)}
    odd = torch.zeros(b.keys.numel() + 4, device=DEV, dtype=BF16)[4:].view(b.keys.shape)
    for wrong, kind in (
        ({"o_weight": given["o_weight"][:, :-64]}, ValueError), ({"o_weight": given["o_weight"].half()}, TypeError), ({"o_weight": given["o_weight"].cpu()}, RuntimeError),
        ({"residual": given["residual"][:2]}, ValueError), ({"residual": given["residual"].half()}, TypeError), ({"next_norm_weight": _normal(64, seed=3)}, ValueError),
        ({"post_norm_weight": _normal(64, seed=3)}, ValueError), ({"gate": _normal(3, 64, seed=3)}, ValueError), ({"eps": -1.0}, ValueError), ({"scale": -1.0}, ValueError),
        ({"window": 0}, ValueError), ({"window": 1.5}, ValueError), ({"qkv_weight": _normal(7 * 64, 128, seed=1), "o_weight": _normal(128, 3 * 64, seed=2)}, ValueError),
        ({"value_cache": odd}, ValueError), ({"normed": given["normed"][:, :64]}, (RuntimeError, ValueError, AssertionError)),
    ):  # fmt: skip
        with pytest.raises(kind):
            attention.qwen3_attention_block(**{**given, **wrong})
        torch.cuda.synchronize()
        assert same_bits(b.keys, keys) and same_bits(b.values, values), wrong.keys()
    before = given["residual"].clone()
    attention.qwen3_attention_block(**given, gate=_normal(3, 1, seed=3), post_norm_weight=_normal(128, seed=4), window=5)
    assert same_bits(given["residual"], before) and not same_bits(b.keys, keys)
    fp32 = {**given, "residual": given["residual"].float()}
    assert attention.qwen3_attention_block(**fp32)[0].dtype == torch.float32


def test_every_call_of_several_threads(attention):
    """What a thread raises is raised here, and all of their calls are counted."""
    from concurrent.futures import ThreadPoolExecutor

    f = attention.rotary_frequencies(128, device=DEV)
    batches = [Batch([(1, 3000 + 100 * s), (5, 2000), (300, 900)], 8, 2, 128, 16, BF16, seed=s) for s in range(4)]
    new = [_normal(306, 2, 128, seed=10 + s) for s in range(4)]

    def call(i):
        q = attention.paged_append(new[i], new[i], *batches[i].where, f, q=batches[i].q)
        return q, attention.paged_attention(q, *batches[i].where)

    want = [call(i) for i in range(4)]
    torch.cuda.synchronize()

    def work(i):
        right = 0
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = call(i)
                right += all(same_bits(g, w) for g, w in zip(got, want[i]))
        return right

    with ThreadPoolExecutor(4) as pool:
        assert [future.result() for future in [pool.submit(work, i) for i in range(4)]] == [20] * 4
