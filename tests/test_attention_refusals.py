"""What rotary positions, appending to a paged cache and attention over it refuse: the C entries on calls that are wrong, before
anything reaches a GPU, the entry points on CPU tensors, and (on a GPU) on tensors that do not go together."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

AT = 1 << 20  # an address that nothing reads: these calls are refused


def _refused(rlk_lib, status, words):
    text = rlk_lib.rlk_last_error().decode()
    assert status == -1 and words in text, (status, text)


def _struct(kind, defaults, kwargs):
    assert set(kwargs) <= set(defaults)
    return ctypes.byref(kind(*({**defaults, **kwargs}[name] for name, _ in kind._fields_)))


def _rotary(**kwargs):
    from rl_engine import _lib

    return _struct(_lib.Rotary, {"frequencies": AT, "positions": AT, "positions_are_64": 1, "pairs": 8, "interleaved": 0, "magnitude": 1.0}, kwargs)


def _rows(heads=2, **kwargs):
    from rl_engine import _lib

    strides = {f"{t}_{name}_stride": 64 for t in "xy" for name in ("outer", "token", "head")}
    return _struct(_lib.HeadRows, {"x": AT, "y": AT, "heads": heads, **strides}, kwargs)


def _cache(**kwargs):
    from rl_engine import _lib

    strides = {f"{t}_{name}_stride": 64 for t in ("key", "value") for name in ("page", "row", "head")}
    fields = {"keys": AT, "values": AT, "table": AT, "lengths": AT, "starts": AT, **strides, "table_row_stride": 4, "pages": 9, "page_size": 16, "key_heads": 2,
              "width": 64, "dtype": 0, "sequences": 3, "table_columns": 4}  # fmt: skip
    return _struct(_lib.PagedCache, fields, kwargs)


def test_rotary_entry(rlk_lib):
    def call(rotary=None, q=None, k=None, tokens=6, inner=6, width=64, dtype=0):
        return rlk_lib.rlk_rotary_embedding(rotary or _rotary(), q or _rows(), k, tokens, inner, width, dtype, 0, None)

    for kwargs, words in (
        ({"rotary": _rotary(pairs=33)}, "pairs"), ({"rotary": _rotary(pairs=-1)}, "pairs"), ({"rotary": _rotary(frequencies=None)}, "frequencies"),
        ({"rotary": _rotary(positions=None)}, "positions"), ({"q": _rows(x=None)}, "null operand"), ({"k": _rows(y=None)}, "null operand"),
        ({"q": _rows(heads=-1)}, "range"), ({"k": _rows(heads=70000)}, "range"), ({"tokens": -1}, "range"), ({"tokens": 2**31}, "range"), ({"width": 0}, "range"),
        ({"width": 1025}, "range"), ({"dtype": 7}, "dtype"), ({"inner": 4}, "inner"), ({"inner": 0}, "inner"), ({"inner": 12}, "inner"),
    ):  # fmt: skip
        _refused(rlk_lib, call(**kwargs), words)
    _refused(rlk_lib, rlk_lib.rlk_rotary_embedding(None, _rows(), None, 6, 6, 64, 0, 0, None), "null")
    assert call(tokens=0, q=_rows(x=None, y=None)) == 0 and call(q=_rows(heads=0, x=None)) == 0


def test_append_entry(rlk_lib):
    def call(cache=None, rotary=None, q=None, k=None, v=None, tokens=6):
        return rlk_lib.rlk_paged_append(cache or _cache(), rotary, q, k or _rows(), v or _rows(), tokens, None)

    for kwargs, words in (
        ({"cache": _cache(page_size=0)}, "range"), ({"cache": _cache(page_size=2**24 + 1)}, "range"), ({"cache": _cache(sequences=-1)}, "range"),
        ({"cache": _cache(table_columns=-1)}, "range"), ({"cache": _cache(pages=-1)}, "range"), ({"cache": _cache(pages=2**31)}, "range"),
        ({"cache": _cache(key_heads=0)}, "range"), ({"cache": _cache(width=0)}, "range"), ({"cache": _cache(starts=None)}, "null"),
        ({"cache": _cache(lengths=None)}, "null"), ({"cache": _cache(table=None)}, "null"), ({"cache": _cache(keys=None)}, "null"),
        ({"cache": _cache(value_row_stride=-64)}, "stride"), ({"cache": _cache(table_row_stride=-1)}, "stride"), ({"cache": _cache(dtype=5)}, "dtype"),
        ({"k": _rows(heads=3)}, "heads"), ({"v": _rows(heads=1)}, "heads"), ({"v": _rows(x=None)}, "null operand"), ({"q": _rows(y=None)}, "null operand"),
        ({"q": _rows(heads=0)}, "heads"), ({"rotary": _rotary(pairs=33)}, "pairs"), ({"rotary": _rotary(frequencies=None)}, "frequencies"),
        ({"tokens": -1}, "range"), ({"tokens": 2**30}, "range"),
    ):  # fmt: skip
        _refused(rlk_lib, call(**kwargs), words)
    assert call(cache=_cache(keys=None, values=None), k=_rows(x=None), tokens=0) == 0


def test_attention_entry(rlk_lib):
    def call(cache=None, q=AT, strides=(256, 64), out=AT, out_strides=(256, 64), tokens=6, heads=4, scale=0.1, causal=1, window=0, config=0, workspace=AT, size=1 << 40):
        return rlk_lib.rlk_paged_attention(
            cache or _cache(), q, *strides, out, *out_strides, None, tokens, heads, scale, causal, window, 1, config, workspace, size, None
        )

    need = int(rlk_lib.rlk_paged_attention_workspace_bytes(_cache(), 6, 4, 0, 0x101))
    assert need > 0 and rlk_lib.rlk_paged_attention_workspace_bytes(_cache(), 6, 4, 0, 3) == 0
    assert rlk_lib.rlk_paged_attention_workspace_bytes(_cache(), 6, 4, 0, 0x103) > 0
    assert rlk_lib.rlk_paged_attention_workspace_bytes(_cache(), 6, 4, -1, 0) == 0
    for kwargs, words in (
        ({"cache": _cache(dtype=2)}, "bf16 nor fp16"), ({"cache": _cache(width=60)}, "multiple of 8"), ({"cache": _cache(width=264)}, "multiple of 8"),
        ({"cache": _cache(sequences=0)}, "without a sequence"), ({"cache": _cache(keys=AT + 8)}, "16 bytes"), ({"cache": _cache(value_head_stride=4)}, "16 bytes"),
        ({"cache": _cache(key_page_stride=68)}, "16 bytes"), ({"q": AT + 2}, "16 bytes"), ({"strides": (255, 64)}, "16 bytes"), ({"out": AT + 8}, "16 bytes"),
        ({"out_strides": (256, 4)}, "16 bytes"), ({"q": None}, "null"), ({"out": None}, "null"), ({"strides": (-256, 64)}, "negative"), ({"heads": 3}, "heads"),
        ({"heads": 0}, "heads"), ({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"), ({"scale": math.nan}, "scale"), ({"scale": math.inf}, "scale"),
        ({"window": -1}, "window"), ({"window": 5, "causal": 0}, "window"), ({"config": 4}, "configuration"), ({"config": 0x104}, "configuration"),
        ({"config": 0x203}, "configuration"), ({"config": 0x100}, "configuration"), ({"config": 0x101, "workspace": None}, "workspace"), ({"config": 0x101, "workspace": AT + 8}, "workspace"),
        ({"config": 0x101, "size": need - 1}, "workspace"), ({"tokens": 2**30}, "range"), ({"tokens": -1}, "range"), ({"cache": _cache(lengths=None)}, "null"),
    ):  # fmt: skip
        _refused(rlk_lib, call(**kwargs), words)
    assert call(tokens=0, q=None, out=None, workspace=None) == 0


def test_entry_points_on_the_cpu():
    from rl_engine.ops import attention

    x = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    cache = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    where = (cache, cache, torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    f = attention.rotary_frequencies(64, device="cpu")
    for call in (
        lambda: attention.rotary_embedding(x, x, torch.arange(3), f), lambda: attention.paged_append(x, x, *where), lambda: attention.paged_attention(x, *where),
    ):  # fmt: skip
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    for args, kwargs in (
        ((3,), {}), ((0,), {}), ((True,), {}), ((64, 1.0), {}), ((64,), {"factor": 0.0}), ((64,), {"scaling": "other"}), ((2,), {"scaling": "base", "factor": 2.0}),
        ((64,), {"scaling": "bands"}), ((64,), {"scaling": "wavelengths", "original_length": 0}),
        ((64,), {"scaling": "bands", "original_length": 4096, "fast_turns": 1.0}), ((64, math.inf), {}), ((64,), {"factor": math.nan}),
    ):  # fmt: skip
        with pytest.raises(ValueError):
            attention.rotary_frequencies(*args, device="cpu", **kwargs)


@pytest.mark.gpu
def test_tensors_that_do_not_go_together():
    from rl_engine.ops import attention

    new = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    x, k = new(3, 4, 64), new(3, 2, 64)
    positions, f = torch.arange(3, device="cuda"), attention.rotary_frequencies(64)
    rotary = lambda q=x, k=k, p=positions, f=f: attention.rotary_embedding(q, k, p, f)  # noqa: E731
    for kwargs, kind, words in (
        ({"q": x.double()}, TypeError, "bf16, fp16 or fp32"), ({"k": k.half()}, TypeError, "as q is"), ({"k": k[:2]}, ValueError, "tokens"), ({"k": k[..., :32]}, ValueError, "width"),
        ({"p": positions[:2]}, ValueError, "shape"), ({"p": positions.float()}, TypeError, "int32"), ({"p": positions.cpu()}, RuntimeError, "on cuda"),
        ({"f": f.float()}, TypeError, "fp64"), ({"f": f.cpu()}, RuntimeError, "on cuda"), ({"f": torch.cat([f, f])}, ValueError, "at most 32"), ({"q": x[0]}, ValueError, "tokens"),
    ):  # fmt: skip
        with pytest.raises(kind, match=words):
            rotary(**kwargs)
    keys, values = new(5, 16, 2, 64), new(5, 16, 2, 64)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    base = {"key_cache": keys, "value_cache": values, "page_table": ints(0, 1).view(1, 2), "context_lengths": ints(3), "query_starts": ints(0, 3)}
    wrong = (
        ({"key_cache": keys[0]}, ValueError, "pages"), ({"value_cache": values[:4]}, ValueError, "shape"), ({"value_cache": values.half()}, TypeError, "as key_cache"),
        ({"key_cache": keys.transpose(2, 3).contiguous().transpose(2, 3)}, ValueError, "contiguous rows"), ({"page_table": base["page_table"].long()}, TypeError, "int32"),
        ({"page_table": ints(0, 1)}, ValueError, "dimension"), ({"context_lengths": ints(3, 3)}, ValueError, "context_lengths"), ({"query_starts": ints(0)}, ValueError, "query_starts"),
        ({"query_starts": base["query_starts"].cpu()}, RuntimeError, "on cuda"), ({"key_cache": keys.cpu()}, RuntimeError, "GPU"),
    )  # fmt: skip
    for kwargs, kind, words in wrong:
        with pytest.raises(kind, match=words):
            attention.paged_attention(x, **{**base, **kwargs})
        with pytest.raises(kind, match=words):
            attention.paged_append(k, k, **{**base, **kwargs})
    for kwargs, kind, words in (
        ({"q": x.half()}, TypeError, "as the cache"), ({"q": x[..., :32]}, ValueError, "heads, 64"), ({"q": x[:, :3]}, ValueError, "whole number"), ({"scale": 0.0}, ValueError, "scale"),
        ({"window": 0}, ValueError, "window"), ({"window": 4, "causal": False}, ValueError, "causal"), ({"window": 1.5}, ValueError, "window"), ({"config": "fast"}, ValueError, "config"),
        ({"out": x[:2]}, ValueError, "shape"), ({"out": x.half()}, TypeError, "out must be"), ({"out": new(3, 4, 128)[..., ::2]}, ValueError, "contiguous"),
        ({"q": x.clone().requires_grad_()}, RuntimeError, "no gradient"),
    ):  # fmt: skip
        with pytest.raises(kind, match=words):
            attention.paged_attention(**{"q": x, **base, **kwargs})
    odd = new(5 * 16 * 2 * 64 + 4)[4:].view(5, 16, 2, 64)
    with pytest.raises(ValueError, match="16 bytes"):
        attention.paged_attention(x, **{**base, "key_cache": odd, "value_cache": odd})
    fp32 = {**base, "key_cache": keys.float(), "value_cache": values.float()}
    with pytest.raises(TypeError, match="bf16 and fp16"):
        attention.paged_attention(x.float(), **fp32)
    narrow = new(5, 16, 2, 20)
    with pytest.raises(ValueError, match="multiple of 8"):
        attention.paged_attention(x[..., :20], **{**base, "key_cache": narrow, "value_cache": narrow})
    for kwargs, kind, words in (
        ({"k": k[:, :1]}, ValueError, "heads as the cache"), ({"v": k[:2]}, ValueError, "tokens"), ({"v": k.half()}, TypeError, "as the cache"), ({"q": x[:2]}, ValueError, "tokens"),
        ({"positions": positions}, ValueError, "without frequencies"), ({"frequencies": f, "positions": positions[:2]}, ValueError, "shape"),
        ({"frequencies": f.float()}, TypeError, "fp64"), ({"k": k.clone().requires_grad_()}, RuntimeError, "no gradient"),
    ):  # fmt: skip
        with pytest.raises(kind, match=words):
            attention.paged_append(**{"k": k, "v": k, **base, **kwargs})
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention.rotary_embedding(dual, k, positions, f)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            attention.paged_attention(dual, **base)
