"""Calls of paged attention and appending beyond what their arithmetic holds: refused by the C entries before anything reaches a GPU."""

from __future__ import annotations

import pytest
import torch

from test_attention_refusals import AT, _cache, _refused, _rows


def _attention(rlk_lib, cache=None, strides=(256, 64), tokens=6, heads=4, scale=0.1):
    return rlk_lib.rlk_paged_attention(cache or _cache(), AT, *strides, AT, *strides, None, tokens, heads, scale, 1, 0, 1, 0, AT, 1 << 40, None)


@pytest.mark.parametrize("scale", (2.4e38, 2.9e38, 3e38))
def test_scales_that_are_infinite_in_units_of_log2(rlk_lib, scale):
    _refused(rlk_lib, _attention(rlk_lib, scale=scale), "scale")


@pytest.mark.gpu
def test_the_largest_scale():
    from rl_engine.ops import attention

    new = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    keys, values = new(1, 16, 1, 64) + 1, new(1, 16, 1, 64) + 2
    where = (keys, values, ints(0).view(1, 1), ints(7), ints(0, 3))
    out, lse = attention.paged_attention(new(3, 2, 64), *where, scale=2.3e38, return_lse=True)
    assert bool((out == 2).all()) and torch.allclose(lse, torch.tensor([5.0, 6.0, 7.0], device="cuda").log()[:, None].expand(3, 2), rtol=1e-6)
    for config in ("auto", "rows64"):
        with pytest.raises(ValueError, match="scale"):
            attention.paged_attention(new(3, 2, 64), *where, scale=2.4e38, config=config)


def test_rows_whose_numbers_do_not_fit(rlk_lib):
    """A row tile's first number and the next tile's are 32-bit numbers: two tiles of 256 rows above the last row must still fit."""
    one = lambda: _cache(key_heads=1, width=8, key_row_stride=8)  # noqa: E731
    for tokens, heads in ((2**31 - 1000, 1), (2**30 - 500, 2), (2**31 - 2, 1)):
        _refused(rlk_lib, _attention(rlk_lib, cache=one(), strides=(8, 8), tokens=tokens, heads=heads), "range")
        assert rlk_lib.rlk_paged_attention_workspace_bytes(one(), tokens, heads, 0, 0x101) == 0


def test_appending_to_memory_that_elements_share(rlk_lib):
    call = lambda **kwargs: rlk_lib.rlk_paged_append(_cache(values=AT << 1, **kwargs), None, None, _rows(), _rows(), 6, None)  # noqa: E731
    for kwargs in ({"key_page_stride": 0}, {"key_row_stride": 0}, {"key_head_stride": 0}, {"value_page_stride": 0}, {"value_row_stride": 0}, {"value_head_stride": 0}):
        _refused(rlk_lib, call(**kwargs), "memory of its own")
    _refused(rlk_lib, rlk_lib.rlk_paged_append(_cache(), None, None, _rows(), _rows(), 6, None), "memory of its own")


@pytest.mark.gpu
def test_appending_to_an_expanded_cache():
    from rl_engine.ops import attention

    new = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    k, behind = new(3, 2, 64), (ints(0, 1).view(1, 2), ints(20), ints(0, 3))
    for keys, values in ((new(1, 16, 2, 64).expand(5, 16, 2, 64), new(5, 16, 2, 64)), (new(5, 16, 2, 64), new(5, 16, 1, 64).expand(5, 16, 2, 64)), (new(5, 16, 2, 64),) * 2):
        with pytest.raises(ValueError, match="memory of its own"):
            attention.paged_append(k, k, keys, values, *behind)
    one = new(1, 16, 1, 64)  # a single page and head may have any strides
    attention.paged_append(k[:, :1], k[:, :1], one.as_strided((1, 16, 1, 64), (0, 64, 0, 1)), torch.zeros_like(one), ints(0).view(1, 1), ints(3), ints(0, 3))
