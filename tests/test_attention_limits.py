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
