"""What attention asks for as a workspace: parts of the runs that a row can see, whatever the table's width (the entries answer on the
host; nothing runs on a GPU)."""

from __future__ import annotations

import pytest

from rl_engine import _lib
from test_attention_refusals import _cache

ROWS64_SPLIT, ROWS128_SPLIT, AUTO = _lib.ATTENTION_CONFIGS["rows64_split"], _lib.ATTENTION_CONFIGS["rows128_split"], 0
TILE = 64


def _run_of_position(p):
    """The run of 256 positions up to 4096, of 512 up to 16384, of 1024 up to 65536, of 2048 behind that a position is in."""
    for size, first, start, end in ((256, 0, 0, 4096), (512, 16, 4096, 16384), (1024, 40, 16384, 65536)):
        if p < end:
            return first + (p - start) // size
    return 88 + (p - 65536) // 2048


def _runs_asked_for(rlk_lib, window, columns=8192, page=16, tokens=3, heads=4, width=64, config=ROWS64_SPLIT):
    size = rlk_lib.rlk_paged_attention_workspace_bytes(
        _cache(table_columns=columns, table_row_stride=columns, page_size=page, width=width, key_row_stride=width), tokens, heads, window, config
    )
    each = tokens * heads * (width + 2) * 4
    assert size % each == 0
    return size // each


@pytest.mark.parametrize("window", (1, 2, 63, 64, 65, 66, 127, 129, 255, 256, 257, 300, 449, 450, 511, 512, 1000, 1024, 2047, 4096, 5000, 20000, 131072))
def test_a_window_has_the_runs_that_it_can_touch(rlk_lib, window):
    runs = _runs_asked_for(rlk_lib, window)
    most = max(_run_of_position(p) - _run_of_position(max(0, p - window + 1)) + 1 for p in range(0, 131072, 1))
    assert most <= runs <= most + 1, (most, runs)


def test_without_a_window_all_runs_of_the_table(rlk_lib):
    assert _runs_asked_for(rlk_lib, 0) == _run_of_position(131072) + 1  # (with the position behind the table)


@pytest.mark.parametrize(
    "sequences, tokens, heads, key_heads, width, positions, window",
    [(64, 320, 64, 8, 128, 2**20, 4096), (64, 320, 64, 8, 128, 131072, 4096), (1, 512, 32, 8, 128, 2**20, 4096), (127, 127 * 16, 32, 8, 128, 131072, 0), (1, 512, 32, 8, 128, 2**20, 0),
     (100, 800, 32, 8, 128, 2**20, 0)],
)  # fmt: skip
def test_a_wide_table_takes_no_more_than_a_gibibyte(rlk_lib, sequences, tokens, heads, key_heads, width, positions, window):
    cache = _cache(sequences=sequences, key_heads=key_heads, width=width, page_size=16, table_columns=positions // 16, table_row_stride=positions // 16,
                   key_row_stride=key_heads * width, value_row_stride=key_heads * width, key_page_stride=16 * key_heads * width,
                   value_page_stride=16 * key_heads * width, key_head_stride=width, value_head_stride=width)  # fmt: skip
    assert rlk_lib.rlk_paged_attention_workspace_bytes(cache, tokens, heads, window, AUTO) <= 2**30
