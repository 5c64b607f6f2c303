"""Writes tests/golden/attention_bits.json: SHA-256 of the raw output bytes of paged attention on seeded inputs, under the id of its
contract (as contract_bits.json holds them of the other contracts). Needs an MI355X:

    python tests/golden/make_attention_bits.py [output.json]
"""

from __future__ import annotations

import json
import sys
from pathlib import Path

import torch

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent.parent
for extra in (HERE, ROOT / "rl-kernel_amd", ROOT / "tests"):
    sys.path.insert(0, str(extra))

import inputs  # noqa: E402
from make_contract_bits import _sha  # noqa: E402

BF16, FP16 = torch.bfloat16, torch.float16
# (new tokens, context) of each sequence; heads, key heads, width, page size, type, how
CASES = {
    "decode_and_chunks": ([(1, 5000), (70, 4300), (3, 20), (1, 1)], 8, 2, 128, 16, BF16, {}),
    "pages_of_7_window_300": ([(40, 900), (1, 333), (2, 5)], 6, 2, 96, 7, FP16, {"window": 300}),
    "wide_heads": ([(5, 300), (30, 30)], 4, 1, 256, 16, BF16, {}),
    "runs_of_every_length": ([(2, 70001)], 4, 1, 64, 64, FP16, {}),
    "whole_context_scaled": ([(33, 200), (1, 77)], 3, 3, 80, 24, BF16, {"causal": False, "scale": 0.25}),
}


def attention_bits() -> dict:
    from rl_engine.ops.attention import attention_contract_id, paged_attention

    out = {}
    for seed, (name, (lengths, heads, key_heads, width, page, dtype, how)) in enumerate(CASES.items()):
        counts = [-(-c // page) for _, c in lengths]
        pool = sum(counts)
        normal = lambda n, rows, scale=1.0: inputs.randn_bf16(20000 + 10 * seed + n, rows, width, scale).to(dtype).cuda()  # noqa: B023, E731
        keys, values = (normal(n, pool * page * key_heads).view(pool, page, key_heads, width) for n in (0, 1))
        tokens = sum(n for n, _ in lengths)
        q = normal(2, tokens * heads, 2.0).view(tokens, heads, width)
        table = torch.zeros((len(lengths), max(counts)), dtype=torch.int32)
        first = 0
        for i, count in enumerate(counts):  # pages in descending order
            table[i, :count] = torch.arange(pool - 1 - first, pool - 1 - first - count, -1)
            first += count
        starts = [0]
        for n, _ in lengths:
            starts.append(starts[-1] + n)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        y, lse = paged_attention(q, keys, values, table.cuda(), ints([c for _, c in lengths]), ints(starts), return_lse=True, **how)
        out[f"{name}.out"], out[f"{name}.lse"] = _sha(y), _sha(lse)
    return {attention_contract_id(): out}


if __name__ == "__main__":
    target = Path(sys.argv[1]) if len(sys.argv) > 1 else HERE / "attention_bits.json"
    target.write_text(json.dumps(attention_bits(), indent=2, sort_keys=True) + "\n")
    print(target.read_text())
