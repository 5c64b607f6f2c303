"""Paged caches with random contents, and attention over them by its definition in 64 bits."""

from __future__ import annotations

import torch

DEV = "cuda"
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


class Batch:
    """``lengths``: (new tokens, context with them) of each sequence. Places that no position lies in hold NaN."""

    def __init__(self, lengths, heads, key_heads, width, page, dtype, seed=0, q_scale=2.0, behind=0, order="rows"):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.lengths, self.heads, self.key_heads, self.width, self.page, self.dtype = lengths, heads, key_heads, width, page, dtype
        normal = lambda *shape: torch.randn(shape, generator=gen, device=DEV).to(dtype)  # noqa: E731
        counts = [-(-c // page) for _, c in lengths]
        pool = sum(counts) + 2
        perm = torch.randperm(pool, generator=gen, device=DEV, dtype=torch.int32)
        self.table = torch.full((len(lengths), max([1, *counts])), -7, device=DEV, dtype=torch.int32)
        # in memory by page, row and head, or by page, head and row, or keys and values of a row side by side
        if order == "rows":
            self.keys, self.values = (torch.full((pool, page, key_heads, width), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
        elif order == "heads":
            self.keys, self.values = (torch.full((pool, key_heads, page, width), float("nan"), device=DEV, dtype=dtype).transpose(1, 2) for _ in range(2))
        else:
            self.keys, self.values = torch.full((pool, page, key_heads, 2, width), float("nan"), device=DEV, dtype=dtype).unbind(3)
        self.k, self.v = [], []  # of every sequence, by position
        first = 0
        for i, ((_, c), count) in enumerate(zip(lengths, counts)):
            pages = perm[first : first + count]
            self.table[i, :count] = pages
            first += count
            self.k.append(normal(c, key_heads, width))
            self.v.append(normal(c, key_heads, width))
            at = torch.arange(c, device=DEV)
            self.keys[pages.long()[at // page], at % page] = self.k[-1]
            self.values[pages.long()[at // page], at % page] = self.v[-1]
        starts = [0]
        for n, _ in lengths:
            starts.append(starts[-1] + n)
        self.starts = torch.tensor(starts, device=DEV, dtype=torch.int32)
        self.contexts = torch.tensor([c for _, c in lengths], device=DEV, dtype=torch.int32)
        self.tokens = starts[-1]
        self.q = (normal(self.tokens + behind, heads, width).float() * q_scale).to(dtype)

    @property
    def where(self):
        return self.keys, self.values, self.table, self.contexts, self.starts

    def definition(self, *, scale=None, causal=True, window=None):
        """(out, what was added up to it: the weighted magnitudes, lse, the largest sum of magnitudes of a score), in 64 bits."""
        scale = self.width**-0.5 if scale is None else scale
        group = self.heads // self.key_heads
        shape = (self.tokens, self.heads, self.width)
        out, size = torch.zeros(shape, dtype=torch.float64, device=DEV), torch.zeros(shape, dtype=torch.float64, device=DEV)
        lse = torch.full(shape[:2], float("-inf"), dtype=torch.float64, device=DEV)
        most = 0.0
        first = 0
        for (n, c), keys, values in zip(self.lengths, self.k, self.v):
            at = torch.arange(c - n, c, device=DEV)[:, None]
            place = torch.arange(c, device=DEV)
            seen = place <= at if causal else torch.ones((n, c), dtype=torch.bool, device=DEV)
            if window:
                seen &= place > at - window
            for h in range(self.heads):
                if n == 0 or c == 0:
                    continue
                q, k, v = self.q[first : first + n, h].double(), keys[:, h // group].double(), values[:, h // group].double()
                s = (q @ k.t() * scale).masked_fill(~seen, float("-inf"))
                most = max(most, float((q.abs() @ k.abs().t() * scale).max()))
                some = seen.any(1)
                lse[first : first + n, h] = torch.logsumexp(s, 1)
                w = torch.where(some[:, None], torch.softmax(s, 1), 0.0)
                out[first : first + n, h], size[first : first + n, h] = w @ v, w @ v.abs()
            first += n
        return out, size, lse, most

    def bounds(self, size, want, most, causal=True):
        """How far out and lse may be off. A score is a chain of `width` products in 32 bits, scaled, subtracted from a maximum and raised: under
        width + 8 roundings of 2^-24 of the sum of its magnitudes, and the hardware's exponential an ulp of 2^-23 more; as many of its logarithm
        move a weight by that factor. Weights are rounded to the type in the sum above (half a step), both
        sums are chains of as many 32-bit additions as there are keys, with a factor for every 64 of them and two for a run. The result is rounded once.
        Weights below 2^-14 are off by up to 2^-25 each in fp16 (2^-134 in bf16), next to a sum of 1 at least: the largest belongs to a key at the maximum."""
        longest = max([1, *(c for _, c in self.lengths)])
        score = (self.width + 8) * 2.0**-24 * most + 2.0**-22
        chain = (longest + longest / 32 + 64) * 2.0**-24
        half = HALF_STEP[self.dtype]
        small = longest * 2.0**-25 * max([0.0, *(float(v.abs().max()) for v in self.v if v.numel())]) if self.dtype == torch.float16 else 0.0
        return half * want.abs() + (half + 2 * score + 2 * chain) * size * (1 + 2.0**-6) + 2.0**-24 + small, score + chain

    def check(self, got, lse=None, **how):
        want, size, want_lse, most = self.definition(**how)
        bound, lse_bound = self.bounds(size, want, most)
        off = (got[: self.tokens].double() - want).abs()
        assert bool((off <= bound).all()), float((off / bound).max())
        if lse is not None:
            empty = want_lse == float("-inf")
            assert bool((lse[: self.tokens][empty] == float("-inf")).all())
            off = (lse[: self.tokens].double() - want_lse)[~empty].abs()
            allowed = lse_bound + 2.0**-22 * want_lse[~empty].abs() + 2.0**-22
            assert bool((off <= allowed).all()), float((off / allowed).max())


def same_bits(a, b):
    kind = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))
