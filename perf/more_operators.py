"""Operators around attention, each in its plain form and as the framework's own call.

Kinds:

``rotary``        rotation of queries and keys by their positions (``rotary_embedding``): pairs side by side or half a head
                  apart, the whole head or its first part
``rotary_train``  the same with the gradients of queries and keys
``append``        new keys and values into a paged cache, keys and queries rotated on the way (``paged_append``)
``attention``     attention of new tokens over a paged cache that holds them already (``paged_attention``): single tokens, a few
                  that are verified together, chunks of a prompt and whole prompts, with grouped heads, windows and ragged batches

The plain forms compute in 32 bits (angles in 64) and round once; ``exact`` computes the definitions in 64.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

# (query heads, key heads, width of a head): the layer of the other workloads, its shards of 4 and 8, and other groupings
_HEADS = [(32, 8, 128), (8, 2, 128), (4, 1, 128), (16, 16, 64), (64, 8, 128), (9, 3, 96), (8, 1, 256), (20, 4, 80)]


def listed():
    return [
        # one token of one sequence: latency counts
        {"name": "rotary_1_token", "kind": "rotary", "tokens": 1, "heads": 32, "key_heads": 8, "width": 128, "part": 128, "pairs": False, "dtype": "bf16", "start": 1023, "factor": 1.0},
        # positions far out, in 32 bits, part of a head, pairs side by side
        {"name": "rotary_2047_tokens_part", "kind": "rotary", "tokens": 2047, "heads": 16, "key_heads": 2, "width": 80, "part": 20, "pairs": True, "dtype": "fp32", "start": 1000000, "factor": 4.0},
        # a packed training batch, both ways
        {"name": "rotary_train_8192_tokens", "kind": "rotary_train", "tokens": 8192, "heads": 32, "key_heads": 8, "width": 128, "part": 128, "pairs": False, "dtype": "bf16", "start": 0, "factor": 1.0},
        # a decode step of 64 rollouts
        {"name": "append_64_tokens", "kind": "append", "sequences": 64, "new": 1, "context": 1024, "ragged": True, "heads": 32, "key_heads": 8, "width": 128, "part": 128, "pairs": False, "page": 16, "dtype": "bf16", "factor": 1.0},
        # chunks of three prompts, part of the head
        {"name": "append_3x1365_tokens", "kind": "append", "sequences": 3, "new": 1365, "context": 2050, "ragged": False, "heads": 32, "key_heads": 8, "width": 128, "part": 64, "pairs": True, "page": 64, "dtype": "fp16", "factor": 4.0},
        # one sequence decoding: the smallest call of attention
        {"name": "decode_1x1025", "kind": "attention", "sequences": 1, "new": 1, "context": 1025, "ragged": False, "heads": 32, "key_heads": 8, "width": 128, "page": 16, "dtype": "bf16", "causal": True, "window": 0},
        # a decode step of 64 rollouts of every length
        {"name": "decode_64x8192", "kind": "attention", "sequences": 64, "new": 1, "context": 8192, "ragged": True, "heads": 32, "key_heads": 8, "width": 128, "page": 16, "dtype": "bf16", "causal": True, "window": 0},
        # long contexts
        {"name": "decode_4x131071", "kind": "attention", "sequences": 4, "new": 1, "context": 131071, "ragged": False, "heads": 32, "key_heads": 8, "width": 128, "page": 256, "dtype": "fp16", "causal": True, "window": 0},
        # five drafted tokens each are verified, within a window
        {"name": "verify_32x5_window", "kind": "attention", "sequences": 32, "new": 5, "context": 4099, "ragged": True, "heads": 64, "key_heads": 8, "width": 128, "page": 32, "dtype": "bf16", "causal": True, "window": 1024},
        # odd sizes, every new token sees the whole context
        {"name": "whole_5x333_odd", "kind": "attention", "sequences": 5, "new": 333, "context": 701, "ragged": True, "heads": 9, "key_heads": 3, "width": 96, "page": 24, "dtype": "fp16", "causal": False, "window": 0},
        # a chunk of a long prompt
        {"name": "chunk_1000_of_65500", "kind": "attention", "sequences": 1, "new": 1000, "context": 65500, "ragged": False, "heads": 32, "key_heads": 8, "width": 128, "page": 64, "dtype": "bf16", "causal": True, "window": 0},
        # prompts of every length at once: the largest case
        {"name": "prompts_4x12000", "kind": "attention", "sequences": 4, "new": 12000, "context": 12000, "ragged": True, "heads": 32, "key_heads": 8, "width": 128, "page": 64, "dtype": "bf16", "causal": True, "window": 0},
    ]  # fmt: skip


def _log_int(rng, low, high):
    """An integer from low to high, its logarithm uniform."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary_train", "append", "attention", "attention", "attention"])
    heads, key_heads, width = rng.choice(_HEADS)
    case = {"kind": kind, "heads": heads, "key_heads": key_heads, "width": width}
    if kind in ("rotary", "rotary_train"):
        case["tokens"] = _log_int(rng, 1, 8192)
        case["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        case["start"] = rng.choice([0, 0, 5000, 1000000])
    else:
        case["sequences"] = _log_int(rng, 1, 64)
        case["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
        case["page"] = rng.choice([16, 16, 64, 256, 32, 1, 17, 24])
        case["ragged"] = rng.random() < 0.6
        most = 4096 if kind == "append" else 65536
        tokens = 1 if rng.random() < 0.4 else _log_int(rng, 1, 4096)
        case["new"] = max(1, tokens // case["sequences"])
        case["context"] = max(case["new"], _log_int(rng, 1, max(1, most // case["sequences"])))
    if kind != "attention":
        case["part"] = rng.choice([width, width, width // 2, width // 4])
        case["pairs"] = rng.random() < 0.4
        case["factor"] = rng.choice([1.0, 1.0, 4.0])
    else:
        case["causal"] = rng.random() < 0.8
        case["window"] = _log_int(rng, 1, 4096) if case["causal"] and rng.random() < 0.3 else 0
        while heads * width * sum(n * c for n, c in _lengths(case)) > 5e11:  # half of the largest listed one
            case["context"] = max(case["new"], case["context"] // 2)
            case["new"] = max(1, case["new"] - case["new"] // 4)
    return case


def _lengths(case):
    """(new tokens, context with them) of each sequence: the same for all, or of every size up to the case's, a few without new ones."""
    count, new, context = case["sequences"], case["new"], case["context"]
    if not case["ragged"]:
        return [(new, context)] * count
    both = []
    for i in range(count):
        share = ((7 * i + 3) % count + 1) / count
        c = max(1, math.ceil(context * share))
        n = min(c, new if context > 2 * new else max(1, math.ceil(new * share)))
        both.append((0 if count > 8 and i % 11 == 10 else n, c))
    return both


def _keys_read(case, n, c):
    """How many keys of a sequence any of its new tokens sees, and how many pairs of a new token and a key there are."""
    if n == 0:
        return 0, 0
    if not case["causal"]:
        return c, n * c
    window = case["window"] or c
    pairs = sum(min(p + 1, window) for p in range(c - n, c))
    return min(c, window + n - 1), pairs


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _frequencies(case):
    """Radians a position, for each pair of the rotated part: a plan that a program makes once."""
    half = case["part"] // 2
    exponents = torch.arange(half, device="cuda", dtype=torch.float64) / half
    return 1e6 ** (-exponents) / case["factor"]


def _projected(gen, tokens, heads, key_heads, width, dtype):
    """Queries, keys and values as a packed projection leaves them: parts of its rows."""
    rows = _normal(gen, tokens, (heads + 2 * key_heads) * width, dtype=dtype)
    q, k, v = rows.split([heads * width, key_heads * width, key_heads * width], dim=1)
    return q.unflatten(1, (heads, width)), k.unflatten(1, (key_heads, width)), v.unflatten(1, (key_heads, width))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    heads, key_heads, width, dtype = case["heads"], case["key_heads"], case["width"], _DTYPES[case["dtype"]]
    if case["kind"] in ("rotary", "rotary_train"):
        tokens = case["tokens"]
        q, k, _ = _projected(gen, tokens, heads, key_heads, width, dtype)
        # packed sequences of a thousand tokens each
        state["positions"] = case["start"] + torch.arange(tokens, device="cuda") % 1000
        state["frequencies"] = _frequencies(case)
        if case["kind"] == "rotary_train":
            q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
            state["g_q"] = _normal(gen, tokens, heads, width, dtype=dtype)
            state["g_k"] = _normal(gen, tokens, key_heads, width, dtype=dtype)
        state["q"], state["k"] = q, k
        return state
    lengths = _lengths(case)
    tokens = sum(n for n, _ in lengths)
    pages = [-(-c // case["page"]) for _, c in lengths]
    pool = sum(pages) + 3
    order = torch.randperm(pool, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.zeros((len(lengths), max(pages)), device="cuda", dtype=torch.int32)
    first = 0
    for i, count in enumerate(pages):
        table[i, :count] = order[first : first + count]
        first += count
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    state["lengths"] = lengths
    state["table"] = table
    state["starts"] = torch.tensor(starts, device="cuda", dtype=torch.int32)
    state["contexts"] = torch.tensor([c for _, c in lengths], device="cuda", dtype=torch.int32)
    for name in ("keys", "values"):
        state[name] = torch.randn((pool, case["page"], key_heads, width), generator=gen, device="cuda", dtype=dtype)
    if case["kind"] == "append":
        state["q"], state["k"], state["v"] = _projected(gen, tokens, heads, key_heads, width, dtype)
        state["frequencies"] = _frequencies(case)
        return state
    # what lies behind the end of a sequence in its last page was never written
    for i, (_, c) in enumerate(lengths):
        if c % case["page"]:
            last = int(order[sum(pages[: i + 1]) - 1])
            state["keys"][last, c % case["page"] :] = float("nan")
            state["values"][last, c % case["page"] :] = float("nan")
    # scores with a deviation of about two
    state["q"] = (2 * _normal(gen, tokens, heads, width)).to(dtype)
    return state


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------


def _rotated(x, positions, frequencies, pairs, sign=1.0):
    """x [tokens, heads, width] with its first 2 len(frequencies) elements rotated, in 32 bits, rounded to its type."""
    angle = positions.double()[:, None] * frequencies
    cos, sin = angle.cos().float()[:, None], sign * angle.sin().float()[:, None]
    half = frequencies.numel()
    y = x.float().clone()
    a, b = (y[..., 0 : 2 * half : 2], y[..., 1 : 2 * half : 2]) if pairs else (y[..., :half], y[..., half : 2 * half])
    new_a, new_b = a * cos - b * sin, b * cos + a * sin
    a.copy_(new_a)
    b.copy_(new_b)
    return y.to(x.dtype)


def _slots(state):
    """Positions of the new tokens, and where in the cache (as rows of all pages) each one goes."""
    tokens = torch.arange(state["q"].size(0), device="cuda")
    starts, contexts = state["starts"].long(), state["contexts"].long()
    sequence = torch.bucketize(tokens, starts[1:], right=True)
    positions = contexts[sequence] - starts[sequence + 1] + tokens
    page = state["table"].long()[sequence, positions // state["page"]]
    return positions, page * state["page"] + positions % state["page"]


def _visible(state, n, c):
    """Which keys each of the n new tokens sees, or None for all."""
    if not state["causal"]:
        return None
    behind = torch.arange(c - n, c, device="cuda")[:, None] - torch.arange(c, device="cuda")
    seen = behind >= 0
    return seen & (behind < state["window"]) if state["window"] else seen


def _attend(state, f):
    """Attention in the type f, one sequence and one key head at a time."""
    heads, key_heads, width = state["heads"], state["key_heads"], state["width"]
    group = heads // key_heads
    out = torch.empty(state["q"].shape, device="cuda", dtype=f if f == torch.float64 else state["q"].dtype)
    first = 0
    for i, (n, c) in enumerate(state["lengths"]):
        if n == 0:
            continue
        used = state["table"][i, : -(-c // state["page"])].long()
        seen = _visible(state, n, c)
        q = state["q"][first : first + n].to(f) * width**-0.5
        for h in range(key_heads):
            k = state["keys"][used, :, h].reshape(-1, width)[:c].to(f)
            v = state["values"][used, :, h].reshape(-1, width)[:c].to(f)
            rows = q[:, h * group : (h + 1) * group].reshape(n * group, width)
            s = (rows @ k.t()).view(n, group, c)
            if seen is not None:
                s.masked_fill_(~seen[:, None], float("-inf"))
            s -= s.amax(2, keepdim=True)
            s.exp_()
            total = s.sum(2, keepdim=True)
            o = (s.view(n * group, c) @ v).view(n, group, width) / total
            out[first : first + n, h * group : (h + 1) * group] = o.to(out.dtype)
            del s
        first += n
    return out


def _plain(state):
    kind = state["kind"]
    if kind == "attention":
        return {"out": _attend(state, torch.float32)}
    with torch.no_grad():
        if kind == "append":
            positions, slots = _slots(state)
            state["keys"].flatten(0, 1)[slots] = _rotated(state["k"], positions, state["frequencies"], state["pairs"])
            state["values"].flatten(0, 1)[slots] = state["v"]
            q = _rotated(state["q"], positions, state["frequencies"], state["pairs"])
            return {"q": q, "keys": state["keys"], "values": state["values"]}
        how = (state["positions"], state["frequencies"], state["pairs"])
        out = {name: _rotated(state[name], *how) for name in ("q", "k")}
        if kind == "rotary_train":
            out |= {"d_" + name: _rotated(state["g_" + name], *how, sign=-1.0) for name in ("q", "k")}
        return out


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------


def _framework():
    package = os.path.join(os.getcwd(), "rl-kernel_amd")
    if package not in sys.path:
        sys.path.insert(0, package)


def _own(state):
    from rl_engine.ops.attention import paged_append, paged_attention, rotary_embedding

    kind = state["kind"]
    if kind == "attention":
        out = paged_attention(
            state["q"], state["keys"], state["values"], state["table"], state["contexts"], state["starts"],
            causal=state["causal"], window=state["window"] or None,
        )  # fmt: skip
        return {"out": out}
    if kind == "append":
        q = paged_append(
            state["k"], state["v"], state["keys"], state["values"], state["table"], state["contexts"], state["starts"],
            state["frequencies"], q=state["q"], interleaved=state["pairs"],
        )  # fmt: skip
        return {"q": q, "keys": state["keys"], "values": state["values"]}
    q, k = rotary_embedding(state["q"], state["k"], state["positions"], state["frequencies"], interleaved=state["pairs"])
    out = {"q": q, "k": k}
    if kind == "rotary_train":
        out["d_q"], out["d_k"] = torch.autograd.grad([q, k], [state["q"], state["k"]], [state["g_q"], state["g_k"]])
    return out


def run(state):
    if own:
        _framework()
        return _own(state)
    return _plain(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    heads, key_heads, width, size = case["heads"], case["key_heads"], case["width"], _BYTES[case["dtype"]]
    if case["kind"] in ("rotary", "rotary_train"):
        tokens = case["tokens"]
        ways = 2 if case["kind"] == "rotary_train" else 1
        rows = tokens * (heads + key_heads)
        return {"bytes": ways * 2 * rows * width * size + 8 * tokens, "flops": ways * 3 * rows * case["part"]}
    lengths = _lengths(case)
    tokens = sum(n for n, _ in lengths)
    if case["kind"] == "append":
        return {"bytes": 2 * tokens * (heads + 2 * key_heads) * width * size, "flops": 3 * tokens * (heads + key_heads) * case["part"]}
    read, pairs = (sum(both) for both in zip(*(_keys_read(case, n, c) for n, c in lengths)))
    return {"bytes": (2 * tokens * heads + 2 * read * key_heads) * width * size, "flops": 4 * width * heads * pairs}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def _turned(x, positions, frequencies, pairs, sign=1):
    """The rotation as a product of complex numbers."""
    part = 2 * frequencies.numel()
    head, rest = x.double()[..., :part], x.double()[..., part:]
    ab = head.unflatten(-1, (-1, 2)) if pairs else head.unflatten(-1, (2, -1)).transpose(-1, -2)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), sign * torch.outer(positions.double(), frequencies))
    turned = torch.view_as_real(torch.view_as_complex(ab.contiguous()) * turn[:, None])
    turned = turned if pairs else turned.transpose(-1, -2)
    return torch.cat([turned.flatten(-2), rest], -1)


def _exact_attention(state):
    """One new token's group of heads at a time would be the definition; here all tokens of a sequence and a head at a time."""
    heads, group = state["heads"], state["heads"] // state["key_heads"]
    result = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, c) in enumerate(state["lengths"]):
        places = torch.arange(c, device="cuda")
        pages, rows = state["table"][i].long()[places // state["page"]], places % state["page"]
        for h in range(heads):
            if n == 0:
                break
            k, v = state["keys"][pages, rows, h // group].double(), state["values"][pages, rows, h // group].double()
            logits = state["q"][first : first + n, h].double() @ k.T / math.sqrt(state["width"])
            if state["causal"]:
                at = places[c - n :, None]
                hidden = places > at
                if state["window"]:
                    hidden |= places <= at - state["window"]
                logits[hidden] = -torch.inf
            result[first : first + n, h] = torch.softmax(logits, 1) @ v
        first += n
    return result


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "attention":
            return {"out": _exact_attention(state)}
        if case["kind"] == "append":
            keys, values = state["keys"].double(), state["values"].double()
            places = []
            for i, (n, c) in enumerate(state["lengths"]):
                places += [(i, p) for p in range(c - n, c)]
            sequence, positions = torch.tensor(places, device="cuda").T
            page, row = state["table"].long()[sequence, positions // case["page"]], positions % case["page"]
            keys[page, row] = _turned(state["k"], positions, state["frequencies"], case["pairs"])
            values[page, row] = state["v"].double()
            return {"q": _turned(state["q"], positions, state["frequencies"], case["pairs"]), "keys": keys, "values": values}
        how = (state["positions"], state["frequencies"], case["pairs"])
        out = {name: _turned(state[name], *how) for name in ("q", "k")}
        if case["kind"] == "rotary_train":
            out |= {"d_" + name: _turned(state["g_" + name], *how, sign=-1) for name in ("q", "k")}
        return out
