"""A paged cache of keys and values: what fills it (csrc/rotary.hip) and the attention that reads it (csrc/paged_attention.hip).

The cache is two tensors of the caller's, ``[pages, page_size, key heads, width]`` in any order in memory whose last dimension is
contiguous. ``page_table[s, i]`` is the page of positions ``i * page_size ...`` of sequence s, ``context_lengths[s]`` counts its
positions with the new tokens of the call, and those are rows ``query_starts[s] ... query_starts[s + 1]`` of the tensors of tokens: the last
ones of the context. ``query_starts`` ascend; where they do not, it is not specified which rows are computed, but nothing outside of the
tensors is touched and no cache row but a new token's written. All three are int32 tensors on the device; nothing of them is read
back, so a call can be captured into a HIP graph and replayed with other lengths.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from rl_engine import _host, _lib
from rl_engine._C import _on, _stream_handle
from rl_engine._checks import enforce, refuse_tangents
from rl_engine.backends.rocm.attention.rotary import _DTYPES, check_frequencies, check_positions, rotary_of
from rl_engine.backends.rocm.gemm.det_gemm import det_gemm_linear
from rl_engine.backends.rocm.norm.block_norm import check_block_norm, gated_residual_norm, rms_norm


def attention_contract_id() -> str:
    """Names the order of a row's sums (what its bits depend on besides its inputs)."""
    return _lib.load().rlk_attention_contract_id().decode()


def _inference_only(who: str, *tensors: Optional[Tensor]) -> None:
    refuse_tangents(who, *tensors)
    if torch.is_grad_enabled() and any(isinstance(t, Tensor) and t.requires_grad for t in tensors):
        raise RuntimeError(f"{who} has no gradient: call it under torch.no_grad(), or with tensors that require none.")


def _check_cache(key_cache: Tensor, value_cache: Tensor, page_table: Tensor, context_lengths: Tensor, query_starts: Tensor) -> None:
    both = (("key_cache", key_cache), ("value_cache", value_cache))
    for name, t in both:
        enforce([
            (isinstance(t, Tensor), TypeError, lambda: f"{name} must be a torch.Tensor, got {type(t)!r}."),
            (lambda: t.dim() == 4, ValueError, lambda: f"{name} must be [pages, page_size, key heads, width], got shape {tuple(t.shape)}."),
            (lambda: t.is_cuda, RuntimeError, lambda: f"{name} must be on a CUDA/ROCm GPU device, got '{t.device}'."),
            (lambda: t.dtype in _DTYPES, TypeError, lambda: f"{name} must be bf16, fp16 or fp32, got {t.dtype}."),
            (lambda: min(t.shape[1:]) >= 1, ValueError, lambda: f"{name} has pages, heads or rows without elements: {tuple(t.shape)}."),
            (lambda: t.stride(3) == 1 or t.size(3) == 1, ValueError, lambda: f"{name} must have contiguous rows (the last stride 1), got strides {t.stride()}."),
        ])  # fmt: skip
    device = key_cache.device
    enforce([
        (value_cache.shape == key_cache.shape, ValueError, lambda: f"value_cache must have the shape of key_cache {tuple(key_cache.shape)}, got {tuple(value_cache.shape)}."),
        (value_cache.dtype == key_cache.dtype, TypeError, lambda: f"value_cache must be {key_cache.dtype} as key_cache is, got {value_cache.dtype}."),
        (value_cache.device == device, RuntimeError, lambda: f"value_cache must be on {device}, got {value_cache.device}."),
    ])  # fmt: skip
    for name, t, dims in (("page_table", page_table, 2), ("context_lengths", context_lengths, 1), ("query_starts", query_starts, 1)):
        enforce([
            (isinstance(t, Tensor), TypeError, lambda: f"{name} must be a torch.Tensor, got {type(t)!r}."),
            (lambda: t.dtype == torch.int32, TypeError, lambda: f"{name} must be int32, got {t.dtype}."),
            (lambda: t.device == device, RuntimeError, lambda: f"{name} must be on {device}, got {t.device}."),
            (lambda: t.dim() == dims, ValueError, lambda: f"{name} must have {dims} dimension{'s' * (dims > 1)}, got shape {tuple(t.shape)}."),
        ])  # fmt: skip
    sequences = page_table.size(0)
    enforce([
        (context_lengths.size(0) == sequences, ValueError, lambda: f"context_lengths must have {sequences} elements, one for each row of page_table, got {context_lengths.size(0)}."),
        (query_starts.size(0) == sequences + 1, ValueError, lambda: f"query_starts must have {sequences + 1} elements, got {query_starts.size(0)}."),
    ])  # fmt: skip


def _check_tokens(t: Tensor, name: str, cache: Tensor, tokens: Optional[int] = None, heads: Optional[int] = None) -> Tensor:
    """``t`` as ``[tokens, heads, width]`` with contiguous heads."""
    enforce([
        (isinstance(t, Tensor), TypeError, lambda: f"{name} must be a torch.Tensor, got {type(t)!r}."),
        (lambda: t.dim() == 3 and t.size(2) == cache.size(3), ValueError, lambda: f"{name} must be [tokens, heads, {cache.size(3)}], got shape {tuple(t.shape)}."),
        (lambda: t.dtype == cache.dtype, TypeError, lambda: f"{name} must be {cache.dtype} as the cache is, got {t.dtype}."),
        (lambda: t.device == cache.device, RuntimeError, lambda: f"{name} must be on {cache.device}, got {t.device}."),
        (lambda: tokens is None or t.size(0) == tokens, ValueError, lambda: f"{name} must have {tokens} tokens, got {t.size(0)}."),
        (lambda: heads is None or t.size(1) == heads, ValueError, lambda: f"{name} must have {heads} heads as the cache has, got {t.size(1)}."),
    ])  # fmt: skip
    return t if t.stride(2) == 1 or t.size(2) == 1 else t.contiguous()


class _Cache:
    """The C description of a cache, and what it points to."""

    __slots__ = ("c", "held")

    def __init__(self, key_cache, value_cache, page_table, context_lengths, query_starts):
        table = page_table if page_table.stride(1) == 1 or page_table.size(1) <= 1 else page_table.contiguous()
        lengths, starts = context_lengths.contiguous(), query_starts.contiguous()
        self.held = (table, lengths, starts)
        self.c = _lib.PagedCache(
            key_cache.data_ptr(), value_cache.data_ptr(), table.data_ptr(), lengths.data_ptr(), starts.data_ptr(), *key_cache.stride()[:3],
            *value_cache.stride()[:3], table.stride(0), key_cache.size(0), *key_cache.shape[1:], _DTYPES[key_cache.dtype], *table.shape,
        )  # fmt: skip


def _rows(x: Tensor, y: Optional[Tensor] = None) -> _lib.HeadRows:
    out = (0, 0) if y is None else (y.stride(0), y.stride(1))
    return _lib.HeadRows(x.data_ptr(), None if y is None else y.data_ptr(), 0, x.stride(0), x.stride(1), 0, *out, x.size(1))


def paged_append(
    k: Tensor,
    v: Tensor,
    key_cache: Tensor,
    value_cache: Tensor,
    page_table: Tensor,
    context_lengths: Tensor,
    query_starts: Tensor,
    frequencies: Optional[Tensor] = None,
    *,
    q: Optional[Tensor] = None,
    positions: Optional[Tensor] = None,
    interleaved: bool = False,
    magnitude: float = 1.0,
) -> Optional[Tensor]:
    """Writes the keys and values of new tokens into their places of a paged cache, the keys turned by their positions on the way
    (``ops.attention.rotary_embedding``, the same bits), and returns ``q`` turned likewise (``None`` without one), in one launch.

    ``k`` and ``v [tokens, key heads, width]``, ``q [tokens, heads, width]`` and the caches have one type, bf16, fp16 or fp32. Without
    ``frequencies`` nothing turns. ``positions [tokens]`` (int32 or int64) are what turns the tokens, by default their places in their sequences:
    ``context_lengths[s] - (query_starts[s + 1] - query_starts[s]) + i``; where they go is always that place. Rows of the cache that no new
    token goes to are left as they are. A token whose place lies before the start, outside of the table or in a page that does not exist is not
    written; neither are tokens behind the last sequence, whose rows of the returned ``q`` are zeros. Pages that are
    written belong to one sequence (others may share the pages in front of them), and the caches share no memory with each other or within
    themselves. The caches count as written in place for autograd; they are not differentiable: arguments that require a gradient are refused.
    """
    if isinstance(k, Tensor) and k.is_cuda and not torch.compiler.is_compiling():
        done = _host.native().paged_append(  # everyday arguments, natively
            k, v, key_cache, value_cache, page_table, context_lengths, query_starts, frequencies, q, positions, interleaved, magnitude
        )
        if done is not None:
            return done[0]
    _inference_only("paged_append", k, v, q, key_cache, value_cache, frequencies)
    where = (key_cache, value_cache, page_table, context_lengths, query_starts)
    _check_cache(*where)
    heads, width, device = key_cache.size(2), key_cache.size(3), key_cache.device
    k = _check_tokens(k, "k", key_cache, heads=heads)
    tokens = k.size(0)
    v = _check_tokens(v, "v", key_cache, tokens, heads)
    if width > _lib.ROTARY_MAX_WIDTH:
        raise ValueError(f"heads of up to {_lib.ROTARY_MAX_WIDTH} elements are served, got {width}.")
    if q is not None:
        q = _check_tokens(q, "q", key_cache, tokens)
    if frequencies is not None:
        frequencies = check_frequencies(frequencies, device, width)
        if positions is not None:
            positions = check_positions(positions, (tokens,), device)
    elif positions is not None:
        raise ValueError("positions without frequencies: nothing turns.")
    args = (k, v, *where, frequencies, q, positions)
    if _host.recorded(*args):
        turned = [_append_operator(*args, bool(interleaved), float(magnitude))]
    else:
        turned = _append(*args, interleaved, float(magnitude))
        increment_version((key_cache, value_cache))  # (what a kernel has written counts as written for autograd)
    return None if q is None else turned[0]


def _append(k, v, key_cache, value_cache, page_table, context_lengths, query_starts, frequencies, q, positions, interleaved, magnitude) -> list:
    """The launch, on arguments that have been checked: ``q`` turned, if there is one."""
    cache = _Cache(key_cache, value_cache, page_table, context_lengths, query_starts)
    device = key_cache.device
    turned = [] if q is None else [torch.empty(q.shape, dtype=q.dtype, device=device)]
    rotary = None if frequencies is None else rotary_of(frequencies, positions, interleaved, magnitude)
    described = _rows(q, turned[0]) if q is not None and q.size(1) > 0 else None
    by = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
    with _on(device):
        status = _lib.load().rlk_paged_append(
            ctypes.byref(cache.c), by(rotary), by(described), by(_rows(k)), by(_rows(v)), k.size(0), _stream_handle(device)
        )
    _lib.check(status, "rlk_paged_append failed")
    return turned


@torch.library.custom_op("rl_kernel::paged_append", mutates_args={"key_cache", "value_cache"})
def _append_operator(
    k: Tensor, v: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor, context_lengths: Tensor, query_starts: Tensor,
    frequencies: Optional[Tensor], q: Optional[Tensor], positions: Optional[Tensor], interleaved: bool, magnitude: float,
) -> Tensor:  # fmt: skip
    turned = _append(k, v, key_cache, value_cache, page_table, context_lengths, query_starts, frequencies, q, positions, interleaved, magnitude)
    return turned[0] if turned else k.new_empty((0,))  # (a compiler wants tensors of an operator that writes)


@_append_operator.register_fake
def _append_operator_fake(
    k, v, key_cache, value_cache, page_table, context_lengths, query_starts, frequencies, q, positions, interleaved, magnitude
):
    return k.new_empty((0,)) if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)


def _on_16_bytes(t: Tensor) -> bool:
    return t.data_ptr() % 16 == 0 and all(stride % 8 == 0 for stride in t.stride()[:-1])


def _check_attention(key_cache: Tensor, value_cache: Tensor, heads: int, scale: float, causal: bool, window: Optional[int], config: str, recorded: bool) -> None:
    key_heads, width = key_cache.shape[2:]
    enforce([
        (key_cache.dtype in (torch.bfloat16, torch.float16), TypeError, lambda: f"attention is served in bf16 and fp16, got {key_cache.dtype}."),
        (width % 8 == 0 and width <= _lib.ATTENTION_MAX_WIDTH, ValueError, lambda: f"heads must have a multiple of 8 elements, up to {_lib.ATTENTION_MAX_WIDTH}, got {width}."),
        (heads >= 1 and heads % key_heads == 0, ValueError, lambda: f"q must have a whole number of heads for each of the {key_heads} key heads, got {heads}."),
        (lambda: recorded or (_on_16_bytes(key_cache) and _on_16_bytes(value_cache)), ValueError, "the rows of key_cache and value_cache must start on 16 bytes."),
        (0.0 < scale <= 2.3e38, ValueError, lambda: f"scale must be positive and at most 2.3e38 (finite in units of log2), got {scale}."),
        (window is None or (isinstance(window, int) and not isinstance(window, bool) and window >= 1), ValueError, lambda: f"window must be a number of positions or None, got {window!r}."),
        (window is None or causal, ValueError, "a window goes with causal=True."),
        (config in _lib.ATTENTION_CONFIGS, ValueError, lambda: f"config must be one of {tuple(_lib.ATTENTION_CONFIGS)}, got {config!r}."),
    ])  # fmt: skip


def paged_attention(
    q: Tensor,
    key_cache: Tensor,
    value_cache: Tensor,
    page_table: Tensor,
    context_lengths: Tensor,
    query_starts: Tensor,
    *,
    scale: Optional[float] = None,
    causal: bool = True,
    window: Optional[int] = None,
    out: Optional[Tensor] = None,
    return_lse: bool = False,
    config: str = "auto",
):
    """Attention of new tokens over a paged cache that holds their keys and values already (:func:`paged_append`).

    ``q [tokens, heads, width]`` and the caches are bf16 or fp16, ``width`` a multiple of 8 up to 256; head h reads key head
    ``h // (heads / key heads)``. A token at position p sees the positions up to p, with a ``window`` the last ``window`` of them; with
    ``causal=False`` the whole context. Weights are ``softmax(scale * q k)``, ``scale`` ``width**-0.5`` by default; they are rounded to the
    type of ``q`` for the product with the values (half a step each: in bf16 the result is off by 0.0022 of its 2-norm, by 0.0017 with weights of 32
    bits), everything else is held in 32 bits. A row that sees nothing is 0 and its logarithm -inf; what a row does not see does
    not reach it, be it NaN. A row that sees a missing page (outside of the table, or an entry that is no page) is NaN, its logarithm too.

    Returns ``[tokens, heads, width]`` (``out`` where given, which overlaps no other argument and counts as written in place for autograd), with
    ``return_lse`` also the fp32 natural logarithm of the sum of exponentials ``[tokens, heads]``. Rows behind the last sequence are zeros (and -inf), in a given ``out`` left as they were.

    A row's bits depend on its query and on the keys, values and positions that it sees: a prompt that comes in chunks, next to
    other sequences or token by token has the same results (:func:`attention_contract_id` names the order of the sums). ``config`` names the
    kernel that runs and never changes them. A call is sized by the width of ``page_table`` (and the window), its temporary memory too, which is
    1 GiB at most: pass ``page_table[:, :n]`` where the longest context is known. No gradient: tensors that require one are refused.
    """
    if out is None and config == "auto" and isinstance(q, Tensor) and q.is_cuda and not torch.compiler.is_compiling():
        both = _host.native().paged_attention(  # everyday arguments, natively
            q, key_cache, value_cache, page_table, context_lengths, query_starts, scale, causal, window, return_lse
        )
        if both is not None:
            return both if return_lse else both[0]
    _inference_only("paged_attention", q, key_cache, value_cache, out)
    where = (key_cache, value_cache, page_table, context_lengths, query_starts)
    _check_cache(*where)
    width, device = key_cache.size(3), key_cache.device
    q = _check_tokens(q, "q", key_cache)
    tokens, heads = q.shape[:2]
    scale = width**-0.5 if scale is None else float(scale)
    recorded = _host.recorded(q, *where, out)  # (then there need not be addresses yet)
    _check_attention(key_cache, value_cache, heads, scale, causal, window, config, recorded)
    window = 0 if window is None else min(window, 2**31 - 1)  # (no position is further out)
    given = out
    if out is None:
        out = torch.empty((tokens, heads, width), dtype=q.dtype, device=device)
    else:
        enforce([
            (isinstance(out, Tensor), TypeError, lambda: f"out must be a torch.Tensor, got {type(out)!r}."),
            (lambda: tuple(out.shape) == tuple(q.shape), ValueError, lambda: f"out must have shape {tuple(q.shape)}, got {tuple(out.shape)}."),
            (lambda: out.dtype == q.dtype, TypeError, lambda: f"out must be {q.dtype}, got {out.dtype}."),
            (lambda: out.device == device, RuntimeError, lambda: f"out must be on {device}, got {out.device}."),
            (lambda: out.stride(2) == 1 and (recorded or _on_16_bytes(out)), ValueError, "the heads of out must be contiguous and start on 16 bytes."),
            (lambda: all(n <= 1 or stride > 0 for n, stride in zip(out.shape, out.stride())), ValueError, lambda: f"out must have memory of its own for every element, got strides {out.stride()}."),
        ])  # fmt: skip
    if page_table.size(0) == 0:
        if given is None:
            out.zero_()
        lse = torch.full((tokens, heads), -math.inf, dtype=torch.float32, device=device)
    elif tokens == 0:
        lse = torch.empty((0, heads), dtype=torch.float32, device=device)
    else:
        args = (q, *where, out, scale, bool(causal), window, given is None, bool(return_lse), config)
        if recorded:
            lse = [_attention_operator(*args)]
        else:
            lse = _attend(*args)
            if given is not None:
                increment_version(out)
        lse = lse[0] if return_lse else None
    return (out, lse) if return_lse else out


def _attend(q, key_cache, value_cache, page_table, context_lengths, query_starts, out, scale, causal, window, zero_rest, with_lse, config) -> list:
    """The launches, on arguments that have been checked: the logarithms, if they are wanted."""
    cache = _Cache(key_cache, value_cache, page_table, context_lengths, query_starts)
    tokens, heads = q.shape[:2]
    device = key_cache.device
    lse = [torch.empty((tokens, heads), dtype=torch.float32, device=device)] if with_lse else []
    q = q if _on_16_bytes(q) else q.clone(memory_format=torch.contiguous_format)
    lib, how = _lib.load(), _lib.ATTENTION_CONFIGS[config]
    size = int(lib.rlk_paged_attention_workspace_bytes(ctypes.byref(cache.c), tokens, heads, window, how))
    workspace = torch.empty((size,), dtype=torch.uint8, device=device) if size else None
    with _on(device):
        status = lib.rlk_paged_attention(
            ctypes.byref(cache.c), q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
            lse[0].data_ptr() if with_lse else None, tokens, heads, scale, int(causal), window, int(zero_rest), how,
            None if workspace is None else workspace.data_ptr(), size, _stream_handle(device),
        )  # fmt: skip
    _lib.check(status, "rlk_paged_attention failed")
    return lse


@torch.library.custom_op("rl_kernel::paged_attention", mutates_args={"out"})
def _attention_operator(
    q: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor, context_lengths: Tensor, query_starts: Tensor, out: Tensor,
    scale: float, causal: bool, window: int, zero_rest: bool, with_lse: bool, config: str,
) -> Tensor:  # fmt: skip
    lse = _attend(q, key_cache, value_cache, page_table, context_lengths, query_starts, out, scale, causal, window, zero_rest, with_lse, config)
    return lse[0] if with_lse else torch.empty((0,), dtype=torch.float32, device=q.device)


@_attention_operator.register_fake
def _attention_operator_fake(
    q, key_cache, value_cache, page_table, context_lengths, query_starts, out, scale, causal, window, zero_rest, with_lse, config
):
    return torch.empty(q.shape[:2] if with_lse else (0,), dtype=torch.float32, device=q.device)


def qwen3_attention_block(
    residual: Tensor,
    normed: Tensor,
    qkv_weight: Tensor,
    o_weight: Tensor,
    key_cache: Tensor,
    value_cache: Tensor,
    page_table: Tensor,
    context_lengths: Tensor,
    query_starts: Tensor,
    frequencies: Optional[Tensor],
    next_norm_weight: Optional[Tensor] = None,
    *,
    q_norm_weight: Optional[Tensor] = None,
    k_norm_weight: Optional[Tensor] = None,
    interleaved: bool = False,
    magnitude: float = 1.0,
    scale: Optional[float] = None,
    window: Optional[int] = None,
    post_norm_weight: Optional[Tensor] = None,
    gate: Optional[Tensor] = None,
    residual_scale: float = 1.0,
    eps: float = 1e-6,
) -> tuple[Tensor, Optional[Tensor]]:
    """One attention block of a transformer, for inference: ``normed [tokens, hidden]``, the norm of the ``residual`` stream, through the
    packed projection ``qkv_weight [(heads + 2 key heads) * width, hidden]``, the norms of each query and key head (where there are weights for them),
    :func:`paged_append`, :func:`paged_attention` and ``o_weight [hidden, heads * width]``, and what stands behind it
    (``ops.norm.gated_residual_norm``). Returns the new residual stream and its norm with ``next_norm_weight``, which the FFN block
    (``ops.ffn.qwen3_ffn_block``) takes. A token's bits do not depend on what else is in the batch or on the chunk that it came in."""
    _inference_only(
        "qwen3_attention_block", residual, normed, qkv_weight, o_weight, key_cache, value_cache, frequencies, q_norm_weight, k_norm_weight, next_norm_weight,
        post_norm_weight, gate,
    )  # fmt: skip
    _check_cache(key_cache, value_cache, page_table, context_lengths, query_starts)
    key_heads, width = key_cache.shape[2:]
    enforce([
        (isinstance(qkv_weight, Tensor) and qkv_weight.dim() == 2, ValueError, "qkv_weight must be [(heads + 2 key heads) * width, hidden]."),
        (lambda: qkv_weight.size(0) % width == 0 and qkv_weight.size(0) // width > 2 * key_heads, ValueError, lambda: f"qkv_weight must have (heads + {2 * key_heads}) * {width} rows, got {qkv_weight.size(0)}."),
        (isinstance(normed, Tensor) and normed.dim() == 2, ValueError, "normed must be [tokens, hidden]."),
    ])  # fmt: skip
    # What the operators behind the append would refuse is refused here, in front of it: a call that fails leaves the caches as they were.
    heads = qkv_weight.size(0) // width - 2 * key_heads
    scale = None if scale is None else float(scale)
    enforce([
        (isinstance(o_weight, Tensor) and o_weight.dim() == 2 and o_weight.size(1) == heads * width, ValueError, lambda: f"o_weight must be [hidden, {heads * width}]."),
        (isinstance(residual, Tensor) and tuple(residual.shape) == (normed.size(0), o_weight.size(0)), ValueError, lambda: f"residual must have shape {(normed.size(0), o_weight.size(0))}."),
        (o_weight.dtype == normed.dtype == key_cache.dtype, TypeError, lambda: f"normed, o_weight and the caches must have one type, got {normed.dtype}, {o_weight.dtype} and {key_cache.dtype}."),
        (normed.device == o_weight.device == key_cache.device, RuntimeError, lambda: f"normed and o_weight must be on {key_cache.device}, got {normed.device} and {o_weight.device}."),
    ])  # fmt: skip
    like = normed if normed.shape == residual.shape else normed.new_empty((1, 1)).expand(residual.shape)
    check_block_norm(like, residual, next_norm_weight, post_norm_weight, gate, eps)
    tensors = (
        residual, normed, qkv_weight, o_weight, key_cache, value_cache, page_table, context_lengths, query_starts, frequencies, next_norm_weight,
        q_norm_weight, k_norm_weight, post_norm_weight, gate,
    )  # fmt: skip
    how = (bool(interleaved), float(magnitude), scale, window, float(residual_scale), float(eps))
    recorded = _host.recorded(*tensors)
    _check_attention(key_cache, value_cache, heads, width**-0.5 if scale is None else scale, True, window, "auto", recorded)
    if recorded:
        total, after = _block_operator(*tensors, *how)
    else:
        total, after = _block(*tensors, *how)
    return total, None if next_norm_weight is None else after


def _block(
    residual, normed, qkv_weight, o_weight, key_cache, value_cache, page_table, context_lengths, query_starts, frequencies, next_norm_weight,
    q_norm_weight, k_norm_weight, post_norm_weight, gate, interleaved, magnitude, scale, window, residual_scale, eps,
) -> tuple[Tensor, Optional[Tensor]]:  # fmt: skip
    """The block, operator by operator."""
    key_heads, width = key_cache.shape[2:]
    heads = qkv_weight.size(0) // width - 2 * key_heads
    with torch.no_grad():
        qkv = det_gemm_linear(normed, qkv_weight)
        q, k, v = (part.unflatten(1, (-1, width)) for part in qkv.split([heads * width, key_heads * width, key_heads * width], dim=1))
        if q_norm_weight is not None:
            q = rms_norm(q, q_norm_weight, eps=eps)
        if k_norm_weight is not None:
            k = rms_norm(k, k_norm_weight, eps=eps)
        where = (key_cache, value_cache, page_table, context_lengths, query_starts)
        q = paged_append(k, v, *where, frequencies, q=q, interleaved=interleaved, magnitude=magnitude)
        y = det_gemm_linear(paged_attention(q, *where, scale=scale, window=window).flatten(1), o_weight)
        return gated_residual_norm(
            y, residual, next_norm_weight, post_weight=post_norm_weight, gate=gate, residual_scale=residual_scale, eps=eps
        )


@torch.library.custom_op("rl_kernel::qwen3_attention_block", mutates_args={"key_cache", "value_cache"})
def _block_operator(
    residual: Tensor, normed: Tensor, qkv_weight: Tensor, o_weight: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor,
    context_lengths: Tensor, query_starts: Tensor, frequencies: Optional[Tensor], next_norm_weight: Optional[Tensor], q_norm_weight: Optional[Tensor],
    k_norm_weight: Optional[Tensor], post_norm_weight: Optional[Tensor], gate: Optional[Tensor], interleaved: bool, magnitude: float,
    scale: Optional[float], window: Optional[int], residual_scale: float, eps: float,
) -> Tuple[Tensor, Tensor]:  # fmt: skip
    total, after = _block(
        residual, normed, qkv_weight, o_weight, key_cache, value_cache, page_table, context_lengths, query_starts, frequencies, next_norm_weight,
        q_norm_weight, k_norm_weight, post_norm_weight, gate, interleaved, magnitude, scale, window, residual_scale, eps,
    )  # fmt: skip
    return total, normed.new_empty((0,)) if after is None else after


@_block_operator.register_fake
def _block_operator_fake(
    residual, normed, qkv_weight, o_weight, key_cache, value_cache, page_table, context_lengths, query_starts, frequencies, next_norm_weight,
    q_norm_weight, k_norm_weight, post_norm_weight, gate, interleaved, magnitude, scale, window, residual_scale, eps,
):  # fmt: skip
    after = normed.new_empty((0,)) if next_norm_weight is None else torch.empty(residual.shape, dtype=normed.dtype, device=normed.device)
    return torch.empty(residual.shape, dtype=residual.dtype, device=residual.device), after


__all__ = ["attention_contract_id", "paged_append", "paged_attention", "qwen3_attention_block"]
