"""Scores of given tokens on gfx950: log-probability, log-sum-exp, entropy and the most likely alternatives.

What :mod:`.vocab_parallel_logp` and :mod:`.linear_logp` answer with ``(logp, lse)``, with the statistics that a policy update
and a sampler ask for next to them, from the same pass over the logits, and differentiable in all of them: an entropy bonus is
``scores.entropy``, a loss on alternatives ``scores.top_logp``. ``logp`` and ``lse`` carry the bits of those entries (of
:func:`~.vocab_parallel_logp.hip_deterministic_logp_from_logits` with its 64 tiles, wherever they divide the vocabulary) but for two
kinds of rows: one with a NaN logit, or one of ``+inf``, is NaN throughout; and where ``|lse|`` is 65536 or more, a row masked
throughout with a finite value, log-probabilities are taken from the row's maximum, as ``lse`` has lost the logarithm of the sum.

Results of a row never depend on the rest of the batch. Nothing is read back from the device unless ``validate`` asks for it,
so a call can be captured in a HIP graph.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from rl_engine import _C, _host, _lib
from rl_engine._checks import enforce, refuse_tangents, without_second_derivative
from rl_engine.backends.rocm.logprob.linear_logp import _logits_to_save, _prepare, _requires_grad

# Logits that nobody keeps go through a buffer of at most this size, whole rows of tiles of 256 tokens at a time: 3328 tokens of
# a vocabulary of 151936.
_LOGITS_BUFFER_BYTES = 2 << 30
_CHUNK_TOKENS = 256


class TokenScores(NamedTuple):
    """fp32 ``logp``, ``lse`` and ``entropy`` in the shape of the target ids; ``top_logp`` and int64 ``top_ids`` with a last
    dimension of ``top_k`` (``None`` for ``top_k=0``): the columns with the largest logits, the largest first, equal ones from the
    lowest id on."""

    logp: torch.Tensor
    lse: torch.Tensor
    entropy: torch.Tensor
    top_logp: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def _checked_top_k(top_k: int, real: int) -> int:
    most = min(_lib.SCORES_MAX_TOP_K, real)
    enforce([
        (isinstance(top_k, int) and not isinstance(top_k, bool), TypeError, f"top_k must be an int, got {type(top_k)!r}"),
        (lambda: 0 <= top_k <= most, ValueError, lambda: f"top_k must be in [0, {most}], got {top_k}"),
    ])  # fmt: skip
    return top_k


def _row_temperature(temperature, rows: int, device: torch.device) -> Optional[torch.Tensor]:
    if temperature is None:
        return None
    if not isinstance(temperature, torch.Tensor):
        return torch.full((rows,), float(temperature), dtype=torch.float32, device=device)
    temp = temperature.detach().to(device=device, dtype=torch.float32).reshape(-1)
    if temp.numel() == 1:
        temp = temp.expand(rows)
    if temp.numel() != rows:
        raise ValueError("temperature must be positive and scalar or per-token")
    return temp.contiguous()


def _validate_values(target_1d: torch.Tensor, temp: Optional[torch.Tensor], real: int) -> None:
    bad_id, bad_temperature = _C.RowChecks(target_1d, 0, real, temp).results()
    if bad_id:
        raise ValueError(f"target_ids must be in the real vocabulary [0, {real})")
    if bad_temperature:
        raise ValueError("temperature must be positive and scalar or per-token")


def _shaped(scores, shape: torch.Size) -> TokenScores:
    logp, lse, entropy, top_logp, top_ids = scores
    if len(shape) != 1:
        logp, lse, entropy = logp.reshape(shape), lse.reshape(shape), entropy.reshape(shape)
        if top_logp is not None:
            top_logp, top_ids = top_logp.reshape(*shape, top_logp.size(-1)), top_ids.reshape(*shape, top_ids.size(-1))
    return TokenScores(logp, lse, entropy, top_logp, top_ids)


# ---------------------------------------------------------------------------
# From logits
# ---------------------------------------------------------------------------


def scores_gradient(logits, target_1d, temp, lse, entropy, top_ids, real, g_logp, g_lse, g_entropy, g_top) -> torch.Tensor:
    """d(logits) of the scores of ``logits [rows, V]``, from the forward's answers and the gradients of its outputs (or ``None``)."""
    grads = (g_logp, g_lse, g_entropy, g_top)
    refuse_tangents("the gradient of token scores", *grads)
    _host.refuse_capture_into_another_graph()
    with torch.no_grad():
        grad = _C.logits_scores_backward(logits, target_1d, real, lse, entropy, top_ids, grads, temperature=temp)
    return without_second_derivative([grad])[0]


class _ScoresFromLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target_1d, temp, real, top_k):
        logp, lse, entropy, top_logp, top_ids = _C.logits_scores(logits, target_1d, real, top_k, temperature=temp)
        ctx.save_for_backward(logits, target_1d, temp, lse, entropy, top_ids)
        ctx.real = real
        ctx.set_materialize_grads(False)
        if top_ids is not None:
            ctx.mark_non_differentiable(top_ids)
        return logp, lse, entropy, top_logp, top_ids

    @staticmethod
    def backward(ctx, g_logp, g_lse, g_entropy, g_top, _g_ids):
        grads = (g_logp, g_lse, g_entropy, g_top)
        if all(g is None for g in grads):
            return (None,) * 5
        return scores_gradient(*ctx.saved_tensors, ctx.real, *grads), None, None, None, None


def hip_deterministic_scores_from_logits(
    logits: torch.Tensor,
    target_ids: torch.Tensor,
    *,
    top_k: int = 0,
    temperature: float | torch.Tensor | None = None,
    real_vocab_size: Optional[int] = None,
    validate: bool = False,
) -> TokenScores:
    """:class:`TokenScores` of ``logits [..., V]`` (bf16 / fp16 / fp32) for ``target_ids [...]``; differentiable in ``logits``.

    ``temperature`` (a number, or one per row; not differentiated) divides the logits; ``real_vocab_size`` leaves out the columns behind it, whatever
    they hold. Logits of ``-inf`` are tokens that cannot be drawn: they add nothing to ``lse`` and ``entropy`` and have ``p = 0``. One that
    is named nevertheless, by its id or among the alternatives, has a log-probability of ``-inf``, whose gradient is that of any
    other: 1 for its own logit, ``-p`` for all. A row without any other has no distribution: its ``lse`` is ``-inf``, its other answers are NaN, its
    gradient is zero. A row that is NaN has a NaN gradient where one of its answers is differentiated with a factor other than 0.

    Without ``validate`` no value is read back: an id outside of the real vocabulary gives ``logp = NaN``, a temperature that is
    not positive NaN throughout. With it such a call raises ``ValueError`` (and cannot be captured into a graph). An infinite
    temperature, or one so small that its reciprocal is, gives NaN throughout as well.
    """
    if not validate and isinstance(logits, torch.Tensor) and logits.dim() == 2 and not torch.compiler.is_compiling():
        real = logits.size(1) if real_vocab_size is None else real_vocab_size
        scores = _host.native().scores(logits, target_ids, temperature, real, top_k)  # everyday arguments, natively
        if scores is not None:
            return TokenScores(*scores)
    refuse_tangents("token scores", logits)
    enforce([
        (isinstance(logits, torch.Tensor) and logits.dim() >= 2, ValueError, "logits must be a tensor [..., vocabulary] of at least two dimensions"),
        (lambda: logits.dtype in (torch.bfloat16, torch.float16, torch.float32), TypeError, lambda: f"logits must be bf16, fp16 or fp32, got {logits.dtype}"),
        (lambda: logits.is_cuda, RuntimeError, lambda: f"token scores require a GPU tensor, got device '{logits.device}'"),
        (lambda: 0 < logits.size(-1) <= _lib.SCORES_MAX_VOCAB, ValueError, lambda: f"the vocabulary must have 1 to {_lib.SCORES_MAX_VOCAB} columns"),
        (lambda: target_ids.device == logits.device, ValueError, "target_ids must share the logits device"),
        (lambda: target_ids.shape == logits.shape[:-1], ValueError, "target_ids must have one id per logits row"),
    ])  # fmt: skip
    vocab = logits.size(-1)
    real = vocab if real_vocab_size is None else int(real_vocab_size)
    if not 0 < real <= vocab:
        raise ValueError(f"real_vocab_size must be in [1, {vocab}], got {real_vocab_size}")
    top_k = _checked_top_k(top_k, real)
    logits_2d = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
    rows = logits_2d.size(0)
    target_1d = target_ids.reshape(-1).to(dtype=torch.long).contiguous()
    temp = _row_temperature(temperature, rows, logits.device)
    if validate and rows:
        _validate_values(target_1d, temp, real)
    if _requires_grad(logits_2d):
        scores = _ScoresFromLogits.apply(logits_2d, target_1d, temp, real, top_k)
    else:
        scores = _C.logits_scores(logits_2d.detach(), target_1d, real, top_k, temperature=temp)
    return _shaped(scores, target_ids.shape)


# ---------------------------------------------------------------------------
# From hidden states
# ---------------------------------------------------------------------------


def _token_chunks(tokens: int, vocab: int):
    """Row ranges whose fp32 logits fit the buffer, whole token tiles where it takes one (a single row always)."""
    rows = max(_LOGITS_BUFFER_BYTES // (4 * _C.linear_logp_logits_row_stride(vocab)), 1)
    step = rows // _CHUNK_TOKENS * _CHUNK_TOKENS or rows
    return [(first, min(first + step, tokens)) for first in range(0, tokens, step)]


def _buffer(rows: int, vocab: int, device) -> torch.Tensor:
    return torch.empty((rows, _C.linear_logp_logits_row_stride(vocab)), dtype=torch.float32, device=device)


def _rows(t: Optional[torch.Tensor], first: int, end: int) -> Optional[torch.Tensor]:
    return None if t is None else t[first:end]


def _linear_scores(hidden, weight, bias, target, temp, real, top_k, kept):
    """The answers, through ``kept`` (all logits, left in it), through a buffer of some rows' logits, or through none."""
    tokens, vocab = hidden.size(0), weight.size(0)
    if kept is not None or tokens == 0 or not _C.linear_scores_needs_logits(hidden, weight, bias, top_k):
        return _C.linear_scores(hidden, weight, target, bias, temp, real, top_k, kept)
    chunks = _token_chunks(tokens, vocab)
    logits = _buffer(chunks[0][1], vocab, hidden.device)
    parts = [
        _C.linear_scores(hidden[first:end], weight, target[first:end], bias, _rows(temp, first, end), real, top_k, logits[: end - first])
        for first, end in chunks
    ]
    if len(parts) == 1:
        return parts[0]
    return [None if column[0] is None else torch.cat(column) for column in zip(*parts)]


def linear_scores_gradients(
    hidden, weight, target, temp, lse, entropy, top_ids, kept, real, g_logp, g_lse, g_entropy, g_top, need_hidden, need_weight, *, bias=None,
) -> tuple:  # fmt: skip
    """The gradients of ``hidden`` and ``weight`` that are wanted, ``None`` for the other; ``kept``: the forward's logits, or ``None``
    where they are computed again, a part of the tokens at a time."""
    grads = (g_logp, g_lse, g_entropy, g_top)
    refuse_tangents("the gradient of token scores", *grads)
    _host.refuse_capture_into_another_graph()
    with torch.no_grad():
        tokens, vocab = hidden.size(0), weight.size(0)
        dz = torch.empty((tokens, _C.linear_dlogits_row_stride(vocab)), dtype=torch.bfloat16, device=hidden.device)
        chunks = [(0, tokens)] if kept is not None or tokens == 0 else _token_chunks(tokens, vocab)
        logits = kept if kept is not None else _buffer(chunks[0][1], vocab, hidden.device)
        for first, end in chunks:
            some = logits[: end - first]
            rows_temp = _rows(temp, first, end)
            if kept is None:  # the bits of the forward's logits
                _C.fused_linear_logp_into(hidden[first:end], weight, target[first:end], bias, rows_temp, real, some)
            _C.logits_scores_backward(
                some[:, :vocab], target[first:end], real, lse[first:end], entropy[first:end], _rows(top_ids, first, end),
                tuple(_rows(g, first, end) for g in grads), temperature=rows_temp, out=dz[first:end],
            )  # fmt: skip
        del logits
        made = _C.linear_dlogits_bwd(dz, hidden, weight, need_hidden, need_weight)
    return tuple(without_second_derivative(made))


class _LinearScores(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, target_1d, temp, real, top_k, kept):
        logp, lse, entropy, top_logp, top_ids = _linear_scores(hidden, weight, bias, target_1d, temp, real, top_k, kept)
        ctx.save_for_backward(hidden, weight, target_1d, temp, lse, entropy, top_ids, kept, bias)
        ctx.real = real
        ctx.set_materialize_grads(False)
        if top_ids is not None:
            ctx.mark_non_differentiable(top_ids)
        return logp, lse, entropy, top_logp, top_ids

    @staticmethod
    def backward(ctx, g_logp, g_lse, g_entropy, g_top, _g_ids):
        grads = (g_logp, g_lse, g_entropy, g_top)
        if all(g is None for g in grads):
            return (None,) * 8
        *saved, bias = ctx.saved_tensors
        two = linear_scores_gradients(*saved, ctx.real, *grads, *ctx.needs_input_grad[:2], bias=bias)
        return *two, None, None, None, None, None, None


def hip_deterministic_linear_scores(
    hidden: torch.Tensor,
    lm_head_weight: torch.Tensor,
    target_ids: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    top_k: int = 0,
    temperature: Optional[torch.Tensor] = None,
    real_vocab_size: int = -1,
    validate: bool = False,
) -> TokenScores:
    """:class:`TokenScores` of ``hidden [..., D]`` through ``lm_head_weight [V, D]`` (bf16) for ``target_ids [...]``;
    differentiable in ``hidden`` and ``lm_head_weight``. Arguments as in
    :func:`~.linear_logp.hip_deterministic_linear_logp`, whose ``logp`` and ``lse`` these are, to the bit.

    A differentiable call keeps its fp32 logits for the backward where memory allows, as that function does (at most 8 GiB in
    all, not under ``recompute_logits``, saved-tensor hooks or graph capture). Otherwise no logits are written for more than 1024
    tokens without ``top_k``, and else they go through a buffer of at most 2 GiB, a part of the tokens at a time. d(logits) is
    rounded to bf16 once, as there, for the matrix instructions of the two products: with it the gradients of 2060 tokens are 0.0023 off
    in the mean where their own rounding leaves 0.0017. A ``bias`` is added but not differentiated.
    """
    refuse_tangents("token scores", hidden, lm_head_weight, bias)
    if bias is not None and torch.is_grad_enabled() and bias.requires_grad:
        raise RuntimeError("token scores do not differentiate the lm_head bias: pass bias.detach()")
    if target_ids.shape != hidden.shape[:-1]:
        raise ValueError(f"hidden leading shape {tuple(hidden.shape[:-1])} must match target_ids shape {tuple(target_ids.shape)}")
    if temperature is not None:
        temperature = _row_temperature(temperature, target_ids.numel(), hidden.device)
    hidden_2d, weight, target_1d, temp = _prepare(hidden, lm_head_weight, target_ids, temperature, False)
    vocab = weight.size(0)
    real = vocab if int(real_vocab_size) < 0 else int(real_vocab_size)
    if not 0 < real <= vocab:
        raise ValueError(f"real_vocab_size must be in [1, {vocab}], got {real_vocab_size}")
    top_k = _checked_top_k(top_k, real)
    if bias is not None:
        bias = bias.detach().contiguous()
    if validate and target_1d.numel():
        _validate_values(target_1d, temp, real)
    if _requires_grad(hidden_2d, weight):
        written_anyway = hidden_2d.size(0) > 0 and _C.linear_scores_needs_logits(hidden_2d, weight, bias, top_k)
        kept = _logits_to_save(hidden_2d, vocab, written_anyway)
        scores = None
        if kept is not None and bias is None and not torch.compiler.is_compiling():
            scores = _host.native().linear_scores(hidden_2d, weight, target_1d, temp, real, top_k, kept)  # everyday operands, natively
        if scores is None:
            scores = _LinearScores.apply(hidden_2d, weight, bias, target_1d, temp, real, top_k, kept)
    else:
        scores = _linear_scores(hidden_2d, weight, bias, target_1d, temp, real, top_k, None)
    return _shaped(scores, target_ids.shape)


__all__ = ["TokenScores", "hip_deterministic_linear_scores", "hip_deterministic_scores_from_logits"]
