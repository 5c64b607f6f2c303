"""Rotary positions of queries and keys (csrc/rotary.hip), differentiable."""

from __future__ import annotations

import ctypes
import math
from typing import List, Optional

import torch
from torch import Tensor

from rl_engine import _host, _lib
from rl_engine._C import _on, _stream_handle
from rl_engine._checks import enforce, refuse_tangents

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}
_SCALINGS = ("linear", "base", "bands", "wavelengths")


def rotary_frequencies(
    rotary_width: int,
    base: float = 10000.0,
    *,
    factor: float = 1.0,
    scaling: str = "linear",
    original_length: Optional[int] = None,
    fast_turns: Optional[float] = None,
    slow_turns: float = 1.0,
    device="cuda",
) -> Tensor:
    """Radians a position of each of the ``rotary_width / 2`` pairs, in 64 bits: ``f_i = base^(-2 i / rotary_width)``, scaled for contexts
    ``factor`` times as long as those of the training:

    ``linear``       ``f_i / factor``: positions are interpolated
    ``base``         a base ``factor^(r / (r - 2))`` times as large (``r`` the rotary width): the slowest pair is interpolated, the fastest kept
    ``bands``        pairs that make more than ``fast_turns`` (32) turns over ``original_length`` positions are kept, those that make
                     fewer than ``slow_turns`` interpolated; in between a ramp over the index of the pair, from whole indices outwards
    ``wavelengths``  the same with a ramp over the number of turns (``fast_turns`` 4)

    A magnitude that goes with a scaling (``0.1 ln(factor) + 1``, say) is an argument of the calls that rotate.
    """
    if isinstance(rotary_width, bool) or not isinstance(rotary_width, int) or rotary_width < 2 or rotary_width % 2:
        raise ValueError(f"rotary_width must be an even number of at least 2, got {rotary_width!r}.")
    base, factor = float(base), float(factor)
    enforce([
        (1.0 < base < math.inf, ValueError, f"base must be above 1 and finite, got {base}."),
        (0.0 < factor < math.inf, ValueError, f"factor must be positive and finite, got {factor}."),
        (scaling in _SCALINGS, ValueError, f"scaling must be one of {_SCALINGS}, got {scaling!r}."),
        (scaling != "base" or rotary_width > 2, ValueError, "scaling 'base' needs a rotary_width of at least 4."),
    ])  # fmt: skip
    half = rotary_width // 2
    index = torch.arange(half, dtype=torch.float64)
    if scaling == "base":
        base *= factor ** (rotary_width / (rotary_width - 2))
    plain = base ** (-index / half)
    if scaling == "base":
        return plain.to(device)
    if scaling == "linear":
        return (plain / factor).to(device)
    fast = float(fast_turns if fast_turns is not None else 32.0 if scaling == "bands" else 4.0)
    if original_length is None or not original_length > 0:
        raise ValueError(f"scaling {scaling!r} needs the original_length (above 0), got {original_length!r}.")
    if not 0.0 < slow_turns < fast < math.inf:
        raise ValueError(f"0 < slow_turns < fast_turns must hold, got {slow_turns} and {fast}.")
    if scaling == "bands":
        at = lambda turns: half * math.log(original_length / (2 * math.pi * turns)) / math.log(base)  # noqa: E731
        first, last = max(math.floor(at(fast)), 0), min(math.ceil(at(slow_turns)), rotary_width - 1)
        kept = 1 - ((index - first) / max(last - first, 1e-3)).clamp(0, 1)
    else:
        kept = ((original_length * plain / (2 * math.pi) - slow_turns) / (fast - slow_turns)).clamp(0, 1)
    return (plain * kept + plain / factor * (1 - kept)).to(device)


def rotary_of(frequencies: Tensor, positions: Optional[Tensor], interleaved: bool, magnitude: float) -> _lib.Rotary:
    return _lib.Rotary(
        frequencies.data_ptr(), None if positions is None else positions.data_ptr(),
        int(positions is not None and positions.dtype == torch.int64), frequencies.numel(), int(interleaved), magnitude,
    )  # fmt: skip


def _leading(t: Tensor) -> Tensor:
    """``t`` with one or two dimensions in front of its heads, a head's elements side by side."""
    if t.dim() > 4:
        t = t.flatten(0, -4)
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


def _head_rows(x: Tensor, y: Tensor) -> _lib.HeadRows:
    outer = lambda t: t.stride(0) if t.dim() == 4 else 0  # noqa: E731
    return _lib.HeadRows(
        x.data_ptr(), y.data_ptr(), outer(x), x.stride(-3), x.stride(-2), outer(y), y.stride(-3), y.stride(-2), x.size(-2),
    )  # fmt: skip


def _rotate(tensors: list, positions: Tensor, frequencies: Tensor, interleaved: bool, magnitude: float, inverse: bool) -> list:
    """``tensors`` (one or two) rotated, into new ones."""
    if _host.recorded(*tensors, positions, frequencies):
        return _rotate_operator(tensors[0], tensors[1] if len(tensors) > 1 else None, positions, frequencies, interleaved, magnitude, inverse)
    return _launch(tensors, positions, frequencies, interleaved, magnitude, inverse)


@torch.library.custom_op("rl_kernel::rotary_embedding", mutates_args=())
def _rotate_operator(
    q: Tensor, k: Optional[Tensor], positions: Tensor, frequencies: Tensor, interleaved: bool, magnitude: float, inverse: bool
) -> List[Tensor]:
    _host.refuse_capture_into_another_graph()  # (in a compiler's backward)
    return _launch([t for t in (q, k) if t is not None], positions, frequencies, interleaved, magnitude, inverse)


@_rotate_operator.register_fake
def _rotate_operator_fake(q, k, positions, frequencies, interleaved, magnitude, inverse):
    return [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k) if t is not None]


def _launch(tensors: list, positions: Tensor, frequencies: Tensor, interleaved: bool, magnitude: float, inverse: bool) -> list:
    device = tensors[0].device
    made, described, held = [], [], []
    for x in tensors:
        y = torch.empty(x.shape, dtype=x.dtype, device=device)
        x = _leading(x)
        made.append(y)
        held.append(x)
        described.append(_head_rows(x, y.view(x.shape)))
    first = held[0]
    tokens = positions.numel()
    inner = first.size(1) if first.dim() == 4 and first.size(0) != 1 else tokens
    rotary = rotary_of(frequencies, positions, interleaved, magnitude)
    with _on(device):
        status = _lib.load().rlk_rotary_embedding(
            ctypes.byref(rotary), ctypes.byref(described[0]), ctypes.byref(described[1]) if len(described) > 1 else None, tokens, inner,
            first.size(-1), _DTYPES[first.dtype], int(inverse), _stream_handle(device),
        )  # fmt: skip
    _lib.check(status, "rlk_rotary_embedding failed")
    return made


class _Rotary(torch.autograd.Function):
    """The gradient of a rotation is the rotation the other way, which is differentiable in turn."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved, magnitude, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (interleaved, magnitude)
        ctx.inverse = inverse
        made = _rotate([t for t in (q, k) if t is not None], positions, frequencies, interleaved, magnitude, inverse)
        return tuple(made) if k is not None else (made[0], None)

    @staticmethod
    def backward(ctx, g_q, g_k):
        return *rotary_gradients(g_q, g_k, *ctx.saved_tensors, *ctx.how, not ctx.inverse), None, None, None, None, None


def rotary_gradients(
    g_q: Optional[Tensor], g_k: Optional[Tensor], positions: Tensor, frequencies: Tensor, interleaved: bool, magnitude: float, inverse: bool = True
) -> tuple[Optional[Tensor], Optional[Tensor]]:
    """The gradients of ``q`` and ``k`` from those of their turned forms, differentiable; ``None`` where there is none."""
    refuse_tangents("the gradient of a rotation", g_q, g_k)
    if not torch.compiler.is_compiling():  # (the operator does it when it runs)
        _host.refuse_capture_into_another_graph()
    given = [g for g in (g_q, g_k) if g is not None]
    if not given:
        return None, None
    turned = iter(_Rotary.apply(given[0], given[1] if len(given) > 1 else None, positions, frequencies, interleaved, magnitude, inverse))
    return tuple(None if g is None else next(turned) for g in (g_q, g_k))


def check_frequencies(frequencies: Tensor, device: torch.device, width: int) -> Tensor:
    enforce([
        (isinstance(frequencies, Tensor), TypeError, lambda: f"frequencies must be a torch.Tensor, got {type(frequencies)!r}."),
        (lambda: frequencies.dtype == torch.float64, TypeError, lambda: f"frequencies must be fp64 (rotary_frequencies makes them), got {frequencies.dtype}."),
        (lambda: not (torch.is_grad_enabled() and frequencies.requires_grad), RuntimeError, "frequencies have no gradient: pass frequencies.detach()."),
        (lambda: frequencies.device == device, RuntimeError, lambda: f"frequencies must be on {device}, got {frequencies.device}."),
        (lambda: frequencies.dim() == 1 and 2 * frequencies.numel() <= width, ValueError, lambda: f"frequencies must be [pairs] with at most {width // 2} of them, got shape {tuple(frequencies.shape)}."),
    ])  # fmt: skip
    return frequencies.contiguous()


def check_positions(positions: Tensor, shape: tuple, device: torch.device) -> Tensor:
    enforce([
        (isinstance(positions, Tensor), TypeError, lambda: f"positions must be a torch.Tensor, got {type(positions)!r}."),
        (lambda: positions.dtype in (torch.int32, torch.int64), TypeError, lambda: f"positions must be int32 or int64, got {positions.dtype}."),
        (lambda: positions.device == device, RuntimeError, lambda: f"positions must be on {device}, got {positions.device}."),
        (lambda: tuple(positions.shape) == tuple(shape), ValueError, lambda: f"positions must have shape {tuple(shape)}, got {tuple(positions.shape)}."),
    ])  # fmt: skip
    return positions.contiguous()


def _check_heads(t: Tensor, name: str) -> None:
    enforce([
        (isinstance(t, Tensor), TypeError, lambda: f"{name} must be a torch.Tensor, got {type(t)!r}."),
        (lambda: t.dim() >= 3, ValueError, lambda: f"{name} must be [..., heads, width] with at least one dimension of tokens, got shape {tuple(t.shape)}."),
        (lambda: t.dtype in _DTYPES, TypeError, lambda: f"{name} must be bf16, fp16 or fp32, got {t.dtype}."),
        (lambda: t.is_cuda, RuntimeError, lambda: f"{name} must be on a CUDA/ROCm GPU device, got '{t.device}'."),
        (lambda: 1 <= t.size(-1) <= _lib.ROTARY_MAX_WIDTH, ValueError, lambda: f"{name} must have heads of 1 to {_lib.ROTARY_MAX_WIDTH} elements, got {t.size(-1)}."),
    ])  # fmt: skip


def rotary_embedding(
    q: Tensor, k: Optional[Tensor], positions: Tensor, frequencies: Tensor, *, interleaved: bool = False, magnitude: float = 1.0
) -> tuple[Tensor, Optional[Tensor]]:
    """``q`` and ``k`` (or ``None``) turned by their positions, as new contiguous tensors; differentiable in both, to any order (not in the
    frequencies: some that require a gradient are refused).

    ``q [..., heads, width]`` and ``k [..., key heads, width]`` are bf16, fp16 or fp32, of any strides, ``positions [...]`` int32 or int64,
    ``frequencies [pairs]`` fp64 (:func:`rotary_frequencies`). The first ``2 * pairs`` elements of a head are turned, the others copied. Pair i is
    the elements ``(i, pairs + i)``, or ``(2 i, 2 i + 1)`` with ``interleaved``:

    ``(a, b) -> magnitude * (a cos t - b sin t, b cos t + a sin t)``, ``t = position * frequencies[i]``

    Angles are reduced to a turn in 64 bits, so that far positions lose nothing; the rest is fp32, rounded once.
    """
    if isinstance(q, Tensor) and q.is_cuda and not torch.compiler.is_compiling():
        both = _host.native().rotary(q, k, positions, frequencies, interleaved, magnitude)  # everyday arguments, natively
        if both is not None:
            return both
    refuse_tangents("rotary_embedding", q, k, frequencies)
    _check_heads(q, "q")
    if k is not None:
        _check_heads(k, "k")
        enforce([
            (k.dtype == q.dtype, TypeError, lambda: f"k must be {q.dtype} as q is, got {k.dtype}."),
            (k.device == q.device, RuntimeError, lambda: f"k must be on {q.device}, got {k.device}."),
            (k.shape[:-2] == q.shape[:-2] and k.size(-1) == q.size(-1), ValueError, lambda: f"k must have the tokens and the width of q {tuple(q.shape)}, got {tuple(k.shape)}."),
        ])  # fmt: skip
    frequencies = check_frequencies(frequencies, q.device, q.size(-1))
    positions = check_positions(positions, q.shape[:-2], q.device)
    magnitude = float(magnitude)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, positions, frequencies, bool(interleaved), magnitude, False)
    made = _rotate([t for t in (q, k) if t is not None], positions, frequencies, bool(interleaved), magnitude, False)
    return made[0], made[1] if k is not None else None


__all__ = ["rotary_embedding", "rotary_frequencies"]
