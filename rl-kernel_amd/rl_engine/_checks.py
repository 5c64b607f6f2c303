"""Argument checking for the host-side facades, written as tables.

A facade states what it requires as rows ``(holds, exception type, message)`` and hands them to
:func:`enforce`, which raises for the first row that does not hold. The exception types and the
message texts are part of the interface the facades keep (callers and tests match on them); the
tables keep them in one place per entry point instead of a chain of ``if`` statements.

``holds`` and ``message`` may be zero-argument callables, evaluated only when the row is reached:
use that for a condition that is only meaningful once the rows before it have passed (a size that
needs a 2-D tensor, a device comparison that needs a tensor at all).
"""

from __future__ import annotations

from collections.abc import Callable, Iterable
from typing import Union

import torch
from torch.autograd import forward_ad

Lazy = Union[bool, Callable[[], bool]]
Text = Union[str, Callable[[], str]]
Rule = tuple[Lazy, type, Text]


def enforce(rules: Iterable[Rule]) -> None:
    """Raise ``exception(message)`` of the first rule whose condition does not hold."""
    for holds, exception, message in rules:
        if callable(holds):
            holds = holds()
        if not holds:
            raise exception(message() if callable(message) else message)


def assert_async_or_raise(condition: torch.Tensor, exception: type, message: str, host_message: str | None = None) -> None:
    """A value check on a 0-d boolean tensor: a device-side assertion for a GPU tensor (the call never
    waits for the host, so it can sit inside a captured graph), an ordinary exception for a CPU one."""
    if condition.is_cuda:
        torch._assert_async(condition, message)
    elif not bool(condition):
        raise exception(host_message or message)


def refuse_tangents(what: str, *tensors) -> None:
    """For a kernel's host side, in front of its first look at the values: a forward-mode tangent would be lost there."""
    if forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: forward-mode derivatives are not implemented")


class _NoSecondDerivative(torch.autograd.Function):
    @staticmethod
    def forward(ctx, count, *tensors):
        return tuple(t.view_as(t) for t in tensors[:count])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("this gradient is not differentiable: it was computed by a kernel without a backward of its own")


def without_second_derivative(grads: list) -> list:
    """``grads`` (tensors or ``None``) that raise when somebody differentiates them, which is possible where a graph of the backward
    is made (``create_graph``); as they are elsewhere."""
    if not torch.is_grad_enabled() or all(g is None for g in grads):
        return grads
    given = [g for g in grads if g is not None]
    anchor = torch.empty((0,), device=given[0].device, requires_grad=True)  # (what they were computed from may be gone)
    given = iter(_NoSecondDerivative.apply(len(given), *given, anchor))
    return [None if g is None else next(given) for g in grads]


def output_buffer_rules(out: torch.Tensor, shape: tuple[int, int], device: torch.device, what: str) -> list[Rule]:
    """Rules for a caller-owned bf16 ``[M, N]`` output with contiguous rows (``what`` prefixes the messages)."""
    return [
        (tuple(out.shape) == tuple(shape), ValueError, f"{what} output must have shape {tuple(shape)}, got {tuple(out.shape)}"),
        (out.dtype == torch.bfloat16, TypeError, f"{what} output must be BF16, got {out.dtype}"),
        (out.device == device, RuntimeError, f"{what} output must live on the input device"),
        (lambda: out.stride(1) == 1, ValueError, f"{what} output rows must be contiguous"),
        (not out.requires_grad, ValueError, f"{what} output buffer must not require gradients"),
    ]
