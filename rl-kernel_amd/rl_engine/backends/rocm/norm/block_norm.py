"""What lies between two blocks of a transformer, in one pass over its rows (csrc/block_norm.hip).

The FFN takes a normed input (``rmsnorm_output``) and returns what is to be added to the residual stream. Between the two stand
the norm of the block's output (where a model has one), a gate, the residual scale, the sum, and the norm that the next block
reads: :func:`gated_residual_norm`. :func:`rms_norm` is the norm alone, in front of the first block. Both are differentiable in
every tensor; a row's results depend on that row only, and nothing is read back from the device.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from rl_engine import _host, _lib
from rl_engine._C import _on, _row_stride, _stream_handle
from rl_engine._checks import enforce, refuse_tangents, without_second_derivative

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}


def _rows(t: Tensor, width: int) -> Tensor:
    """``t`` as rows that follow one another at any distance."""
    t = t if t.dim() == 2 else t.reshape(-1, width)
    return t if t.stride(1) == 1 and t.stride(0) >= width else t.contiguous()


def _address(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _code(t: Optional[Tensor], dtype: torch.dtype) -> int:
    return _DTYPES[dtype if t is None else t.dtype]


def _describe(block, residual, gate, gate_kind, post, pre, rstd, dtype, eps, scale) -> _lib.BlockNorm:
    tokens, width = residual.shape
    return _lib.BlockNorm(
        _address(block), residual.data_ptr(), _address(gate), _address(post), _address(pre), _address(rstd),
        width if block is None else _row_stride(block), _row_stride(residual), 0 if gate is None or gate_kind == _lib.GATE_CHANNEL else _row_stride(gate),
        tokens, width, _DTYPES[dtype], _DTYPES[residual.dtype], gate_kind, _code(gate, dtype), _code(post, dtype), _code(pre, dtype), eps, scale,
    )  # fmt: skip


def _forward(block, residual, gate, gate_kind, post, pre, dtype, eps, scale, with_total, keep):
    """``(total, normed, rstd)``; ``keep``: the row factors that a backward reads are wanted."""
    tokens, width = residual.shape
    device = residual.device
    total = torch.empty((tokens, width), dtype=residual.dtype, device=device) if with_total else None
    normed = torch.empty((tokens, width), dtype=dtype, device=device) if pre is not None else None
    rstd = torch.empty((2, tokens), dtype=torch.float32, device=device) if keep else None
    norm = _describe(block, residual, gate, gate_kind, post, pre, rstd, dtype, eps, scale)
    with _on(device):
        status = _lib.load().rlk_block_norm_forward(ctypes.byref(norm), _address(total), _address(normed), _stream_handle(device))
    _lib.check(status, "rlk_block_norm_forward failed")
    return total, normed, rstd


def norm_gradients(
    block, residual, gate, post, pre, rstd, gate_kind, eps, scale, g_total, g_normed, need_block, need_residual, need_gate, need_post, need_pre,
    *, dtype: Optional[torch.dtype] = None,
) -> tuple:  # fmt: skip
    """The gradients of ``block``, ``residual``, ``gate`` and the weights that are wanted, ``None`` for the others. ``block`` and
    ``residual`` are rows or batches of rows; ``dtype``: the type of the normed result (that of ``block``, or of ``residual``)."""
    refuse_tangents("the gradient of a norm", g_total, g_normed)
    _host.refuse_capture_into_another_graph()
    dtype = dtype or (residual if block is None else block).dtype
    device, width = residual.device, residual.size(-1)
    with torch.no_grad():
        rows = [None if t is None else _rows(t, width) for t in (block, residual)]
        tokens = rows[1].size(0)
        g_rows = [None if g is None else g.reshape(tokens, width).to(t).contiguous() for g, t in ((g_total, residual.dtype), (g_normed, dtype))]
        new = lambda t, want: torch.empty(t.shape, dtype=t.dtype, device=device) if want else None  # noqa: E731
        made = [new(block, need_block), new(residual, need_residual), new(gate, need_gate), new(post, need_post), new(pre, need_pre)]
        lib = _lib.load()
        size = int(lib.rlk_block_norm_workspace_bytes(tokens, width))
        workspace = torch.empty((size,), dtype=torch.uint8, device=device)
        flat_gate = gate if gate is None or gate_kind == _lib.GATE_CHANNEL else _rows(gate, gate.size(-1))
        norm = _describe(*rows, flat_gate, gate_kind, post, pre, rstd, dtype, eps, scale)
        with _on(device):
            status = lib.rlk_block_norm_backward(
                ctypes.byref(norm), *(_address(g) for g in g_rows), *(_address(d) for d in made), workspace.data_ptr(), size,
                _stream_handle(device),
            )  # fmt: skip
        _lib.check(status, "rlk_block_norm_backward failed")
    return tuple(without_second_derivative(made))


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, block, residual, gate, post, pre, gate_kind, dtype, eps, scale, with_total):
        total, normed, rstd = _forward(block, residual, gate, gate_kind, post, pre, dtype, eps, scale, with_total, True)
        ctx.save_for_backward(block, residual, gate, post, pre, rstd)
        ctx.how = (gate_kind, eps, scale)
        ctx.dtype = dtype
        ctx.set_materialize_grads(False)
        return total, normed

    @staticmethod
    def backward(ctx, g_total, g_normed):
        if g_total is None and g_normed is None:
            return (None,) * 10
        grads = norm_gradients(*ctx.saved_tensors, *ctx.how, g_total, g_normed, *ctx.needs_input_grad[:5], dtype=ctx.dtype)
        return *grads, None, None, None, None, None


def _check_rows(t: Tensor, name: str) -> None:
    enforce([
        (isinstance(t, Tensor), TypeError, lambda: f"{name} must be a torch.Tensor, got {type(t)!r}."),
        (lambda: t.dim() >= 1 and 1 <= t.size(-1) <= _lib.NORM_MAX_WIDTH, ValueError, lambda: f"{name} must have rows of 1 to {_lib.NORM_MAX_WIDTH} elements, got shape {tuple(t.shape)}."),
        (lambda: t.dtype in _DTYPES, TypeError, lambda: f"{name} must be bf16, fp16 or fp32, got {t.dtype}."),
        (lambda: t.is_cuda, RuntimeError, lambda: f"{name} must be on a CUDA/ROCm GPU device, got '{t.device}'."),
    ])  # fmt: skip


def _check_eps(eps: float) -> float:
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must be at least 0, got {eps}.")
    return eps


def _check_beside(t: Tensor, name: str, home: Tensor, dtype: torch.dtype) -> None:
    enforce([
        (isinstance(t, Tensor), TypeError, lambda: f"{name} must be a torch.Tensor, got {type(t)!r}."),
        (lambda: t.device == home.device, RuntimeError, lambda: f"{name} must be on {home.device}, got {t.device}."),
        (lambda: t.dtype in (dtype, torch.float32), TypeError, lambda: f"{name} must be {dtype} or fp32, got {t.dtype}."),
    ])  # fmt: skip


def _vector(t: Optional[Tensor], name: str, home: Tensor, dtype: torch.dtype) -> Optional[Tensor]:
    if t is None:
        return None
    _check_beside(t, name, home, dtype)
    if tuple(t.shape) != (home.size(-1),):
        raise ValueError(f"{name} must have shape ({home.size(-1)},), got {tuple(t.shape)}.")
    return t.contiguous()


def _gate_rows(gate: Optional[Tensor], block: Tensor) -> tuple:
    """The gate as the kernels take it, and its kind."""
    if gate is None:
        return None, _lib.GATE_NONE
    _check_beside(gate, "gate", block, block.dtype)
    width = block.size(-1)
    if tuple(gate.shape) == (width,):
        return gate.contiguous(), _lib.GATE_CHANNEL
    if gate.shape == block.shape:
        return _rows(gate, width), _lib.GATE_FULL
    if tuple(gate.shape) == (*block.shape[:-1], 1):
        return gate.reshape(-1, 1), _lib.GATE_TOKEN
    raise ValueError(f"gate must have shape ({width},), {(*block.shape[:-1], 1)} or {tuple(block.shape)}, got {tuple(gate.shape)}.")


def _differentiable(*tensors: Optional[Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def gated_residual_norm(
    block: Tensor,
    residual: Tensor,
    weight: Optional[Tensor] = None,
    *,
    post_weight: Optional[Tensor] = None,
    gate: Optional[Tensor] = None,
    residual_scale: float = 1.0,
    eps: float = 1e-6,
) -> tuple[Tensor, Optional[Tensor]]:
    """``(residual + residual_scale * gate * norm(block), norm of that sum)``; differentiable in every tensor.

    ``norm(block) = block / sqrt(mean(block^2) + eps) * post_weight`` over the last dimension, or ``block`` itself without a
    ``post_weight``; the second result is the sum normed with ``weight`` in the same way (``None`` without one), taken from
    the sum before it is rounded to the residual's type. ``gate``: ``[width]``, ``[..., 1]``, ``[..., width]`` or ``None``.

    ``block [..., width]`` is bf16, fp16 or fp32 and the normed result has its type; ``residual`` (and the sum), ``gate`` and the
    weights have that type or fp32. Arithmetic is in fp32 with one rounding per result. Rows have up to 16384 elements.
    """
    if isinstance(block, Tensor) and not torch.compiler.is_compiling():
        both = _host.native().norm(block, residual, gate, post_weight, weight, eps, residual_scale)  # everyday arguments, natively
        if both is not None:
            return both
    refuse_tangents("gated_residual_norm", block, residual, weight, post_weight, gate)
    _check_rows(block, "block")
    _check_beside(residual, "residual", block, block.dtype)
    if residual.shape != block.shape:
        raise ValueError(f"residual must have the shape of block {tuple(block.shape)}, got {tuple(residual.shape)}.")
    shape, width = block.shape, block.size(-1)
    post = _vector(post_weight, "post_weight", block, block.dtype)
    pre = _vector(weight, "weight", block, block.dtype)
    gate_rows, kind = _gate_rows(gate, block)
    args = (_rows(block, width), _rows(residual, width), gate_rows, post, pre)
    how = (block.dtype, _check_eps(eps), float(residual_scale), True)
    if _differentiable(*args):
        total, normed = _BlockNorm.apply(*args, kind, *how)
    else:
        total, normed, _ = _forward(*args[:3], kind, *args[3:], *how, False)
    if len(shape) == 2:
        return total, normed
    return total.reshape(shape), None if normed is None else normed.reshape(shape)


def rms_norm(x: Tensor, weight: Tensor, *, eps: float = 1e-6, dtype: Optional[torch.dtype] = None) -> Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in ``dtype`` (that of ``x``; an fp32 ``x`` may be normed
    to any); differentiable in ``x`` and ``weight``, which has the result's type or fp32. Rows have up to 16384 elements."""
    if dtype is None and not torch.compiler.is_compiling():
        both = _host.native().norm(None, x, None, None, weight, eps, 1.0)
        if both is not None:
            return both[1]
    refuse_tangents("rms_norm", x, weight)
    _check_rows(x, "x")
    dtype = x.dtype if dtype is None else dtype
    if dtype not in _DTYPES or x.dtype not in (dtype, torch.float32):
        raise TypeError(f"the norm of {x.dtype} is {x.dtype}, of fp32 also bf16 or fp16; got {dtype}.")
    if weight is None:
        raise TypeError("weight must be a torch.Tensor, got None.")
    pre = _vector(weight, "weight", x, dtype)
    rows = _rows(x, x.size(-1))
    how = (dtype, _check_eps(eps), 1.0, False)
    if _differentiable(rows, pre):
        normed = _BlockNorm.apply(None, rows, None, None, pre, _lib.GATE_NONE, *how)[1]
    else:
        normed = _forward(None, rows, None, _lib.GATE_NONE, None, pre, *how, False)[1]
    return normed.reshape(x.shape)


__all__ = ["gated_residual_norm", "rms_norm"]
