"""Eight-bit copies of activations on a real MI355X: the codes of the definition, to the bit, and SwiGLU and the FFN on them."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def native():
    from rl_engine import _C

    return _C


def _normal(*shape, seed=0, dtype=torch.bfloat16, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def _definition(x):
    """(codes, scale bytes, values in 64 bits) of finite x."""
    rows, cols = x.shape
    runs = torch.nn.functional.pad(x.double(), (0, -cols % 32)).view(rows, (cols + 31) // 32, 32)
    most = runs.abs().amax(2, keepdim=True)
    exponent = (torch.frexp(most).exponent.double() - 1).where(most > 0, torch.full_like(most, -1000.0))
    exponent = (exponent - 6).clamp_min(-126)
    scale = torch.exp2(exponent)
    codes = (runs / scale).round().clamp(-127, 127)
    values = (codes * scale).flatten(1)[:, :cols]
    return codes.flatten(1)[:, :cols].to(torch.int8), (exponent[:, :, 0] + 127).to(torch.uint8), values


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 257), (300, 1000), (4, 12288), (1025, 48), (0, 64), (5, 0)])
def test_codes_are_those_of_the_definition(native, rows, cols, dtype):
    x = _normal(rows, cols, seed=rows + cols, dtype=dtype)
    if cols > 20:
        x[:, 5] *= 100.0
        x[::2, cols // 2 :] = 0.0
    codes, scales = native.mx8_encode(x)
    want_codes, want_scales, values = _definition(x)
    assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales)
    for out in DTYPES:
        assert torch.equal(native.mx8_decode(codes, scales, out), values.to(out))
    if rows and cols:
        # half a scale off, a whole one where 127 scales end short of the value; the largest of a run is at least 64 scales
        most = torch.nn.functional.pad(x.double(), (0, -cols % 32)).view(rows, -1, 32).abs().amax(2).repeat_interleave(32, 1)[:, :cols]
        assert bool(((values - x.double()).abs() <= most / 64 + 2.0**-126).all())


def test_values_at_the_ends_of_the_range(native):
    top = torch.finfo(torch.float32).max
    for value in (top, -top, 2.0**-126, 2.0**-149, 1.9921875, 1.99999988, 127.5, 63.5, 64.5, 2.0**-120, 2.0**-121):
        x = torch.zeros((2, 64), device=DEV)
        x[0, 3], x[1, 40] = value, value / 3
        codes, scales = native.mx8_encode(x)
        want_codes, want_scales, values = _definition(x)
        assert torch.equal(codes, want_codes) and torch.equal(scales, want_scales), value
        assert torch.equal(native.mx8_decode(codes, scales, torch.float32).double(), values), value


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_run_that_is_not_finite_is_nan(native, bad, dtype):
    x = _normal(3, 100, seed=2, dtype=dtype)
    clean = native.mx8_decode(*native.mx8_encode(x), dtype)
    x[1, 40], x[2, 99] = bad, bad
    got = native.mx8_decode(*native.mx8_encode(x), dtype)
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[1, 32:64], hit[2, 96:] = True, True
    assert bool(torch.isnan(got[hit]).all()) and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 7), (33, 256), (65, 1001), (16, 12288)])
def test_swiglu_is_that_of_the_copies(native, rows, cols, dtype):
    from rl_engine.ops.ffn import checkpointed_swiglu

    gate, up = _normal(rows, cols, seed=1, dtype=dtype, scale=2.0), _normal(rows, cols, seed=2, dtype=dtype)
    dy = _normal(rows, cols, seed=3, dtype=dtype)
    y, *kept = native.swiglu_mx8_forward(gate, up)
    for got, want in zip(kept, [*native.mx8_encode(gate), *native.mx8_encode(up)]):
        assert torch.equal(got, want)
    # fp16 results are rounded from the fp32 ones (the fp16 kernels of swiglu_forward may round a last product once, not twice)
    f = torch.float32 if dtype == torch.float16 else dtype
    kept_gate, kept_up = native.mx8_decode(*kept[:2], f), native.mx8_decode(*kept[2:], f)
    got = native.swiglu_mx8_backward(dy, *kept, with_activation=True)
    want = [*native.swiglu_backward(dy.to(f), kept_gate, kept_up), native.swiglu_forward(kept_gate, kept_up), native.swiglu_forward(gate.to(f), up.to(f))]
    for g, w in zip([*got, y], want):
        assert torch.equal(_bits(g), _bits(w.to(dtype)))

    g1, u1 = gate.clone().requires_grad_(True), up.clone().requires_grad_(True)
    out = checkpointed_swiglu(g1, u1)
    grads = torch.autograd.grad(out, [g1, u1], dy)
    for g, w in zip([out.detach(), *grads], [y, *got[:2]]):
        assert torch.equal(_bits(g), _bits(w))


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_result_is_the_same_without_a_gradient(dtype):
    from rl_engine.ops.ffn import checkpointed_swiglu

    gate, up = _normal(40, 1000, seed=1, dtype=dtype, scale=2.0), _normal(40, 1000, seed=2, dtype=dtype)
    want = checkpointed_swiglu(gate.clone().requires_grad_(True), up).detach()
    assert torch.equal(_bits(checkpointed_swiglu(gate, up)), _bits(want))
    both = torch.cat([gate, up], dim=1).chunk(2, dim=1)
    assert torch.equal(_bits(checkpointed_swiglu(*both)), _bits(want))


def test_gradient_of_what_was_kept_against_differences(native):
    """Central differences of SwiGLU in 64 bits at the kept values; fp32 gradients, off by 2^-20 of their factors."""
    gate, up, dy = _normal(4, 64, seed=5, dtype=torch.float32), _normal(4, 64, seed=6, dtype=torch.float32), _normal(4, 64, seed=7, dtype=torch.float32)
    _, *kept = native.swiglu_mx8_forward(gate, up)
    d_gate, d_up, _ = native.swiglu_mx8_backward(dy, *kept)
    g, u = native.mx8_decode(*kept[:2], torch.float32).double(), native.mx8_decode(*kept[2:], torch.float32).double()
    h = 1e-4
    f = lambda g, u: torch.nn.functional.silu(g) * u * dy.double()  # noqa: E731
    for got, want in ((d_gate, (f(g + h, u) - f(g - h, u)) / (2 * h)), (d_up, (f(g, u + h) - f(g, u - h)) / (2 * h))):
        assert bool(((got.double() - want).abs() <= (2.0**-20 + h * h) * (1 + g.abs()) * (1 + u.abs()) * dy.double().abs() + 1e-10).all())


def test_strided_rows_and_batches(native):
    from rl_engine.ops.ffn import checkpointed_swiglu

    both = _normal(6, 2 * 100, seed=8)
    gate, up = both.chunk(2, dim=1)
    want = native.swiglu_mx8_forward(gate.contiguous(), up.contiguous())
    for g, w in zip(native.swiglu_mx8_forward(gate, up), want):
        assert torch.equal(g, w)
    odd = torch.empty(6 * 100 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(6, 100).copy_(gate)
    for g, w in zip(native.mx8_encode(odd), want[1:3]):
        assert torch.equal(g, w)
    g3 = gate.reshape(2, 3, 100).requires_grad_(True)
    out = checkpointed_swiglu(g3, up.reshape(2, 3, 100))
    (grad,) = torch.autograd.grad(out.sum(), [g3])
    assert out.shape == g3.shape == grad.shape and torch.equal(out.reshape(6, 100), want[0])
    one = native.mx8_encode(_normal(100, seed=9).expand(1, 100))
    assert torch.equal(one[0], native.mx8_encode(_normal(100, seed=9)[None].contiguous())[0])


def test_more_than_four_gigabytes(native):
    rows, cols = 180000, 12288
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=DEV)
    x[-3:] = _normal(3, cols, seed=4)
    codes, scales = native.mx8_encode(x)
    last = native.mx8_encode(x[-3:].clone())
    assert torch.equal(codes[-3:], last[0]) and torch.equal(scales[-3:], last[1])
    assert torch.equal(native.mx8_decode(codes, scales)[-3:], native.mx8_decode(*last))


def test_ffn_keeps_eight_bits(native):
    """The output has the bits of the ordinary call; the gradients are those of an FFN whose backward sees the copies."""
    from rl_engine.backends.rocm.gemm.det_gemm import det_gemm_linear, det_gemm_linear_input_gradient, det_gemm_linear_weight_gradient
    from rl_engine.ops.ffn import Qwen3FFNOp, qwen3_ffn

    tokens, hidden, inter = 137, 256, 384
    x = _normal(tokens, hidden, seed=1).requires_grad_(True)
    weights = [_normal(*s, seed=2 + i, scale=0.08).requires_grad_(True) for i, s in enumerate([(inter, hidden), (inter, hidden), (hidden, inter)])]
    gy = _normal(tokens, hidden, seed=9)
    y = qwen3_ffn(x, *weights, checkpoint_bits=8)
    assert torch.equal(y, qwen3_ffn(x, *weights))
    grads = torch.autograd.grad(y, [x, *weights], gy)
    with torch.no_grad():
        wg, wu, wd = weights
        kept = [native.mx8_decode(*native.mx8_encode(t)) for t in (x, det_gemm_linear(x, wg), det_gemm_linear(x, wu))]
        dg, du = native.swiglu_backward(det_gemm_linear_input_gradient(gy, wd), kept[1], kept[2])
        want = [
            det_gemm_linear_input_gradient(dg, wg) + det_gemm_linear_input_gradient(du, wu), det_gemm_linear_weight_gradient(kept[0], dg),
            det_gemm_linear_weight_gradient(kept[0], du), det_gemm_linear_weight_gradient(native.swiglu_forward(kept[1], kept[2]), gy),
        ]  # fmt: skip
    for g, w in zip(grads, want):
        assert torch.equal(_bits(g), _bits(w))
    fused = torch.cat([wg, wu]).detach()
    packed = torch.autograd.grad(Qwen3FFNOp()(x, *weights, fused_gate_up_weight=fused, checkpoint_bits=8), [x, *weights], gy)
    for g, w in zip(packed, grads):
        assert torch.equal(_bits(g), _bits(w))
    # within the eight bits of the ordinary gradients: copies off by 2^-7 of a run's largest value at most, 2^-9 in the mean square of
    # half a step; through three factors of a term and a run's spread of ten that is 3 * 10 * 2^-9 of the norm
    plain = torch.autograd.grad(qwen3_ffn(x, *weights), [x, *weights], gy)
    for g, w in zip(grads, plain):
        assert float((g.double() - w.double()).norm() / w.double().norm()) < 30 * 2.0**-9
    (only,) = torch.autograd.grad(qwen3_ffn(x.detach(), weights[0].detach(), weights[1], weights[2].detach(), checkpoint_bits=8), [weights[1]], gy)
    assert torch.equal(only, grads[2])


def test_what_is_kept_is_small():
    from rl_engine.ops.ffn import qwen3_ffn

    tokens, hidden, inter = 512, 1024, 2048
    x = _normal(tokens, hidden, seed=1).requires_grad_(True)
    weights = [_normal(*s, seed=2 + i, scale=0.03) for i, s in enumerate([(inter, hidden), (inter, hidden), (hidden, inter)])]
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t.nbytes) or t, lambda t: t):
        qwen3_ffn(x, *weights, checkpoint_bits=8)
    kept = sum(saved) - sum(w.nbytes for w in weights)
    assert kept == tokens * (hidden + 2 * inter) * 33 // 32


def test_in_a_graph_and_on_another_stream(native):
    from rl_engine.ops.ffn import checkpointed_swiglu

    gate, up = _normal(40, 333, seed=1).requires_grad_(True), _normal(40, 333, seed=2).requires_grad_(True)
    dy = _normal(40, 333, seed=3)

    def step():
        y = checkpointed_swiglu(gate, up)
        return [y.detach(), *torch.autograd.grad(y, [gate, up], dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            gate.copy_(_normal(40, 333, seed=30 + seed))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_refused_calls(native):
    from rl_engine.ops.ffn import checkpointed_swiglu, qwen3_ffn

    x = _normal(4, 64)
    codes, scales = native.mx8_encode(x)
    for bad in (x.cpu(), x.double(), x[0]):
        with pytest.raises(RuntimeError):
            native.mx8_encode(bad)
    for args in ((codes, scales[:, :1]), (codes.cpu(), scales.cpu()), (codes.t(), scales), (codes.float(), scales)):
        with pytest.raises(RuntimeError):
            native.mx8_decode(*args)
    with pytest.raises(RuntimeError):
        native.mx8_decode(codes, scales, torch.float64)
    with pytest.raises(RuntimeError):
        native.swiglu_mx8_forward(x, x.float())
    with pytest.raises(RuntimeError):
        native.swiglu_mx8_backward(x[:2], codes, scales, codes, scales)
    with pytest.raises(ValueError):
        checkpointed_swiglu(x, x[:2])
    w = _normal(64, 64)
    for bits in (4, True, "8"):
        with pytest.raises(ValueError, match="checkpoint_bits"):
            qwen3_ffn(x, w, w, w, checkpoint_bits=bits)
