"""Token scores, norms between blocks and eight-bit copies: the native host side against the general way, to the bit, and both
where the arguments are more than values in memory."""

from __future__ import annotations

import gc

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


class _Nothing:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture()
def general(monkeypatch):
    """A function that runs its argument the general way."""
    from rl_engine import _host

    def run(call):
        with monkeypatch.context() as m:
            m.setattr(_host, "_native", _Nothing())
            return call()

    return run


def _normal(*shape, seed=0, dtype=BF16, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _same(got, want):
    assert len(got) == len(want)
    for g, w in zip(got, want):
        assert (g is None) == (w is None)
        if g is not None:
            assert g.shape == w.shape and g.dtype == w.dtype and g.requires_grad == w.requires_grad
            assert torch.equal(g.detach().nan_to_num(7.0), w.detach().nan_to_num(7.0))


@pytest.mark.parametrize("top_k", [0, 5])
@pytest.mark.parametrize("tempered", [False, True])
def test_scores(general, top_k, tempered):
    from rl_engine import _host
    from rl_engine.ops.logprob import deterministic_scores_from_logits

    z = _normal(9, 777, seed=1, scale=3.0).requires_grad_(True)
    target = torch.arange(9, device=DEV) * 70
    temp = 0.5 + torch.rand(9, device=DEV) if tempered else None
    assert _host.native().scores(z, target, temp, 770, top_k) is not None

    def call():
        s = deterministic_scores_from_logits(z, target, top_k=top_k, temperature=temp, real_vocab_size=770)
        outputs = [s.logp, s.lse, s.entropy] + ([s.top_logp] if top_k else [])
        grads = [_normal(*o.shape, seed=10 + i, dtype=FP32) for i, o in enumerate(outputs)]
        one = torch.autograd.grad(s.entropy, [z], grads[2], retain_graph=True)
        late = torch.autograd.grad(s.logp, [z], torch.ones((), device=DEV).expand(9), retain_graph=True)  # a gradient with stride 0
        return [*s, *torch.autograd.grad(outputs, [z], grads), *one, *late]

    _same(call(), general(call))
    with torch.no_grad():
        _same(list(deterministic_scores_from_logits(z, target, top_k=top_k)), general(lambda: list(deterministic_scores_from_logits(z, target, top_k=top_k))))


@pytest.mark.parametrize("top_k", [0, 5])
@pytest.mark.parametrize("tokens", [7, 1100])
def test_linear_scores(general, top_k, tokens):
    from rl_engine.ops.logprob import deterministic_linear_scores

    h, w = _normal(tokens, 1536, seed=1).requires_grad_(True), _normal(500, 1536, seed=2, scale=0.05).requires_grad_(True)
    target = torch.arange(tokens, device=DEV) % 500
    temp = 0.5 + torch.rand(tokens, device=DEV)

    def call():
        s = deterministic_linear_scores(h, w, target, top_k=top_k, temperature=temp, real_vocab_size=497)
        outputs = [s.logp, s.lse, s.entropy] + ([s.top_logp] if top_k else [])
        grads = [_normal(*o.shape, seed=10 + i, dtype=FP32) for i, o in enumerate(outputs)]
        one = torch.autograd.grad(s.entropy, [w], grads[2], retain_graph=True)
        late = torch.autograd.grad(s.logp, [h], torch.ones((), device=DEV).expand(tokens), retain_graph=True)
        return [*s, *torch.autograd.grad(outputs, [h, w], grads), *one, *late]

    _same(call(), general(call))


@pytest.mark.parametrize("shape", [(6, 200), (2, 3, 200), (200,)])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("wide", [BF16, FP32])
def test_norm(general, shape, gate, post, wide):
    from rl_engine import _host
    from rl_engine.ops.norm import gated_residual_norm

    width = shape[-1]
    block, residual = _normal(*shape, seed=1), _normal(*shape, seed=2, dtype=wide)
    gates = {"none": None, "channel": (width,), "token": (*shape[:-1], 1), "full": shape}
    g = _normal(*gates[gate], seed=3) if gates[gate] else None
    w_post = _normal(width, seed=4, dtype=FP32) if post else None
    w_pre = _normal(width, seed=5)
    leaves = [t.requires_grad_(True) for t in (block, residual, g, w_post, w_pre) if t is not None]
    assert _host.native().norm(block, residual, g, w_post, w_pre, 1e-6, 0.5) is not None
    g_total, g_normed = _normal(*shape, seed=6, dtype=wide), _normal(*shape, seed=7)

    def call():
        total, normed = gated_residual_norm(block, residual, w_pre, post_weight=w_post, gate=g, residual_scale=0.5)
        some = torch.autograd.grad(normed, [residual, w_pre], g_normed, retain_graph=True)
        return [total, normed, *some, *torch.autograd.grad([total, normed], leaves, [g_total, g_normed])]

    _same(call(), general(call))

    def partly():  # gradients of some tensors only, and an output without a weight
        total, normed = gated_residual_norm(block.detach(), residual, None, post_weight=w_post, gate=g)
        assert normed is None
        return [total, *torch.autograd.grad(total, [t for t in (residual, g) if t is not None], g_total)]

    _same(partly(), general(partly))
    with torch.no_grad():
        inference = lambda: list(gated_residual_norm(block, residual, w_pre, post_weight=w_post, gate=g))  # noqa: E731
        _same(inference(), general(inference))


def test_rms_norm(general):
    from rl_engine.ops.norm import rms_norm

    x, w = _normal(3, 5, 96, seed=1).requires_grad_(True), _normal(96, seed=2, dtype=FP32).requires_grad_(True)

    def call():
        y = rms_norm(x, w)
        return [y, *torch.autograd.grad(y, [x, w], _normal(3, 5, 96, seed=3))]

    _same(call(), general(call))


@pytest.mark.parametrize("shape", [(4, 100), (2, 3, 64), (33,)])
def test_checkpointed_swiglu(general, shape):
    from rl_engine import _host
    from rl_engine.ops.ffn import checkpointed_swiglu, mx8_encode

    gate, up = _normal(*shape, seed=1).requires_grad_(True), _normal(*shape, seed=2).requires_grad_(True)
    assert _host.native().mx8_swiglu(gate, up) is not None

    def call():
        y = checkpointed_swiglu(gate, up)
        one = torch.autograd.grad(y, [up], _normal(*shape, seed=4), retain_graph=True)
        return [y, *one, *torch.autograd.grad(y, [gate, up], _normal(*shape, seed=3))]

    _same(call(), general(call))
    flat = gate.detach().reshape(-1, shape[-1])
    _same(mx8_encode(flat), general(lambda: mx8_encode(flat)))


def test_the_entry_points_take_the_native_way():
    for name, call in _calls().items():
        out = call(_normal(4, 64, seed=1).requires_grad_(True))
        assert type(out.grad_fn).__name__ == "CppFunction", name


def _calls():
    from rl_engine.ops.ffn import checkpointed_swiglu
    from rl_engine.ops.logprob import deterministic_linear_scores, deterministic_scores_from_logits
    from rl_engine.ops.norm import gated_residual_norm

    ids = torch.arange(4, device=DEV)
    w = _normal(64, 64, seed=3)
    return {
        "scores": lambda x: deterministic_scores_from_logits(x, ids, top_k=2).entropy,
        "linear": lambda x: deterministic_linear_scores(x, w, ids).entropy,
        "norm": lambda x: gated_residual_norm(x, x, w[0])[1],
        "swiglu": lambda x: checkpointed_swiglu(x, x),
    }


@pytest.mark.parametrize("name", ["scores", "linear", "norm", "swiglu"])
def test_a_gradient_of_a_gradient_is_refused(general, name):
    call = _calls()[name]
    x = _normal(4, 64, seed=1).requires_grad_(True)

    def twice():
        (grad,) = torch.autograd.grad(call(x).float().square().sum(), [x], create_graph=True)
        plain = torch.autograd.grad(call(x).float().square().sum(), [x])
        assert torch.equal(grad, plain[0])
        with pytest.raises(RuntimeError, match="not differentiable"):
            grad.float().sum().backward()

    twice()
    general(twice)


@pytest.mark.parametrize("name", ["scores", "linear", "norm"])  # (the SwiGLU keeps copies, not its inputs)
def test_an_input_changed_before_the_backward_is_noticed(general, name):
    call = _calls()[name]

    def changed():
        x = _normal(4, 64, seed=1).requires_grad_(True)
        z = x * 1
        out = call(z)
        z.data.add_(0)  # (not seen)
        with torch.no_grad():
            z.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()

    changed()
    general(changed)


@pytest.mark.parametrize("name", ["scores", "linear", "norm", "swiglu"])
def test_saved_tensors_under_hooks(general, name):
    """What is kept passes through saved-tensor hooks (offloading, checkpointing) and comes back."""
    call = _calls()[name]
    x = _normal(4, 64, seed=1).requires_grad_(True)
    want = torch.autograd.grad(call(x).sum(), [x])[0]

    def hooked():
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
            out = call(x)
        return torch.autograd.grad(out.sum(), [x])[0]

    assert torch.equal(hooked(), want) and torch.equal(general(hooked), want)
    again = torch.utils.checkpoint.checkpoint(lambda t: call(t).sum(), x, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(again, [x])[0], want)


def test_backward_on_the_stream_of_the_forward():
    """The engine runs a backward on its forward's stream; another stream waits for it as for any operator."""
    from rl_engine.ops.norm import gated_residual_norm

    x, w = _normal(3000, 4096, seed=1).requires_grad_(True), _normal(4096, seed=2)
    want = torch.autograd.grad(gated_residual_norm(x, x, w)[1].float().square().mean(), [x])[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = gated_residual_norm(x, x, w)[1]
    torch.cuda.current_stream().wait_stream(side)
    got = torch.autograd.grad(out.float().square().mean(), [x])[0]
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", ["scores", "linear", "norm", "swiglu", "ffn", "behind a cast"])
def test_a_backward_is_not_captured_into_another_graph(general, name):
    """The leaf's gatherer belongs to the stream that an earlier graph was made on; the default stream cannot join a capture: refused in
    front of any launch. The capture goes on, and so does the earlier graph; without it the same capture is taken."""
    from rl_engine.ops.ffn import qwen3_ffn

    w = _normal(64, 64, seed=3)
    calls = _calls()
    swiglu = calls["swiglu"]
    call = {"ffn": lambda x: qwen3_ffn(x, w, w, w, checkpoint_bits=8), "behind a cast": lambda x: swiglu(x.float()), **calls}[name]

    def refused():
        x = _normal(4, 64, seed=1).requires_grad_(True)
        g = torch.ones_like(call(x).detach())
        step = lambda: torch.autograd.grad(call(x), [x], g)[0]  # noqa: E731
        want = step()
        held = call(x)
        a = torch.ones(64, device=DEV)
        a + 1
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            inside = call(x)
            with pytest.raises(RuntimeError, match="cannot be captured"):
                torch.autograd.grad(inside, [x], g)
            b = a + 1
        for start in (3.0, 5.0):
            a.fill_(start)
            graph.replay()
            torch.cuda.synchronize()
            assert bool((b == start + 1).all())
        assert torch.equal(torch.autograd.grad(held, [x], g)[0], want)
        del held, inside
        gc.collect()  # (what the refusal's traceback holds)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)

    refused()
    general(refused)


def test_what_wants_no_gradient_is_no_obstacle(general):
    """An earlier graph may hold a leaf whose gradient the captured backward does not compute."""
    from rl_engine.ops.norm import gated_residual_norm

    def captured():
        x, w = _normal(4, 64, seed=1).requires_grad_(True), _normal(64, seed=2).requires_grad_(True)
        g = _normal(4, 64, seed=3)
        step = lambda: torch.autograd.grad(gated_residual_norm(x, x, w)[1], [x], g)[0]  # noqa: E731
        want = step()
        held = w * 2  # noqa: F841
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)

    captured()
    general(captured)


def test_a_leaf_of_the_default_stream_is_seen(general):
    """Outside of a capture such a backward runs, on the stream of its forward."""
    from rl_engine import _host

    x = _normal(4, 64, seed=1).requires_grad_(True)
    seen = []

    class Look(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 2

        @staticmethod
        def backward(ctx, g):
            seen.append(_host.native().reaches_default_stream())
            return g * 2

    held = Look.apply(x)  # noqa: F841
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            torch.autograd.grad(Look.apply(x).sum(), [x])
    assert seen == [False, True] and not _host.native().reaches_default_stream()
    call = _calls()["norm"]
    held = call(x)  # noqa: F841
    want = torch.autograd.grad(call(x).sum(), [x])[0]
    with torch.cuda.stream(side):
        got = torch.autograd.grad(call(x).sum(), [x])[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
