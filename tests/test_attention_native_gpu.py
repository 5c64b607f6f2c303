"""Rotary positions, appending and attention through the native host side against the general way: the same bits of results, caches and
gradients, and the general way for everything that is more than values in memory."""

from __future__ import annotations

import pytest
import torch

from attention_cases import DEV, Batch, same_bits

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


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


@pytest.fixture(scope="module")
def attention():
    from rl_engine.ops import attention

    return attention


@pytest.fixture(scope="module")
def native():
    from rl_engine import _host

    return _host.native()


def _normal(*shape, seed=0, dtype=BF16):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def _same(got, want):
    assert len(got) == len(want)
    for g, w in zip(got, want):
        assert (g is None) == (w is None)
        assert g is None or same_bits(g, w)


@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("leading", ((1,), (37,), (3, 5)))
@pytest.mark.parametrize("with_k", (False, True))
def test_rotary(attention, native, general, dtype, leading, with_k):
    q, k = _normal(*leading, 4, 48, seed=1, dtype=dtype), _normal(*leading, 2, 48, seed=2, dtype=dtype) if with_k else None
    if leading == (37,):
        q = _normal(4, *leading, 48, seed=3, dtype=dtype).transpose(0, 1)
    f = attention.rotary_frequencies(32, device=DEV)
    for positions in (torch.arange(q[..., 0, 0].numel(), device=DEV).view(leading) * 7, torch.full(leading, 100003, device=DEV, dtype=torch.int32)):
        for interleaved in (False, True):
            assert native.rotary(q, k, positions, f, interleaved, 0.7) is not None
            run = lambda: attention.rotary_embedding(q, k, positions, f, interleaved=interleaved, magnitude=0.7)  # noqa: B023, E731
            _same(run(), general(run))

            def gradients():
                leaves = [t.detach().clone().requires_grad_() for t in (q, k) if t is not None]
                out = [t for t in attention.rotary_embedding(leaves[0], leaves[1] if with_k else None, positions, f, interleaved=interleaved) if t is not None]  # noqa: B023
                sent = [_normal(*t.shape, seed=5 + i, dtype=dtype) for i, t in enumerate(out)]
                found = list(torch.autograd.grad(out, leaves, sent, retain_graph=True))
                if with_k:  # of one of them alone; repeated numbers; another order in memory
                    found += torch.autograd.grad(out[1], leaves, sent[1], retain_graph=True, allow_unused=True)
                found += torch.autograd.grad(out[0].sum(), leaves[:1], retain_graph=True)
                found += torch.autograd.grad(out[0], leaves[:1], sent[0].transpose(-1, -2).contiguous().transpose(-1, -2), retain_graph=True)
                (first,) = torch.autograd.grad((out[0].float() ** 2).sum(), leaves[:1], create_graph=True)
                return found + list(torch.autograd.grad(first.float().sum(), leaves[:1]))

            _same(gradients(), general(gradients))


def test_one_of_two_wants_a_gradient(attention):
    q, k, positions = _normal(9, 4, 32, seed=1), _normal(9, 2, 32, seed=2), torch.arange(9, device=DEV)
    f = attention.rotary_frequencies(32, device=DEV)
    for wants_q in (True, False):
        leaf = (q if wants_q else k).clone().requires_grad_()
        both = attention.rotary_embedding(leaf if wants_q else q, k if wants_q else leaf, positions, f)
        (sum(t.float().sum() for t in both)).backward()
        want = attention.rotary_embedding(torch.ones_like(leaf), None, -positions, f)[0]
        assert same_bits(leaf.grad, want)


@pytest.mark.parametrize("dtype", (BF16, FP16, FP32))
@pytest.mark.parametrize("order", ("rows", "heads", "pairs"))
def test_append(attention, native, general, dtype, order):
    f = attention.rotary_frequencies(64, device=DEV)

    def run(with_q, with_f, with_positions):
        b = Batch([(3, 20), (1, 33), (0, 5), (17, 17)], 4, 2, 64, 8, dtype, order=order)
        k, v = _normal(b.tokens, 2, 64, seed=8, dtype=dtype), _normal(b.tokens, 2, 64, seed=9, dtype=dtype)
        positions = torch.arange(b.tokens, device=DEV) * 3 if with_positions else None
        how = dict(q=b.q if with_q else None, positions=positions, interleaved=with_q)
        turned = attention.paged_append(k, v, *b.where, f if with_f else None, **how)
        return [turned, b.keys.contiguous(), b.values.contiguous()]

    b = Batch([(3, 20)], 4, 2, 64, 8, dtype, order=order)
    assert native.paged_append(b.q[:, :2], b.q[:, 2:], *b.where, f, b.q, None, False, 1.0) is not None
    for with_q, with_f, with_positions in ((True, True, False), (False, True, True), (True, False, False), (False, False, False)):
        _same(run(with_q, with_f, with_positions), general(lambda: run(with_q, with_f, with_positions)))  # noqa: B023


@pytest.mark.parametrize("dtype", (BF16, FP16))
@pytest.mark.parametrize("order", ("rows", "heads", "pairs"))
def test_attention(attention, native, general, dtype, order):
    b = Batch([(3, 700), (1, 33), (0, 5), (90, 90)], 8, 2, 72, 12, dtype, order=order, behind=2)
    assert native.paged_attention(b.q, *b.where, None, True, None, False) is not None
    for how in ({}, {"causal": False}, {"window": 40}, {"scale": 0.3, "return_lse": True}, {"window": 1, "return_lse": True}):
        run = lambda: attention.paged_attention(b.q, *b.where, **how)  # noqa: B023, E731
        got, want = run(), general(run)
        _same(got if "return_lse" in how else [got], want if "return_lse" in how else [want])


def test_what_is_not_everyday_goes_the_general_way(attention, native):
    b = Batch([(3, 20), (1, 33)], 4, 2, 64, 8, BF16)
    k, v, f = _normal(b.tokens, 2, 64, seed=8), _normal(b.tokens, 2, 64, seed=9), attention.rotary_frequencies(64, device=DEV)
    positions = torch.arange(b.tokens, device=DEV)
    asks = b.q.clone().requires_grad_()
    refused = (None, True, None, False)
    assert native.paged_attention(asks, *b.where, *refused) is None and native.paged_attention(b.q[:, :3], *b.where, *refused) is None
    assert native.paged_attention(b.q.float(), *b.where, *refused) is None and native.paged_attention(b.q[:0], *b.where, *refused) is None
    assert native.paged_attention(b.q, b.keys, b.values, b.table.long(), b.contexts, b.starts, *refused) is None
    assert native.paged_attention(b.q, b.keys, b.values, b.table, b.contexts, b.starts[:-1], *refused) is None
    assert native.paged_attention(b.q, b.keys, b.values[:-1], b.table, b.contexts, b.starts, *refused) is None
    assert native.paged_attention(b.q, *b.where, -1.0, True, None, False) is None and native.paged_attention(b.q, *b.where, None, False, 5, False) is None
    assert native.paged_attention(b.q, *b.where, None, True, 0, False) is None and native.paged_attention(b.q, *b.where, None, True, True, False) is None
    assert native.paged_append(k.clone().requires_grad_(), v, *b.where, f, None, None, False, 1.0) is None
    assert native.paged_append(k, v[:-1], *b.where, f, None, None, False, 1.0) is None and native.paged_append(k, v, *b.where, None, None, positions, False, 1.0) is None
    assert native.paged_append(k, v, *b.where, f.float(), None, None, False, 1.0) is None and native.paged_append(k, v, *b.where, f, b.q[:-1], None, False, 1.0) is None
    assert native.rotary(b.q, None, positions[:-1], f, False, 1.0) is None and native.rotary(b.q, None, positions.cpu(), f, False, 1.0) is None
    assert native.rotary(b.q, k[..., :32], positions, f, False, 1.0) is None and native.rotary(b.q, k.float(), positions, f, False, 1.0) is None
    assert native.rotary(b.q.double(), None, positions, f, False, 1.0) is None and native.rotary(b.q[..., :32], None, positions, f, False, 1.0) is None
    with pytest.raises(RuntimeError, match="gradient"):
        attention.paged_attention(asks, *b.where)
    with torch.no_grad():
        assert native.paged_attention(asks, *b.where, *refused) is not None
    seen = []

    class Mode(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return func(*args, **(kwargs or {}))

    with Mode():
        got = attention.rotary_embedding(b.q, None, positions, f)[0]
    assert seen and same_bits(got, attention.rotary_embedding(b.q, None, positions, f)[0])


def test_another_stream(attention):
    b = Batch([(3, 700), (1, 33)], 4, 2, 64, 16, BF16)
    want = attention.paged_attention(b.q, *b.where)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = attention.paged_attention(b.q, *b.where)
    stream.synchronize()
    assert same_bits(got, want)


def test_a_backward_is_not_captured_beside_an_eager_graph_of_its_leaves(attention):
    f, positions = attention.rotary_frequencies(32, device=DEV), torch.arange(9, device=DEV)
    leaf, sent = _normal(9, 4, 32, seed=1).requires_grad_(), _normal(9, 4, 32, seed=2)
    eager = attention.rotary_embedding(leaf, None, positions, f)[0]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="earlier calls"):
        with torch.cuda.graph(graph):
            attention.rotary_embedding(leaf, None, positions, f)[0].backward(sent)
    del eager
    leaf.grad = None
    torch.cuda.synchronize()
    other = _normal(9, 4, 32, seed=1).requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (grad,) = torch.autograd.grad(attention.rotary_embedding(other, None, positions, f)[0], other, sent)
    for i in range(3):
        sent.copy_(_normal(9, 4, 32, seed=20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert same_bits(grad, attention.rotary_embedding(sent, None, -positions, f)[0])
