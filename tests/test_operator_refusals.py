"""What the token scores, the norm between blocks and the eight-bit copies refuse, before anything reaches a GPU: the C entries on
calls that are wrong, the native host side on what is not everyday, the entry points on CPU tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

BF16 = torch.bfloat16
AT = 1 << 20  # an address that nothing reads: these calls are refused


def _refused(rlk_lib, status, words):
    text = rlk_lib.rlk_last_error().decode()
    assert status != 0 and words in text, (status, text)


def _scores(rlk_lib, *, logits=AT, dtype=0, stride=100, target=AT, rows=4, vocab=100, real=100, top_k=0, logp=AT, entropy=AT, top=None,
            ids=None, workspace=AT, size=1 << 30):  # fmt: skip
    return rlk_lib.rlk_logits_scores(logits, dtype, stride, target, None, rows, vocab, real, top_k, logp, AT, entropy, top, ids, workspace, size, None)


def test_scores_of_logits(rlk_lib):
    from rl_engine import _lib

    rows = 2**24 - 1
    for kwargs, words in (
        ({"vocab": (1 << 28) + 1, "stride": 1 << 30}, "V at most"), ({"real": 101}, "real_vocab"), ({"top_k": 65}, "top_k"), ({"top_k": -1}, "top_k"),
        ({"top_k": 8, "real": 7}, "top_k"), ({"top_k": 3}, "null"), ({"target": None}, "null"), ({"entropy": None}, "null"),
        ({"size": 4 * 1024 - 1}, "workspace"), ({"workspace": None}, "workspace"), ({"workspace": AT + 4}, "workspace"), ({"rows": rows + 1}, "rows"),
        ({"stride": 99}, ""), ({"dtype": 9}, ""), ({"rows": -1}, ""), ({"real": 0}, ""), ({"logits": None}, ""),
    ):  # fmt: skip
        _refused(rlk_lib, _scores(rlk_lib, **kwargs), words)
    assert rlk_lib.rlk_logits_scores_workspace_bytes(4, 0) == 4 * 1024 and rlk_lib.rlk_logits_scores_workspace_bytes(0, 5) == 0
    assert _scores(rlk_lib, rows=0, logits=None, target=None, workspace=None) == 0
    assert (_lib.SCORES_MAX_TOP_K, _lib.SCORES_MAX_VOCAB) == (64, 1 << 28)


def test_gradient_of_scores(rlk_lib):
    def call(*, dtype=0, lse=AT, entropy=AT, g_entropy=None, ids=None, g_top=None, top_k=0, grad=AT, grad_dtype=0, stride=100, cols=100, rows=4, target=AT, g_logp=AT):
        return rlk_lib.rlk_logits_scores_backward(
            AT, dtype, 100, target, None, lse, entropy, g_logp, None, g_entropy, ids, g_top, top_k, grad, grad_dtype, stride, cols, rows, 100, 100, None
        )

    for kwargs, words in (
        ({"grad_dtype": 2}, "type"), ({"lse": None}, "null"), ({"grad": None}, "null"), ({"target": None}, "null"), ({"entropy": None, "g_entropy": AT}, "null"),
        ({"g_top": AT, "top_k": 3}, "null"), ({"cols": 99}, "grad_cols"), ({"stride": 99}, "grad_cols"), ({"g_top": AT, "ids": AT, "top_k": 65}, "top_k"),
        ({"rows": 1 << 24}, "rows"),
    ):  # fmt: skip
        _refused(rlk_lib, call(**kwargs), words)
    assert call(rows=0, lse=None, grad=None) == 0


def test_scores_of_hidden_states(rlk_lib):
    def call(*, rows=4, hidden=64, vocab=100, real=100, top_k=0, logp=AT, top=None, logits=AT, stride=128, workspace=AT, size=1 << 30, bias=None):
        return rlk_lib.rlk_linear_scores_fwd(
            AT, hidden, AT, hidden, AT, bias, None, logp, AT, AT, top, top, logits, stride, workspace, size, rows, hidden, vocab, real, top_k, None
        )

    for kwargs, words in (
        ({"top_k": 65, "top": AT}, "top_k"), ({"top_k": 2}, "null output"), ({"logp": None}, "null output"), ({"logits": None}, "needs logits"),
        ({"logits": AT + 4}, "aligned"), ({"stride": 127}, "aligned"), ({"stride": 130}, "aligned"), ({"size": 16}, "workspace"),
        ({"workspace": None}, "workspace"), ({"workspace": AT + 8}, "workspace"), ({"rows": 1 << 24}, "rows"), ({"rows": -1}, ""),
        ({"vocab": (1 << 28) + 1}, "columns"), ({"top_k": 5, "real": 4, "top": AT}, "top_k"),
    ):  # fmt: skip
        _refused(rlk_lib, call(**kwargs), words)
    assert rlk_lib.rlk_linear_scores_workspace_bytes(0, 100, 0) == 0
    # logits or none: never none with alternatives or a bias
    for bias, top_k in ((0, 3), (1, 0)):
        assert rlk_lib.rlk_linear_scores_needs_logits(AT, 64, AT, 64, bias, 4096, 64, 4096, top_k) == 1


def test_gradients_of_the_projection(rlk_lib):
    def call(*, dz=AT, hidden=AT, stride=64, rows=4, out=AT):
        return rlk_lib.rlk_linear_dlogits_bwd(dz, hidden, stride, AT, 64, out, stride, None, 64, rows, 64, 100, None)

    for kwargs, words in (({"dz": None}, "null"), ({"dz": AT + 64}, "unaligned"), ({"hidden": None}, "null"), ({"stride": 63}, "stride"), ({"rows": 0}, "positive")):
        _refused(rlk_lib, call(**kwargs), words)
    assert rlk_lib.rlk_linear_dlogits_row_stride(0) == 0 and rlk_lib.rlk_linear_dlogits_row_stride(100) >= 100


def _norm(**kwargs):
    from rl_engine import _lib

    fields = {"block": AT, "residual": AT, "gate": None, "post_weight": None, "pre_weight": AT, "rstd": AT, "block_row_stride": 64, "residual_row_stride": 64,
              "gate_row_stride": 0, "tokens": 4, "width": 64, "dtype": 0, "residual_dtype": 0, "gate_kind": 0, "gate_dtype": 0, "post_dtype": 0, "pre_dtype": 0,
              "eps": 1e-6, "residual_scale": 1.0, **kwargs}  # fmt: skip
    return ctypes.byref(_lib.BlockNorm(*(fields[name] for name, _ in _lib.BlockNorm._fields_)))


def test_norm_between_blocks(rlk_lib):
    fp32 = 2
    for kwargs, words in (
        ({"width": 0}, "width"), ({"width": 16385}, "width"), ({"tokens": -1}, "tokens"), ({"dtype": 9}, "type"), ({"residual_dtype": 1}, "type"),
        ({"dtype": fp32, "residual_dtype": 0}, "type"), ({"gate_kind": 4}, "gate kind"), ({"gate_kind": 1}, "null"), ({"residual": None}, "null"),
        ({"residual_row_stride": 63}, "stride"), ({"block_row_stride": 63}, "stride"), ({"gate_kind": 3, "gate": AT, "gate_row_stride": 63}, "stride"),
        ({"block": None, "gate_kind": 1, "gate": AT}, "without a block"), ({"block": None, "post_weight": AT}, "without a block"),
        ({"pre_weight": None}, "goes with"), ({"eps": -1e-6}, "eps"), ({"eps": float("nan")}, "eps"),
    ):  # fmt: skip
        _refused(rlk_lib, rlk_lib.rlk_block_norm_forward(_norm(**kwargs), AT, AT, None), words)
    _refused(rlk_lib, rlk_lib.rlk_block_norm_forward(None, AT, AT, None), "null")
    _refused(rlk_lib, rlk_lib.rlk_block_norm_forward(_norm(), AT, None, None), "goes with")
    assert rlk_lib.rlk_block_norm_forward(_norm(tokens=0, residual=None), None, AT, None) == 0


def test_gradients_of_the_norm(rlk_lib):
    def call(n, *, d_block=AT, d_gate=None, d_post=None, d_pre=None, workspace=AT, size=1 << 30):
        return rlk_lib.rlk_block_norm_backward(n, AT, AT, d_block, AT, d_gate, d_post, d_pre, workspace, size, None)

    for n, kwargs, words in (
        (_norm(), {"d_gate": AT}, "not there"), (_norm(), {"d_post": AT}, "not there"), (_norm(pre_weight=None), {"d_pre": AT}, "not there"),
        (_norm(block=None), {}, "not there"), (_norm(rstd=None), {}, "rstd"), (_norm(), {"workspace": None}, "workspace"), (_norm(), {"size": 8}, "workspace"),
        (_norm(), {"workspace": AT + 2}, "workspace"),
    ):  # fmt: skip
        _refused(rlk_lib, call(n, **kwargs), words)
    assert rlk_lib.rlk_block_norm_workspace_bytes(0, 64) == 0 and rlk_lib.rlk_block_norm_workspace_bytes(7, 0) == 0


def test_eight_bit_copies(rlk_lib):
    for args, words in (
        ((AT, 63, 0, AT, AT, 4, 64, None), "stride"), ((None, 64, 0, AT, AT, 4, 64, None), "null"), ((AT, 64, 0, None, AT, 4, 64, None), "null"),
        ((AT, 64, 0, AT, None, 4, 64, None), "null"), ((AT, 64, 7, AT, AT, 4, 64, None), "dtype"), ((AT, 64, 0, AT, AT, -1, 64, None), "sizes"),
        ((AT, 1 << 29, 0, AT, AT, 1, (1 << 28) + 1, None), "sizes"),
    ):  # fmt: skip
        _refused(rlk_lib, rlk_lib.rlk_mx8_encode(*args), words)
    for args, words in (((None, AT, AT, 64, 0, 4, 64, None), "null"), ((AT, AT, AT, 63, 0, 4, 64, None), "stride"), ((AT, AT, AT, 64, 5, 4, 64, None), "dtype")):
        _refused(rlk_lib, rlk_lib.rlk_mx8_decode(*args), words)
    for missing in range(7):
        addresses = [None if i == missing else AT for i in range(7)]
        gate, up, y, *kept = addresses
        _refused(rlk_lib, rlk_lib.rlk_mx8_swiglu_forward(gate, 64, up, 64, 0, y, *kept, 4, 64, None), "null")
        dy, *kept, d_gate, d_up = addresses
        _refused(rlk_lib, rlk_lib.rlk_mx8_swiglu_backward(dy, 64, 0, *kept, d_gate, d_up, None, 4, 64, None), "null")
    assert rlk_lib.rlk_mx8_encode(None, 0, 0, None, None, 0, 64, None) == 0 and rlk_lib.rlk_mx8_decode(None, None, None, 0, 0, 4, 0, None) == 0


def test_cpu_tensors_are_not_everyday(rlk_lib):
    from rl_engine import _host

    native = _host.native()
    x, ids = torch.zeros(4, 64, dtype=BF16), torch.zeros(4, dtype=torch.long)
    logits = torch.zeros(4, 64)
    assert native.scores(x, ids, None, 64, 0) is None and native.scores(x, None, None, 64, 0) is None and native.scores(x) is None
    assert native.scores(x, ids, 0.5, 64, "3") is None
    assert native.linear_scores(x, x, ids, None, 64, 0, logits) is None and native.linear_scores(x, x, ids) is None
    assert native.norm(x, x, None, None, x[0], 1e-6, 1.0) is None and native.norm(None, x, None, None, x[0], 1e-6, 1.0) is None
    assert native.norm(x, x, None, None, x[0], "1e-6", 1.0) is None and native.norm(x) is None
    assert native.mx8_swiglu(x, x) is None and native.mx8_swiglu(x) is None and native.mx8_encode(x) is None and native.mx8_encode(3) is None
    assert native.reaches_default_stream() is False


def test_the_entry_points_word_their_errors():
    from rl_engine.ops.ffn import checkpointed_swiglu, mx8_decode, mx8_encode, qwen3_ffn
    from rl_engine.ops.logprob import deterministic_linear_scores, deterministic_scores_from_logits
    from rl_engine.ops.norm import gated_residual_norm, rms_norm

    x, ids = torch.zeros(4, 64, dtype=BF16), torch.zeros(4, dtype=torch.long)
    with pytest.raises(RuntimeError, match="require a GPU tensor"):
        deterministic_scores_from_logits(x, ids)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        deterministic_scores_from_logits(x.double(), ids)
    with pytest.raises(ValueError, match="at least two dimensions"):
        deterministic_scores_from_logits(x[0], ids)
    with pytest.raises(ValueError, match="must match target_ids"):
        deterministic_linear_scores(x, x, ids[:3])
    with pytest.raises(RuntimeError, match="bias.detach"):
        deterministic_linear_scores(x, x, ids, torch.zeros(64, requires_grad=True))
    for bad in (lambda: gated_residual_norm(x, x, x[0]), lambda: rms_norm(x, x[0])):
        with pytest.raises(RuntimeError, match="must be on a CUDA/ROCm GPU"):
            bad()
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        gated_residual_norm(None, x)
    with pytest.raises(ValueError, match="share shape"):
        checkpointed_swiglu(x, x[:2])
    with pytest.raises(TypeError, match="torch.Tensors"):
        checkpointed_swiglu(x, None)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        mx8_encode(x)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        mx8_decode(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8))
    with pytest.raises(ValueError, match="checkpoint_bits"):
        qwen3_ffn(x, x, x, x, checkpoint_bits=4)


def test_division_of_a_piece_by_the_pieces_of_a_row():
    """The product that stands for n / d in the kernels of the eight-bit copies (n < 2^31, d even, up to 2^24), at the ends of the
    quotients and at random."""
    gen = torch.Generator().manual_seed(0)
    divisors = [2, 4, 6, 10, 62, 64, 66, 254, 256, 258, 768, 9496, 2**23 - 2, 2**23, 2**23 + 2, 2**24 - 2, 2**24]
    divisors += (torch.randint(1, 2**23, (200,), generator=gen) * 2).tolist()
    for d in divisors:
        shift = 0
        while (1 << shift) < d:
            shift += 1
        factor = ((1 << 32) * ((1 << shift) - d)) // d + 1
        assert factor < 2**32
        quotients = torch.randint(0, 2**31 // d + 1, (100,), generator=gen).tolist() + [1, 2, (2**31 - 1) // d]
        for n in {m for q in quotients for m in (q * d - 1, q * d, q * d + 1)} | {0, 2**31 - 1}:
            if not 0 <= n < 2**31:
                continue
            total = ((n * factor) >> 32) + n
            assert total < 2**32 and total >> shift == n // d, (n, d)


def test_parts_of_the_tokens_fit_their_buffer(rlk_lib):
    from rl_engine import _C
    from rl_engine.backends.rocm.logprob import token_scores

    for tokens, vocab in ((1, 151936), (3328, 151936), (3329, 151936), (70000, 1000), (5, 1 << 28), (300, 1 << 23), (0, 100), (1000, 9_000_000)):
        parts = token_scores._token_chunks(tokens, vocab)
        per_row = 4 * _C.linear_logp_logits_row_stride(vocab)
        assert [r for first, end in parts for r in range(first, end)] == list(range(tokens))
        assert all((end - first) * per_row <= token_scores._LOGITS_BUFFER_BYTES or end - first == 1 for first, end in parts)
        assert all(first % 256 == 0 for first, _ in parts) or token_scores._LOGITS_BUFFER_BYTES // per_row < 256
    assert len(token_scores._token_chunks(3328, 151936)) == 1 and len(token_scores._token_chunks(3329, 151936)) == 2


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("differentiated", [False, True])
def test_bits_of_a_block(fused, differentiated):
    """The packed way of an inference call looks at them as well."""
    from rl_engine.ops.ffn import qwen3_ffn_block

    x = torch.zeros(64, 64, dtype=BF16)
    for bits in (4, 16, True, "8"):
        with torch.set_grad_enabled(differentiated), pytest.raises(ValueError, match="checkpoint_bits"):
            qwen3_ffn_block(x, x, x, x, x, fused_gate_up_weight=torch.zeros(128, 64, dtype=BF16) if fused else None, checkpoint_bits=bits)
