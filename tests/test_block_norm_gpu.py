"""Norm, gate, residual sum and next norm on a real MI355X against their definitions in 64 bits.

Tolerances: a sum over a row is a chain of at most 16 products in a thread, 6 butterflies and 16 waves, under 40 roundings of 2^-24;
a value passes two such sums forward and two backward and about 20 products: 200 steps of 2^-24 of the sizes that were added up
to it (not of what cancellation left of them), then half a step of its type. Sums over rows add T of them."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0**-8, FP16: 2.0**-11, FP32: 2.0**-24}
STEPS = 200 * 2.0**-24
EPS, SCALE = 1e-5, 0.7


@pytest.fixture(scope="module")
def norm():
    from rl_engine.ops import norm

    return norm


def _normal(*shape, seed=0, dtype=BF16, scale=1.0, mean=0.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=DEV) * scale + mean).to(dtype)


def _near(got, want, size, name, dtype, extra=0):
    got = got.double()
    tiny = 2.0**-24 if dtype == FP16 else 2.0**-126
    bound = HALF_STEP[dtype] * want.abs() + (STEPS + extra * 2.0**-24) * size + tiny
    assert got.shape == want.shape and bool(((got - want).abs() <= bound).all()), (name, float(((got - want).abs() / bound).max()))


def _definition(block, residual, gate, post, pre, g_total, g_normed):
    """name -> (value, size of what was added up to it), in 64 bits, rows and widths as they are."""
    d = lambda t: None if t is None else t.double()  # noqa: E731
    x, r, gate, post, pre, gt, gn = (d(t) for t in (block, residual, gate, post, pre, g_total, g_normed))
    out = {}
    g = torch.ones((), dtype=torch.float64, device=DEV) if gate is None else gate
    if x is not None:
        r1 = 1 / (x.square().mean(1, keepdim=True) + EPS).sqrt() if post is not None else 1.0
        h1 = x * r1
        w1 = post if post is not None else 1.0
        u = h1 * w1
        total, total_size = r + SCALE * g * u, r.abs() + (SCALE * g * u).abs()
    else:
        total, total_size = r, r.abs()
    out["total"] = (total, total_size)
    r2 = 1 / (total.square().mean(1, keepdim=True) + EPS).sqrt()
    back, back_size = torch.zeros_like(r), torch.zeros_like(r)
    if gt is not None:
        back, back_size = gt, gt.abs()
    if pre is not None:
        out["normed"] = (total * r2 * pre, total_size * r2 * pre.abs())
        if gn is not None:
            h2, h2_size, a = total * r2, total_size * r2, gn * pre
            back = back + r2 * (a - h2 * (a * h2).mean(1, keepdim=True))
            back_size = back_size + r2 * (a.abs() + h2_size * (a.abs() * h2_size).mean(1, keepdim=True))
            out["d_pre"] = ((gn * h2).sum(0), (gn.abs() * h2_size).sum(0))
    out["d_residual"] = (back, back_size)
    if x is not None:
        du, du_size = SCALE * g * back, (SCALE * g).abs() * back_size
        if gate is not None:
            dg, dg_size = SCALE * u * back, (SCALE * u).abs() * back_size
            if gate.dim() == 1:
                dg, dg_size = dg.sum(0), dg_size.sum(0)
            elif gate.size(1) == 1 and x.size(1) > 1:
                dg, dg_size = dg.sum(1, keepdim=True), dg_size.sum(1, keepdim=True)
            out["d_gate"] = (dg, dg_size)
        if post is not None:
            out["d_post"] = ((du * h1).sum(0), (du_size * h1.abs()).sum(0))
            b, b_size = du * post, du_size * post.abs()
            du = r1 * (b - h1 * (b * h1).mean(1, keepdim=True))
            du_size = r1 * (b_size + h1.abs() * (b_size * h1.abs()).mean(1, keepdim=True))
        out["d_block"] = (du, du_size)
    return out


def _case(tokens, width, dtype, wide, gate_kind, post, pre, seed=0, weights=None):
    weights = dtype if weights is None else weights
    shape = {"none": None, "channel": (width,), "token": (tokens, 1), "full": (tokens, width)}[gate_kind]
    t = {
        "block": _normal(tokens, width, seed=seed, dtype=dtype, scale=3.0),
        "residual": _normal(tokens, width, seed=seed + 1, dtype=wide, scale=2.0),
        "gate": _normal(*shape, seed=seed + 2, dtype=weights) if shape else None,
        "post": _normal(width, seed=seed + 3, dtype=weights, mean=1.0, scale=0.2) if post else None,
        "pre": _normal(width, seed=seed + 4, dtype=weights, mean=1.0, scale=0.2) if pre else None,
    }
    if tokens > 2:
        with torch.no_grad():
            t["block"][2] = 0.0  # (its norm is eps alone)
    return t, _normal(tokens, width, seed=seed + 5, dtype=wide), _normal(tokens, width, seed=seed + 6, dtype=dtype) if pre else None


def _run(norm, t, g_total, g_normed):
    leaves = {k: v.requires_grad_(True) for k, v in t.items() if v is not None}
    total, normed = norm.gated_residual_norm(
        t["block"], t["residual"], t["pre"], post_weight=t["post"], gate=t["gate"], residual_scale=SCALE, eps=EPS
    )
    got = {"total": total.detach()} | ({} if normed is None else {"normed": normed.detach()})
    outputs = [(o, g) for o, g in ((total, g_total), (normed, g_normed)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in outputs], list(leaves.values()), [g for _, g in outputs])
    return got | {"d_" + k: g for k, g in zip(leaves, grads)}


def _compare(got, want, t, tokens):
    source = {"total": "residual", "normed": "block"}
    assert set(got) == set(want)
    for name, value in got.items():
        like = t[source.get(name, name[2:])]
        assert value.dtype == like.dtype and value.shape == like.shape, name
        _near(value, *want[name], name, value.dtype, tokens if name in ("d_pre", "d_post", "d_gate") else 0)


SIZES = [(1, 1), (3, 7), (5, 64), (2, 513), (700, 100), (33, 1024), (9, 1537), (600, 2048), (17, 4096), (5, 5000), (3, 8192), (2, 8195), (3, 16384)]


@pytest.mark.parametrize("dtype,wide", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP16, FP32), (FP32, FP32)])
@pytest.mark.parametrize("tokens,width", SIZES)
def test_results_and_gradients(norm, tokens, width, dtype, wide):
    kinds = ["none", "channel", "token", "full"]
    kind, post = kinds[(tokens + width) % 4], (tokens * 3 + width) % 3 > 0
    t, g_total, g_normed = _case(tokens, width, dtype, wide, kind, post, True, seed=width)
    want = _definition(*(t[k] for k in ("block", "residual", "gate", "post", "pre")), g_total, g_normed)
    _compare(_run(norm, t, g_total, g_normed), want, t, tokens)


@pytest.mark.parametrize("gate", ["channel", "token", "full"])
@pytest.mark.parametrize("wide", [BF16, FP32])
@pytest.mark.parametrize("tokens,width", [(40001, 6), (36005, 64), (17003, 128), (9001, 129), (8300, 256), (4200, 301), (2100, 1024), (1100, 2050), (700, 4096), (260, 8190), (259, 16384)])
def test_rows_that_take_turns(norm, tokens, width, wide, gate):
    """More rows than the workgroups of a backward take at a time, at both ends of every number of threads to a row."""
    t, g_total, g_normed = _case(tokens, width, BF16, wide, gate, True, True, seed=width)
    want = _definition(*(t[k] for k in ("block", "residual", "gate", "post", "pre")), g_total, g_normed)
    _compare(_run(norm, t, g_total, g_normed), want, t, tokens)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("weights", [BF16, FP32])
def test_every_combination(norm, gate, post, pre, weights):
    t, g_total, g_normed = _case(530, 260, BF16, BF16, gate, post, pre, weights=weights)
    want = _definition(*(t[k] for k in ("block", "residual", "gate", "post", "pre")), g_total, g_normed)
    _compare(_run(norm, t, g_total, g_normed), want, t, 530)


@pytest.mark.parametrize("only", ["total", "normed"])
@pytest.mark.parametrize("post", [False, True])
def test_a_gradient_of_one_output(norm, only, post):
    t, g_total, g_normed = _case(70, 640, BF16, FP32, "token", post, True)
    if only == "total":
        g_normed = None
    else:
        g_total = None
    leaves = {k: v.requires_grad_(True) for k, v in t.items() if v is not None and not (only == "total" and k == "pre")}
    total, normed = norm.gated_residual_norm(t["block"], t["residual"], t["pre"], post_weight=t["post"], gate=t["gate"], residual_scale=SCALE, eps=EPS)
    grads = torch.autograd.grad(total if only == "total" else normed, list(leaves.values()), g_total if only == "total" else g_normed)
    want = _definition(*(t[k] for k in ("block", "residual", "gate", "post", "pre")), g_total, g_normed)
    for (name, leaf), grad in zip(leaves.items(), grads):
        _near(grad, *want["d_" + name], name, leaf.dtype, 70)


def test_gradient_against_differences(norm):
    """Central differences of the definition in 64 bits with h = 1e-4, fp32 throughout. Third derivatives are of a few, so they
    leave 1e-8; but in row 2, whose block is zero, x / sqrt(x^2 / width + eps) = x / sqrt(eps) (1 - x^2 / (2 width eps) + ...), so
    the difference is h^2 / (2 width eps) = 2e-5 of the slope short, twice that with the same in the sum's norm behind it."""
    t, g_total, g_normed = _case(3, 24, FP32, FP32, "channel", True, True)
    got = _run(norm, t, g_total, g_normed)
    names = ("block", "residual", "gate", "post", "pre")
    base = {k: t[k].detach().double() for k in names}

    def loss(values):
        d = _definition(*(values[k] for k in names), None, None)
        return (d["total"][0] * g_total.double()).sum() + (d["normed"][0] * g_normed.double()).sum()

    for name in names:
        flat = base[name].reshape(-1)
        for at in (0, 5, flat.numel() - 1):
            ends = []
            for sign in (1, -1):
                moved = dict(base)
                moved[name] = flat.clone()
                moved[name][at] += sign * 1e-4
                moved[name] = moved[name].reshape(base[name].shape)
                ends.append(loss(moved))
            slope = float((ends[0] - ends[1]) / 2e-4)
            assert abs(slope - float(got["d_" + name].reshape(-1)[at])) < 1e-4 + abs(slope) * 1e-8 / (24 * EPS), (name, at)


@pytest.mark.parametrize("dtype,out", [(BF16, None), (FP16, None), (FP32, None), (FP32, BF16), (FP32, FP16)])
@pytest.mark.parametrize("shape", [(64,), (5, 1000), (2, 3, 4096)])
def test_rms_norm(norm, dtype, out, shape):
    x = _normal(*shape, seed=3, dtype=dtype, scale=2.0).requires_grad_(True)
    result = out or dtype
    weight = _normal(shape[-1], seed=4, dtype=result, mean=1.0, scale=0.2).requires_grad_(True)
    gy = _normal(*shape, seed=5, dtype=result)
    y = norm.rms_norm(x, weight, eps=EPS, dtype=out)
    grads = torch.autograd.grad(y, [x, weight], gy)
    rows = x.detach().reshape(-1, shape[-1])
    want = _definition(None, rows, None, None, weight.detach(), None, gy.reshape(-1, shape[-1]))
    assert y.dtype == result and y.shape == x.shape and grads[0].dtype == dtype
    _near(y.detach().reshape(rows.shape), *want["normed"], "normed", result)
    _near(grads[0].reshape(rows.shape), *want["d_residual"], "x", dtype)
    _near(grads[1], *want["d_pre"], "weight", result, rows.size(0))


def test_layouts(norm):
    t, g_total, g_normed = _case(6, 100, BF16, BF16, "full", True, True)
    want = norm.gated_residual_norm(t["block"], t["residual"], t["pre"], post_weight=t["post"], gate=t["gate"])
    wide = torch.full((6, 309), float("nan"), dtype=BF16, device=DEV)
    wide[:, 1:101], wide[:, 103:203], wide[:, 205:305] = t["block"], t["residual"], t["gate"]
    pre = torch.stack([t["pre"], t["pre"]], 1)[:, 1]
    for args in (
        (wide[:, 1:101], wide[:, 103:203], wide[:, 205:305]),
        (t["block"].t().contiguous().t(), t["residual"].t().contiguous().t(), t["gate"].t().contiguous().t()),
        (t["block"].view(2, 3, 100), t["residual"].view(2, 3, 100), t["gate"].view(2, 3, 100)),
    ):
        got = norm.gated_residual_norm(args[0], args[1], pre, post_weight=t["post"], gate=args[2])
        for g, w in zip(got, want):
            assert g.shape == args[0].shape and torch.equal(g.reshape(6, 100), w)
    row = t["block"][:1].expand(6, 100)
    a = norm.gated_residual_norm(row, t["residual"], t["pre"], gate=t["gate"][:, :1].expand(6, 1))
    b = norm.gated_residual_norm(row.contiguous(), t["residual"], t["pre"], gate=t["gate"][:, :1].contiguous())
    assert torch.equal(a[1], b[1])
    one = norm.rms_norm(t["block"][0].expand(1, 100), t["pre"])
    assert torch.equal(one[0], norm.rms_norm(t["block"], t["pre"])[0])


@pytest.mark.parametrize("width", [20, 130, 384, 1000])
def test_a_row_does_not_depend_on_its_batch(norm, width):
    t, g_total, g_normed = _case(3000, width, BF16, BF16, "token", True, True)
    whole = _run(norm, t, g_total, g_normed)
    for rows in (slice(0, 1), slice(2999, 3000), slice(1000, 1077)):
        some = {k: (v if v is None or v.dim() == 1 else v.detach()[rows]) for k, v in t.items()}
        part = _run(norm, some, g_total[rows], g_normed[rows])
        for name in ("total", "normed", "d_block", "d_residual", "d_gate"):
            assert torch.equal(part[name], whole[name][rows]), name
    again = _run(norm, t, g_total, g_normed)
    for name, value in whole.items():
        assert torch.equal(value, again[name]), name


def test_in_a_graph_and_on_another_stream(norm):
    t, g_total, g_normed = _case(130, 700, BF16, FP32, "channel", True, True)

    def step():
        return list(_run(norm, t, g_total, g_normed).values())

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
            t["block"].copy_(_normal(130, 700, seed=50 + seed))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_no_tokens(norm):
    t, g_total, g_normed = _case(0, 64, BF16, BF16, "channel", True, True)
    got = _run(norm, t, g_total, g_normed)
    assert got["total"].shape == (0, 64) and not any(bool(got[k].any()) for k in ("d_pre", "d_post", "d_gate"))


def test_more_rows_than_one_launch_has():
    """A launch of the forward has fewer than 2^32 threads, 64 to a row of up to 512 columns."""
    from rl_engine.ops.norm import rms_norm

    rows = 2**31 // 64 + 5
    x = torch.ones((rows, 8), dtype=BF16, device=DEV)
    x[-7:] = _normal(7, 8, seed=1)
    w = _normal(8, seed=2)
    got = rms_norm(x, w)
    assert torch.equal(got[-7:], rms_norm(x[-7:].clone(), w)) and bool((got[:-7] == got[0]).all())


def test_infinities_stay_in_their_rows(norm):
    t, *_ = _case(4, 128, BF16, BF16, "none", True, True)
    clean = norm.gated_residual_norm(t["block"], t["residual"], t["pre"], post_weight=t["post"])
    t["block"][1, 5], t["residual"][3, 7] = float("nan"), float("inf")
    got = norm.gated_residual_norm(t["block"], t["residual"], t["pre"], post_weight=t["post"])
    for g, c in zip(got, clean):
        assert torch.equal(g[[0, 2]], c[[0, 2]])
    assert bool(torch.isnan(got[1][1]).all()) and bool(torch.isnan(got[1][3, 7]))


def test_refused_calls(norm):
    x, w = _normal(4, 64), _normal(64)
    call = norm.gated_residual_norm
    for args, kwargs, error in (
        ((x, x[:2], w), {}, ValueError), ((x, x, w[:3]), {}, ValueError), ((x, x, w), {"gate": _normal(4, 2)}, ValueError),
        ((x, x, w), {"gate": _normal(4)}, ValueError), ((x, x, w), {"post_weight": w[:5]}, ValueError), ((x, x.half(), w), {}, TypeError),
        ((x.float(), x, w.float()), {}, TypeError), ((x, x, w.half()), {}, TypeError), ((x.double(), x.double(), w.double()), {}, TypeError),
        ((x.cpu(), x.cpu(), w.cpu()), {}, RuntimeError), ((x, x.cpu(), w), {}, RuntimeError), ((x, x, w.cpu()), {}, RuntimeError),
        ((_normal(2, 16385),) * 2, {}, ValueError), ((x, x, w), {"gate": 0.5}, TypeError),
    ):  # fmt: skip
        with pytest.raises(error):
            call(*args, **kwargs)
    for eps in (-1e-6, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            call(x, x, w, eps=eps)
        with pytest.raises(ValueError, match="eps"):
            norm.rms_norm(x, w, eps=eps)
    for args, kwargs in (((x, None), {}), ((x, w), {"dtype": FP32}), ((x.half(), w), {})):
        with pytest.raises(TypeError):
            norm.rms_norm(*args, **kwargs)
