"""Routing, expert order, dispatch and combine (torch_api) against plain 64-bit implementations.

No reference counterpart.  Scores and weights: a float32 exponential, sum and quotient, a few
2^-24 each, so 2e-6 of the weight; a choice by score + bias may go either way where two choices
lie within 1e-6 (scores are at most 1), and nowhere else.  Gradients: differences of terms of at
most scale * |g| rounded in float32, so 4e-6 of that, plus one rounding of the output's type.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import batch_topk_b200 as bt
import lm_reference as ref
from batch_topk_b200 import torch_api as api

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
HALF_ULP = {"fp16": 2.0**-11, "bf16": 2.0**-8, "fp32": 2.0**-23}
INVALID = bt.CUDA_ERROR_INVALID_VALUE
FAKE = 1 << 20


def rand(*shape, seed, dtype="fp32", scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(DTYPES[dtype])


def check_route(x, weights, experts, k, score="softmax", bias=None, groups=1, topk_groups=1,
                renormalize=True, scale=1.0):
    xs, w, e = x.detach().float().cpu().numpy(), weights.detach().cpu().numpy(), experts.cpu().numpy()
    b = None if bias is None else bias.cpu().numpy()
    assert w.shape == e.shape == (xs.shape[0], k)
    for t in range(xs.shape[0]):
        c, want_e, want_w, s = ref.route_row(xs[t], k, score, b, groups, topk_groups, renormalize,
                                             scale)
        if not np.array_equal(e[t], want_e):
            assert bias is not None, (t, e[t], want_e)  # logits are compared as they are
            got_c, want_c = c[e[t]], c[want_e]
            assert len(set(e[t])) == k and np.abs(got_c - want_c).max() <= 1e-6, (t, e[t], want_e)
            sel = s[e[t]]
            want_w = scale * (sel / (sel.sum() + 1e-20) if renormalize else sel)
        assert np.abs(w[t] - want_w).max() <= 2e-6 * scale, (t, w[t], want_w)


CASES = [
    dict(k=1),
    dict(k=2, renormalize=False),
    dict(k=8, score="sigmoid", scale=2.5),
    dict(k=6, groups=4, topk_groups=2),
    dict(k=6, score="sigmoid", groups=4, topk_groups=3, bias=True),
    dict(k=4, score="sigmoid", bias=True, renormalize=False),
    dict(k=3, score="softmax", bias=True),
    dict(k=5, score="sigmoid", groups=2, topk_groups=1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,experts", [(1, 8), (33, 8), (5, 16), (129, 64), (70, 100),
                                            (19, 160), (257, 256), (3, 260), (40, 512), (9, 1024)])
def test_route(dtype, tokens, experts):
    x = rand(tokens, experts, seed=experts + tokens, dtype=dtype, scale=1.5)
    for i, kw in enumerate(CASES):
        kw = dict(kw)
        if kw["k"] > experts // kw.get("groups", 1) * kw.get("topk_groups", 1):
            continue
        if kw.get("bias"):
            kw["bias"] = rand(experts, seed=i, scale=0.1)
        weights, chosen = api.route(x, **kw)
        check_route(x, weights, chosen, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_go_to_the_lower_index(score):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(-1, 2, (50, 96), generator=g, device="cuda").float()
    x[0] = 0.0
    x[1] = -0.0
    x[1, ::2] = 0.0
    for kw in (dict(k=8), dict(k=6, groups=8, topk_groups=3), dict(k=32)):
        weights, chosen = api.route(x, score=score, **kw)
        check_route(x, weights, chosen, score=score, **kw)
    weights, chosen = api.route(x, 4, score=score, bias=torch.zeros(96, device="cuda"))
    check_route(x, weights, chosen, 4, score=score, bias=torch.zeros(96, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_closed_experts(score, with_bias):
    """-inf and NaN logits and biases close an expert; slots that stay empty hold -1 and 0."""
    inf, nan = float("inf"), float("nan")
    x = rand(10, 64, seed=4)
    x[0] = -inf
    x[1] = nan
    x[2, 3:] = -inf
    x[3, ::2] = nan
    x[4, 5] = inf
    x[5, 7:9] = inf
    x[6] = -1e30
    x[7, 8:] = -inf
    x[8] = 200.0
    bias = None
    if with_bias:
        bias = rand(64, seed=5, scale=0.1)
        bias[1] = -inf
        bias[2] = nan
    for kw in (dict(k=4), dict(k=8, groups=8, topk_groups=2), dict(k=3, renormalize=False)):
        weights, chosen = api.route(x, score=score, bias=bias, **kw)
        check_route(x, weights, chosen, score=score, bias=bias, **kw)
        if not with_bias:
            assert (chosen[0] == -1).all() and (weights[0] == 0).all()


MANY = [  # experts and settings; at least 32 tokens an expert, a warp takes several tokens
    (5, dict(k=2)), (8, dict(k=4)), (8, dict(k=8)), (16, dict(k=8, score="sigmoid")),
    (24, dict(k=3, score="sigmoid", bias=True)), (33, dict(k=5, renormalize=False)),
    (40, dict(k=4, groups=8, topk_groups=5)), (60, dict(k=8, groups=12, topk_groups=9)),
    (64, dict(k=6, score="sigmoid", groups=8, topk_groups=3, bias=True)),
    (64, dict(k=8, groups=32, topk_groups=20)),
    (96, dict(k=4, score="softmax", bias=True)), (128, dict(k=1, score="sigmoid", scale=0.5)),
    (128, dict(k=4, score="sigmoid", groups=4, topk_groups=1)),
    (200, dict(k=8, score="sigmoid", bias=True)), (256, dict(k=7)),
    (256, dict(k=8, score="sigmoid", groups=8, topk_groups=4, bias=True, scale=2.5)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("experts,kw", MANY)
def test_route_many_tokens(dtype, experts, kw):
    """Ordinary rows next to rows of ties, closed experts and infinities, which need other paths
    than their neighbours; every row like the same row in a small call."""
    inf = float("inf")
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = rand(experts, seed=experts, scale=0.1)
    tokens = 32 * experts + 37
    x = rand(tokens, experts, seed=experts, dtype=dtype, scale=1.5)
    x[1::11] = x[1::11].round()
    x[3::13] = 0.5
    x[4::17, 1:] = -inf
    x[5::19] = -inf
    x[6::23, ::2] = float("nan")
    x[7::29, 2] = inf
    x[8::31, :3] = inf
    x[9::37] = 200.0
    weights, chosen = api.route(x, **kw)
    rows = torch.cat([torch.arange(30), torch.arange(tokens - 10, tokens)]).cuda()
    check_route(x[rows], weights[rows], chosen[rows], **kw)
    for t in range(0, tokens, 32 * experts // 3):
        part_w, part_e = api.route(x[t:t + 32], **kw)
        assert torch.equal(chosen[t:t + 32], part_e)
        # each within 2e-6 of the definition
        assert (weights[t:t + 32] - part_w).abs().max() <= 4e-6 * kw.get("scale", 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("experts,k", [(5, 2), (8, 8), (40, 4), (64, 8), (100, 10), (128, 6),
                                       (128, 16), (200, 9), (256, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_gradient_many_tokens(dtype, experts, k, score):
    tokens = 32 * experts + 5
    x = rand(tokens, experts, seed=experts, dtype=dtype, scale=2.0)
    x[0, 1] = float("-inf")
    x[tokens - 2] = float("-inf")
    x.requires_grad_()
    weights, chosen = api.route(x, k, score=score, scale=2.0)
    g = rand(tokens, k, seed=9)
    dx, = torch.autograd.grad(weights, x, g)
    xs, e, gs = x.detach().float().cpu().numpy(), chosen.cpu().numpy(), g.cpu().numpy()
    for t in [*range(12), *range(tokens - 8, tokens)]:
        if t == tokens - 2:
            assert (dx[t] == 0).all()
            continue
        want = ref.route_grad_row(xs[t], e[t], gs[t], score, True, 2.0)
        tol = 8e-6 * np.abs(gs[t]).max() + HALF_ULP[dtype] * np.abs(want) + 1e-7
        assert (np.abs(dx[t].float().cpu().numpy() - want) <= tol).all(), t


@pytest.mark.gpu
def test_route_strides_and_no_tokens():
    big = rand(20, 131, seed=6)
    for x in (big[:, 1:129], big[::3, 3:131], big.t().contiguous().t()[:, :128]):
        weights, chosen = api.route(x, 8, score="sigmoid")
        check_route(x, weights, chosen, 8, score="sigmoid")
    weights, chosen = api.route(big[:0, :128], 8)
    assert weights.shape == chosen.shape == (0, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,experts", [(1, 8), (37, 64), (20, 100), (65, 256), (5, 1024)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_gradient_formula(dtype, tokens, experts, score, renormalize):
    x = rand(tokens, experts, seed=experts, dtype=dtype, scale=2.0)
    x[0, 1] = float("-inf")
    x.requires_grad_()
    k = min(6, experts)
    weights, chosen = api.route(x, k, score=score, renormalize=renormalize, scale=2.0)
    g = rand(tokens, k, seed=9)
    dx, = torch.autograd.grad(weights, x, g)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    xs, e, gs = x.detach().float().cpu().numpy(), chosen.cpu().numpy(), g.cpu().numpy()
    for t in range(tokens):
        want = ref.route_grad_row(xs[t], e[t], gs[t], score, renormalize, 2.0)
        tol = 8e-6 * np.abs(gs[t]).max() + HALF_ULP[dtype] * np.abs(want) + 1e-7
        assert (np.abs(dx[t].float().cpu().numpy() - want) <= tol).all(), t


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_gradient_differences(score, renormalize):
    """Central differences of sum(g * weights): the step of 1/64 leaves an error of its square
    times a third derivative below 4, and 2^-22 over the step: 2e-3 bounds both."""
    x = rand(3, 24, seed=21).requires_grad_()
    g = rand(3, 4, seed=22)
    kw = dict(score=score, renormalize=renormalize)
    weights, chosen = api.route(x, 4, **kw)
    dx, = torch.autograd.grad(weights, x, g)
    h = 1.0 / 64

    def value(xv):  # the chosen experts stay those of x: the choice has no gradient
        w = torch.zeros_like(g)
        for t in range(3):
            _, _, _, s = ref.route_row(xv[t].cpu().numpy(), 4, score, None, 1, 1, False, 1.0)
            sel = s[chosen[t].cpu().numpy()]
            w[t] = torch.from_numpy(sel / (sel.sum() + 1e-20) if renormalize else sel)
        return (w * g).sum(1)

    for e in range(24):
        step = torch.zeros_like(g[:1, :1]).expand(3, 24).clone()
        step[:, e] = h
        got = (value(x.detach() + step) - value(x.detach() - step)) / (2 * h)
        assert (got - dx[:, e]).abs().max() <= 2e-3, e


@pytest.mark.gpu
def test_route_gradient_of_empty_slots():
    x = rand(4, 16, seed=23)
    x[0] = float("-inf")
    x[1, 2:] = float("-inf")
    x.requires_grad_()
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            weights, chosen = api.route(x, 4, score=score, renormalize=renorm)
            dx, = torch.autograd.grad(weights, x, rand(4, 4, seed=24))
            assert torch.isfinite(dx).all() and (dx[0] == 0).all() and (dx[1, 2:] == 0).all()


def make_experts(tokens, k, num, seed, popular=False):
    r = np.random.default_rng(seed)
    if popular:
        e = np.minimum(r.geometric(0.3, (tokens, k)) - 1, num - 1)
    else:
        e = r.integers(0, num, (tokens, k))
    e[r.random((tokens, k)) < 0.05] = -1
    return torch.from_numpy(e.astype(np.int32)).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,k,num", [(1, 1, 1), (1, 8, 256), (3, 2, 5), (31, 1, 1024),
                                          (33, 8, 64), (1000, 6, 160), (4099, 8, 256),
                                          (40000, 4, 1024), (65521, 8, 8), (100003, 7, 511),
                                          (1400003, 6, 33)])
@pytest.mark.parametrize("popular", [False, True])
def test_expert_order(tokens, k, num, popular):
    e = make_experts(tokens, k, num, tokens + num, popular)
    plan = api.expert_order(e, num)
    offsets, order, position = ref.order(e.cpu().numpy(), num)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    assert np.array_equal(plan.order.cpu().numpy(), order)
    assert np.array_equal(plan.position.cpu().numpy(), position)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,k,num", [(1100003, 3, 1000), (9000001, 1, 2), (590001, 1, 256),
                                          (589824, 1, 64)])
def test_expert_order_long(tokens, k, num):
    """Runs of several tiles, and lengths about a block's smallest run times the blocks."""
    test_expert_order(tokens, k, num, False)


@pytest.mark.gpu
def test_expert_order_numbers_out_of_range_and_extremes():
    e = torch.tensor([[5, -7], [2**31 - 1, 0], [-2**31, 5], [6, 3]], dtype=torch.int32, device="cuda")
    plan = api.expert_order(e, 6)
    offsets, order, position = ref.order(np.where(e.cpu().numpy() < 6, e.cpu().numpy(), -1), 6)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    assert np.array_equal(plan.order.cpu().numpy(), order)
    assert np.array_equal(plan.position.cpu().numpy(), position)
    for value in (-1, 3):
        e = torch.full((5000, 3), value, dtype=torch.int32, device="cuda")
        plan = api.expert_order(e, 4)
        offsets, order, position = ref.order(e.cpu().numpy(), 4)
        assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
        assert np.array_equal(plan.order.cpu().numpy(), order)
        assert np.array_equal(plan.position.cpu().numpy(), position)
    plan = api.expert_order(torch.empty((0, 8), dtype=torch.int32, device="cuda"), 7)
    assert plan.offsets.tolist() == [0] * 8 and plan.position.shape == (0, 8)


ROWS = [(1, 1, 1, 1), (2, 3, 4, 7), (33, 8, 16, 64), (100, 6, 12, 1000), (65, 2, 8, 4099),
        (17, 32, 64, 256), (300, 8, 32, 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,num,width", ROWS)
@pytest.mark.parametrize("shift", [0, 1])
def test_dispatch(dtype, tokens, k, num, width, shift):
    """Rows are copied bit for bit; their gradient is a float32 sum over at most k rows."""
    plan = api.expert_order(make_experts(tokens, k, num, width), num)
    base = rand(tokens, width + 9, seed=width, dtype=dtype)
    x = base[:, shift:shift + width].detach().requires_grad_()
    rows = api.dispatch(x, plan)
    order, position = plan.order.cpu().numpy(), plan.position.cpu().numpy()
    xs = x.detach().float().cpu().numpy()
    want = np.where((order >= 0)[:, None], xs[np.maximum(order, 0) // k], 0.0)
    assert rows.dtype == x.dtype and np.array_equal(rows.detach().float().cpu().numpy(), want)
    g = rand(tokens * k, width, seed=3, dtype=dtype)
    dx, = torch.autograd.grad(rows, x, g)
    gs = g.double().cpu().numpy()
    got = np.where((position >= 0)[..., None], gs[np.maximum(position, 0)], 0.0)
    total, size = got.sum(1), np.abs(got).sum(1)
    err = np.abs(dx.double().cpu().numpy() - total)
    assert (err <= HALF_ULP[dtype] * np.abs(total) + k * 2.0**-24 * size + 1e-7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,num,width", ROWS)
@pytest.mark.parametrize("shift", [0, 1])
def test_combine(dtype, tokens, k, num, width, shift):
    """Float32 sums of at most k (y) or width (the weights' gradient) products."""
    plan = api.expert_order(make_experts(tokens, k, num, width + 1), num)
    flat = rand(tokens * k * width + 8, seed=width, dtype=dtype)
    rows = flat[shift:shift + tokens * k * width].view(tokens * k, width).detach().requires_grad_()
    weights = rand(tokens, k, seed=4).detach().requires_grad_()
    y = api.combine(rows, plan, weights)
    position, order = plan.position.cpu().numpy(), plan.order.cpu().numpy()
    r = rows.detach().double().cpu().numpy()
    w = weights.detach().double().cpu().numpy()
    got = np.where((position >= 0)[..., None], r[np.maximum(position, 0)], 0.0)
    want, size = (w[..., None] * got).sum(1), np.abs(w[..., None] * got).sum(1)
    err = np.abs(y.detach().double().cpu().numpy() - want)
    assert y.dtype == rows.dtype
    assert (err <= HALF_ULP[dtype] * np.abs(want) + (k + 1) * 2.0**-24 * size + 1e-7).all()

    g = rand(tokens, width + 1, seed=6, dtype=dtype)[:, 1:]
    d_rows, d_weights = torch.autograd.grad(y, (rows, weights), g)
    gs = g.double().cpu().numpy()
    want = (got * gs[:, None, :]).sum(2)
    size = np.abs(got * gs[:, None, :]).sum(2)
    err = np.abs(d_weights.double().cpu().numpy() - want)
    assert (err <= (8 + width / 8) * 2.0**-24 * size + 1e-7).all()
    a = np.maximum(order, 0)
    want = np.where((order >= 0)[:, None], w.reshape(-1)[a][:, None] * gs[a // k], 0.0)
    err = np.abs(d_rows.double().cpu().numpy() - want)
    assert (err <= (HALF_ULP[dtype] + 2.0**-24) * np.abs(want) + 1e-7).all()
    # one gradient alone
    only_w, = torch.autograd.grad(api.combine(rows.detach(), plan, weights), weights, g)
    assert torch.equal(only_w, d_weights)
    only_r, = torch.autograd.grad(api.combine(rows, plan, weights.detach()), rows, g)
    assert torch.equal(only_r, d_rows)


@pytest.mark.gpu
def test_dispatch_offsets_beyond_32_bits():
    """Rows more than 2^31 elements apart."""
    big = torch.empty((3, 2**30 + 24), dtype=torch.bfloat16, device="cuda")
    x = big[:, -64:]
    x.copy_(rand(3, 64, seed=1, dtype="bf16"))
    plan = api.expert_order(torch.tensor([[1, 0], [0, 2], [2, 1]], dtype=torch.int32,
                                         device="cuda"), 3)
    assert torch.equal(api.dispatch(x, plan), x[plan.order.long() // 2])


@pytest.mark.gpu
def test_rows_gradient_differences():
    """combine(dispatch(x)) is linear in x and in the weights: differences give the gradients up to
    the rounding of float32 sums (2^-20 of terms of size below 64)."""
    e = make_experts(9, 3, 5, 8)
    plan = api.expert_order(e, 5)
    x = rand(9, 12, seed=31).requires_grad_()
    w = rand(9, 3, seed=32).requires_grad_()
    g = rand(9, 12, seed=33)

    def value(xv, wv):
        return (api.combine(api.dispatch(xv, plan) * 2.0, plan, wv) * g).sum()

    dx, dw = torch.autograd.grad(value(x, w), (x, w))
    with torch.no_grad():
        for i, j in ((0, 0), (3, 7), (8, 11)):
            step = torch.zeros_like(x)
            step[i, j] = 1.0
            got = (value(x + step, w) - value(x - step, w)) / 2
            assert abs(got - dx[i, j]) <= 1e-4
        for i, j in ((0, 0), (4, 1), (8, 2)):
            step = torch.zeros_like(w)
            step[i, j] = 1.0
            got = (value(x, w + step) - value(x, w - step)) / 2
            assert abs(got - dw[i, j]) <= 1e-4


@pytest.mark.gpu
def test_whole_layer_on_another_stream():
    """route -> order -> dispatch -> combine on a side stream equals the current stream's."""
    x, logits = rand(257, 512, seed=41, dtype="bf16"), rand(257, 64, seed=42)

    def layer():
        weights, experts = api.route(logits, 4)
        plan = api.expert_order(experts, 64)
        return api.combine(api.dispatch(x, plan), plan, weights)

    want = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer()
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_second_order_gradients_are_refused():
    x = rand(4, 16, seed=1).requires_grad_()
    weights, _ = api.route(x, 2)
    g = rand(4, 2, seed=2).requires_grad_()
    with pytest.raises(RuntimeError, match="first-order"):
        torch.autograd.grad(weights, x, g, create_graph=True)


@pytest.mark.gpu
def test_refusals():
    x = rand(4, 16, seed=1)
    for args, kw in (((0,), {}), ((17,), {}), ((2,), dict(score="relu")),
                     ((2,), dict(groups=3)), ((2,), dict(groups=4, topk_groups=5)),
                     ((5,), dict(groups=4, topk_groups=1)),
                     ((2,), dict(bias=torch.zeros(15, device="cuda"))),
                     ((2,), dict(bias=torch.zeros(16, device="cuda", dtype=torch.float16))),
                     ((2,), dict(bias=torch.zeros(16)))):
        with pytest.raises(ValueError):
            api.route(x, *args, **kw)
    with pytest.raises(ValueError):
        api.route(rand(2, 1025, seed=1), 2)
    e = make_experts(4, 2, 8, 1)
    with pytest.raises(ValueError):
        api.expert_order(e.long(), 8)
    with pytest.raises(ValueError):
        api.expert_order(e, 0)
    plan = api.expert_order(e, 8)
    with pytest.raises(ValueError):
        api.dispatch(x[:3], plan)
    with pytest.raises(ValueError):
        api.dispatch(x.double(), plan)
    rows = api.dispatch(x, plan)
    with pytest.raises(ValueError):
        api.combine(rows[:7], plan, torch.ones((4, 2), device="cuda"))
    with pytest.raises(ValueError):
        api.combine(rows, plan, torch.ones((4, 2), device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError):
        api.combine(rows, plan._replace(order=plan.order[:7]), torch.ones((4, 2), device="cuda"))


def test_host_tensors_are_refused():
    with pytest.raises(ValueError):
        api.route(torch.zeros((2, 8)), 2)
    with pytest.raises(ValueError):
        api.expert_order(torch.zeros((2, 2), dtype=torch.int32), 4)
    plan = api.ExpertOrder(*(torch.zeros(s, dtype=torch.int32) for s in ((5,), (4,), (2, 2))))
    with pytest.raises(ValueError):
        api.dispatch(torch.zeros((2, 8)), plan)
    with pytest.raises(ValueError):
        api.combine(torch.zeros((4, 8)), plan, torch.ones((2, 2)))


def test_abi_argument_errors():
    """Rejected on the host before any CUDA work."""
    def route(x=FAKE, elem=2, t=4, e=16, stride=16, k=2, score=0, bias=0, groups=1, tg=1, w=FAKE,
              o=FAKE):
        return bt.route(x, elem, t, e, stride, k, score, bias, groups, tg, 1, 1.0, w, o)

    for kw in (dict(x=0), dict(w=0), dict(o=0), dict(elem=5), dict(t=0), dict(e=0), dict(e=1025),
               dict(k=0), dict(k=17), dict(k=33, e=64), dict(score=2), dict(groups=3),
               dict(groups=0), dict(groups=4, tg=5), dict(groups=4, tg=0), dict(k=5, groups=4),
               dict(stride=-1), dict(x=FAKE + 2), dict(bias=FAKE + 2), dict(o=FAKE + 1)):
        assert route(**kw) == INVALID, kw

    def back(x=FAKE, elem=0, t=4, e=16, k=2, score=1, ch=FAKE, g=FAKE, o=FAKE):
        return bt.route_backward(x, elem, t, e, 16, k, score, 1, 1.0, ch, g, o)

    for kw in (dict(x=0), dict(ch=0), dict(g=0), dict(o=0), dict(elem=-1), dict(t=0), dict(k=17),
               dict(score=9), dict(o=FAKE + 1), dict(g=FAKE + 2)):
        assert back(**kw) == INVALID, kw

    need = bt.expert_order_workspace_size(8, 4)
    assert need > 0 and need % 256 == 0
    assert bt.expert_order_workspace_size(0, 4) == 0 and bt.expert_order_workspace_size(8, 0) == 0
    assert bt.expert_order_workspace_size(bt.MAX_ASSIGNMENTS + 1, 4) == 0
    assert bt.expert_order_workspace_size(8, bt.MAX_EXPERTS + 1) == 0

    def order(e=FAKE, n=8, num=4, off=FAKE, o=FAKE, pos=FAKE, ws=FAKE, wsb=need):
        return bt.expert_order(e, n, num, off, o, pos, ws, wsb)

    for kw in (dict(e=0), dict(n=0), dict(num=0), dict(num=1025), dict(off=0), dict(o=0),
               dict(pos=0), dict(pos=FAKE + 2), dict(ws=0), dict(ws=FAKE + 8), dict(wsb=need - 1)):
        assert order(**kw) == INVALID, kw

    def disp(x=FAKE, elem=0, t=4, k=2, width=8, stride=8, o=FAKE, r=FAKE):
        return bt.dispatch(x, elem, t, k, width, stride, o, r)

    for kw in (dict(x=0), dict(o=0), dict(r=0), dict(t=0), dict(k=0), dict(k=33), dict(width=0),
               dict(stride=-1), dict(t=1 << 30, k=4), dict(r=FAKE + 1), dict(elem=7)):
        assert disp(**kw) == INVALID, kw

    def comb(r=FAKE, elem=0, t=4, k=2, width=8, pos=FAKE, w=FAKE, y=FAKE):
        return bt.combine(r, elem, t, k, width, pos, w, y)

    for kw in (dict(r=0), dict(pos=0), dict(y=0), dict(t=0), dict(k=33), dict(width=0),
               dict(w=FAKE + 2), dict(y=FAKE + 1)):
        assert comb(**kw) == INVALID, kw

    def cback(r=FAKE, g=FAKE, elem=0, t=4, k=2, width=8, gs=8, pos=FAKE, live=FAKE, w=FAKE,
              dr=FAKE, dw=FAKE):
        return bt.combine_backward(r, g, elem, t, k, width, gs, pos, live, w, dr, dw)

    for kw in (dict(g=0), dict(pos=0), dict(dr=0, dw=0), dict(r=0), dict(live=0), dict(gs=-1),
               dict(t=0), dict(width=0), dict(dr=FAKE + 1), dict(dw=FAKE + 2)):
        assert cback(**kw) == INVALID, kw


@pytest.mark.gpu
def test_expert_order_keeps_no_memory():
    """A call's scratch is its own and goes back to the allocator with it."""
    e = make_experts(9001, 8, 512, 1)
    with torch.cuda.stream(torch.cuda.Stream()):
        before = torch.cuda.memory_allocated()
        plan = api.expert_order(e, 512)
        del plan
        assert torch.cuda.memory_allocated() == before


@pytest.mark.gpu
def test_expert_order_in_graphs():
    """Graphs captured on one stream, replayed beside each other, beside calls on that stream and
    after larger ones there; nothing is written to memory that others hold by then."""
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    inputs = [make_experts(16001, 8, 256, s) for s in (1, 2)]
    want = [ref.order(e.cpu().numpy(), 256) for e in inputs]
    large = make_experts(150001, 4, 1024, 3)
    large_want = ref.order(large.cpu().numpy(), 1024)
    graphs, plans = [], []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for e in inputs:
            api.expert_order(e, 256)
    for e in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            plans.append(api.expert_order(e, 256))
        graphs.append(graph)

    def check(plan, expected):
        for got, exp in zip(plan, expected):
            assert np.array_equal(got.cpu().numpy(), exp)

    with torch.cuda.stream(stream):
        check(api.expert_order(large, 1024), large_want)
        held = [torch.zeros(1 << 18, dtype=torch.uint8, device="cuda") for _ in range(32)]
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(stream):
            graphs[0].replay()
            eager = api.expert_order(large, 1024)
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        check(eager, large_want)
        for plan, expected in zip(plans, want):
            check(plan, expected)
            for t in plan:
                t.fill_(-7)
    torch.cuda.synchronize()
    assert not any(t.any().item() for t in held)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [64, 4099])
def test_combine_gradient_of_absent_assignments(dtype, width):
    """Gradients of infinities and NaN: a weight without a row still has gradient 0."""
    experts = torch.tensor([[0, -1, 2], [-1, -1, -1], [1, 2, -1]], dtype=torch.int32, device="cuda")
    plan = api.expert_order(experts, 3)
    rows = rand(9, width, seed=1, dtype=dtype).requires_grad_()
    weights = rand(3, 3, seed=2).requires_grad_()
    g = rand(3, width, seed=3, dtype=dtype)
    g[0, 5] = float("inf")
    g[1, 7] = float("nan")
    g[2, 0] = -float("inf")
    d_rows, d_weights = torch.autograd.grad(api.combine(rows, plan, weights), (rows, weights), g)
    absent = experts < 0
    assert (d_weights[absent] == 0).all() and not torch.isfinite(d_weights[~absent]).any()
    assert (d_rows[4:] == 0).all()  # five of nine places are empty


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused():
    """A tangent that the operators cannot carry on is not dropped."""
    import torch.autograd.forward_ad as forward_ad

    x, weights = rand(4, 16, seed=1), rand(4, 2, seed=2)
    plan = api.expert_order(make_experts(4, 2, 8, 1), 8)
    rows = api.dispatch(x, plan)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: api.route(dual(x), 2), lambda: api.dispatch(dual(x), plan),
                     lambda: api.combine(dual(rows), plan, weights),
                     lambda: api.combine(rows, plan, dual(weights))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        weights, _ = api.route(x.requires_grad_(), 2)  # a level alone changes nothing
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(weights, x, dual(torch.ones((4, 2), device="cuda")))


@pytest.mark.gpu
def test_second_order_terms_are_not_dropped():
    """Gradients taken with create_graph and a constant upstream gradient are those of the first
    order; differentiating them again is refused, also where another path gives a gradient."""
    x, one = rand(4, 16, seed=1).requires_grad_(), torch.ones((4, 2), device="cuda")
    want, = torch.autograd.grad(api.route(x, 2)[0], x, one)
    dx, = torch.autograd.grad(api.route(x, 2)[0], x, one, create_graph=True)
    assert torch.equal(dx, want)
    for differentiate in (lambda v: v.backward(), lambda v: torch.autograd.grad(v, x)):
        dx, = torch.autograd.grad(api.route(x, 2)[0], x, one, create_graph=True)
        with pytest.raises(RuntimeError, match="first-order"):
            differentiate(dx.square().sum() + x.square().sum())

    plan = api.expert_order(make_experts(4, 2, 8, 1), 8)
    rows, weights = rand(8, 16, seed=2).requires_grad_(), rand(4, 2, seed=3).requires_grad_()
    g = rand(4, 16, seed=4)
    want = torch.autograd.grad(api.combine(rows, plan, weights), (rows, weights), g)
    got = torch.autograd.grad(api.combine(rows, plan, weights), (rows, weights), g,
                              create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for d, source in ((got[0], weights), (got[1], rows)):
        with pytest.raises(RuntimeError, match="first-order"):
            torch.autograd.grad(d.sum() + source.sum(), source, retain_graph=True)
    # the gradient of rows under constant weights, and dispatch's, depend on nothing more
    d_rows, = torch.autograd.grad(api.combine(rows, plan, weights.detach()), rows, g,
                                  create_graph=True)
    assert torch.equal(d_rows, want[0]) and not d_rows.requires_grad
    d_x, = torch.autograd.grad(api.dispatch(x, plan), x, rand(8, 16, seed=5), create_graph=True)
    assert not d_x.requires_grad


@pytest.mark.gpu
def test_route_of_the_largest_number_of_tokens():
    """2^31 - 1 tokens (one row of logits for all): the number of blocks passes through no overflow."""
    n = 2**31 - 1
    x = torch.zeros((1, 2), dtype=torch.float16, device="cuda").expand(n, 2).requires_grad_()
    weights, experts = api.route(x, 1, score="sigmoid", renormalize=False)
    dx, = torch.autograd.grad(weights, x, torch.ones((1, 1), device="cuda").expand(n, 1))
    for t in (slice(0, 100), slice(n // 2, n // 2 + 100), slice(n - 100, n)):
        assert (experts[t] == 0).all() and (weights[t] == 0.5).all()
        assert (dx[t, 0] == 0.25).all() and (dx[t, 1] == 0).all()


@pytest.mark.gpu
def test_arguments_that_cannot_be_read():
    """An error raised while an argument is read is the call's error."""
    class Unclear:
        def __bool__(self):
            raise ZeroDivisionError

    x = rand(4, 16, seed=1)
    with pytest.raises(ZeroDivisionError):
        api.route(x, 2, renormalize=Unclear())
    with pytest.raises(ValueError):
        api.route(x, 2, score="\ud800")


@pytest.mark.gpu
def test_whole_layer_in_a_graph():
    """A training step of route, order, dispatch and combine, captured and replayed on new inputs."""
    x = rand(517, 256, seed=51, dtype="bf16").requires_grad_()
    logits = rand(517, 64, seed=52).requires_grad_()
    g = rand(517, 256, seed=53, dtype="bf16")

    def step():
        weights, experts = api.route(logits, 9, score="sigmoid")
        plan = api.expert_order(experts, 64)
        y = api.combine(api.dispatch(x, plan), plan, weights)
        return (y, *torch.autograd.grad(y, (x, logits), g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (54, 55):
        with torch.no_grad():
            x.copy_(rand(517, 256, seed=seed, dtype="bf16"))
            logits.copy_(rand(517, 64, seed=seed + 10))
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_calls_from_threads():
    """Each thread on a stream of its own, with orders of one and of several blocks."""
    import threading

    def layer(seed, tokens):
        weights, experts = api.route(rand(tokens, 64, seed=seed), 8)
        plan = api.expert_order(experts, 64)
        y = api.combine(api.dispatch(rand(tokens, 64, seed=seed + 1), plan), plan, weights)
        return (*plan, y)

    sizes = [(i, (300, 4001)[i % 2]) for i in range(4)]
    want = [layer(*s) for s in sizes]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = layer(*sizes[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
