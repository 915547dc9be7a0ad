"""The selection operators together: the example's decode step, and the registered operators under
fake tensors and torch.compile."""
from __future__ import annotations

import pytest
import torch

import batch_topk_b200.torch_api  # noqa: F401  (registers the operators)

OPS = torch.ops.batch_topk_b200


def test_fake_kernels_give_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty((7, 1000), dtype=torch.bfloat16, device="cuda")
        t, lp = OPS.sample(x, torch.empty((7, 1000), device="cuda"), top_k=5)
        assert t.shape == lp.shape == (7,) and t.dtype == torch.int32 and lp.dtype == torch.float32
        w, e = OPS.route(x, 4)
        assert w.shape == e.shape == (7, 4) and w.dtype == torch.float32 and e.dtype == torch.int32
        offsets, order, position = OPS.expert_order(e, 1000)
        assert offsets.shape == (1001,) and order.shape == (28,) and position.shape == (7, 4)
        rows = OPS.dispatch(x, offsets, order, position)
        assert rows.shape == (28, 1000) and rows.dtype == torch.bfloat16
        assert OPS.combine(rows, offsets, order, position, w).shape == (7, 1000)


def test_fake_kernels_reject_wrong_types():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty((2, 10), dtype=torch.float64, device="cuda")
        with pytest.raises(ValueError):
            OPS.sample(x, x)
        with pytest.raises(ValueError):
            OPS.route(x, 2)
        with pytest.raises(ValueError):
            OPS.expert_order(x, 4)


@pytest.mark.gpu
def test_operators_under_torch_compile():
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((33, 64), generator=g, device="cuda")
    q = torch.empty((33, 64), device="cuda").exponential_(generator=g)

    def f(t, q):
        w, e = OPS.route(t * 2, 4, score="sigmoid")
        offsets, order, position = OPS.expert_order(e, 64)
        y = OPS.combine(OPS.dispatch(t, offsets, order, position), offsets, order, position, w)
        return OPS.sample(y, q, temperature=0.5, top_p=0.9)

    want = f(x, q)
    got = torch.compile(f, fullgraph=True)(x, q)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,k", [(1, 8, 1), (32, 64, 4), (100, 16, 2)])
def test_layer_equals_plain_torch(tokens, experts, k):
    """Half-precision products and sums in the same order, rounded to half once or twice more on
    either side: differences below 2^-9 of the result's norm."""
    from batch_topk_b200.moe_decode import MoeDecoder

    model = MoeDecoder(128, 96, experts, k, 512, 2, seed=tokens)
    x = model.embed[:tokens]
    for layer in model.layers:
        got, want = layer(x), layer.plain(x)
        assert (got - want).float().norm() <= 2.0**-9 * want.float().norm()
        x = got


@pytest.mark.gpu
def test_decode_steps_repeat():
    from batch_topk_b200.moe_decode import MoeDecoder

    model = MoeDecoder(128, 64, 16, 2, 1000, 2, seed=7)
    g = torch.Generator(device="cuda").manual_seed(8)
    noise = [torch.empty((9, 1000), device="cuda").exponential_(generator=g) for _ in range(3)]

    def run():
        tokens, out = torch.arange(9, dtype=torch.int32, device="cuda"), []
        for q in noise:
            tokens, lp = model.step(tokens, q, temperature=0.8, top_k=50, top_p=0.95)
            assert ((tokens >= 0) & (tokens < 1000)).all() and torch.isfinite(lp).all()
            out += [tokens, lp]
        return out

    assert all(torch.equal(a, b) for a, b in zip(run(), run()))
