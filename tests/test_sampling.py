"""Sampling (torch_api.sample, bt_sample) against a plain 64-bit implementation.

No reference counterpart.  Tokens: the kernel's weights carry relative errors of a few 2^-24 (the
scaled logit, at most about 90 in size where the weight matters, its exponential, the quotient and
sums), below 2e-5 in all; the plain implementation says which tokens such an error admits, almost
always one.  Log-probabilities: the scaled logit and the logarithm are each rounded to float32, so
an error of 2^-22 of their size plus 4e-6 for the sum.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import batch_topk_b200 as bt
from batch_topk_b200 import torch_api as api
from lm_reference import sample_row

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SLACK = 2e-5
INVALID = bt.CUDA_ERROR_INVALID_VALUE
FAKE = 1 << 20  # a 16-byte aligned address that is never dereferenced


def as_rows(value, n):
    return (value.cpu().numpy() if isinstance(value, torch.Tensor) else np.full(n, value))


def check(logits, noise, tokens, logprobs, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    x, q = logits.float().cpu().numpy(), noise.cpu().numpy()
    tok, lp = tokens.cpu().numpy(), logprobs.cpu().numpy()
    n = x.shape[0]
    t, k, p, mp = (as_rows(v, n) for v in (temperature, top_k, top_p, min_p))
    for r in range(n):
        ok, want = sample_row(x[r], q[r], float(np.float32(t[r])), int(k[r]),
                              float(np.float32(p[r])), float(np.float32(mp[r])), SLACK)
        if ok is None:
            assert tok[r] == -1 and lp[r] == -np.inf, r
            continue
        assert int(tok[r]) in ok, (r, int(tok[r]), ok)
        w = want[tok[r]]
        if np.isfinite(w):
            assert abs(lp[r] - w) <= 4e-6 + 2.0**-21 * abs(w), (r, lp[r], w)
        else:
            assert lp[r] == w, r


def inputs(n, v, dtype, seed, scale=4.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, v), generator=g, device="cuda") * scale
    q = torch.empty((n, v), device="cuda").exponential_(generator=g).clamp_(min=1e-20)
    return x.to(DTYPES[dtype]), q


SETTINGS = [
    dict(),
    dict(temperature=0.0),
    dict(temperature=0.7, top_k=50),
    dict(temperature=1.3, top_k=1),
    dict(temperature=0.9, top_p=0.9),
    dict(top_p=0.0),
    dict(temperature=1.5, min_p=0.05),
    dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.01),
    dict(temperature=2.5, top_k=1000, top_p=0.99),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", [(1, 1), (3, 2), (5, 17), (2, 1000), (3, 4097), (4, 32000),
                                 (1, 200001)])
def test_sizes_and_settings(dtype, n, v):
    x, q = inputs(n, v, dtype, 100 + n + v)
    for kw in SETTINGS:
        tokens, logprobs = api.sample(x, q, **kw)
        check(x, q, tokens, logprobs, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("scale", [0.3, 3.0])
def test_long_rows(dtype, scale):
    x, q = inputs(1, 3000017, dtype, 5, scale)
    for kw in (dict(), dict(top_k=100), dict(top_k=5000, temperature=0.5), dict(top_p=0.7),
               dict(min_p=0.2), dict(temperature=0.0)):
        tokens, logprobs = api.sample(x, q, **kw)
        check(x, q, tokens, logprobs, **kw)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows more than 2^31 elements apart."""
    big = torch.empty((3, 2**30 + 24), dtype=torch.bfloat16, device="cuda")
    x, q = inputs(3, 2003, "bf16", 19)
    view = big[:, -2003:]
    view.copy_(x)
    for kw in (dict(), dict(top_k=20, top_p=0.9)):
        tokens, logprobs = api.sample(view, q, **kw)
        check(x, q, tokens, logprobs, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [150, 300, 600])
def test_many_rows(dtype, n):
    """Batches that take one, two or more blocks a row."""
    x, q = inputs(n, 6007, dtype, n, 3.0)
    for kw in (dict(), dict(top_k=20), dict(top_p=0.9), dict(top_p=0.95, temperature=3.0)):
        tokens, logprobs = api.sample(x, q, **kw)
        check(x, q, tokens, logprobs, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, 0.05, 0.6, 30.0])
def test_flat_and_peaked_rows(dtype, scale):
    """Rows from constant (every cut runs through ties) to one token with all the weight."""
    x, q = inputs(3, 20011, dtype, 7, scale)
    for kw in SETTINGS:
        tokens, logprobs = api.sample(x, q, **kw)
        check(x, q, tokens, logprobs, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_at_the_cut(dtype):
    """Few distinct values: the cuts of top-k and top-p fall among equal elements."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-3, 3, (6, 3001), generator=g, device="cuda").to(DTYPES[dtype])
    x[0] = -2.0
    x[1, ::2] = -0.0
    x[1, 1::2] = 0.0
    q = torch.empty((6, 3001), device="cuda").exponential_(generator=g).clamp_(min=1e-20)
    for kw in (dict(top_k=7), dict(top_k=600), dict(top_p=0.3), dict(top_p=0.77, top_k=1100),
               dict(min_p=0.5), dict(temperature=0.0), dict(temperature=0.2, top_p=0.5)):
        tokens, logprobs = api.sample(x, q, **kw)
        check(x, q, tokens, logprobs, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows(dtype):
    """Rows with nothing open, one open token, the type's lowest value, infinities and NaN."""
    x, q = inputs(9, 5003, dtype, 11)
    lowest = torch.finfo(x.dtype).min
    x[0] = float("-inf")
    x[1] = float("nan")
    x[2] = float("-inf")
    x[2, 4321] = -5.0
    x[3, ::3] = float("nan")
    x[4, 10:5000] = float("-inf")
    x[5, 77] = float("inf")
    x[6, 5:4000:7] = float("inf")
    x[7] = lowest
    x[8, 1:] = lowest
    for kw in SETTINGS:
        tokens, logprobs = api.sample(x, q, **kw)
        check(x, q, tokens, logprobs, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e5, 3e8, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("temperature", [1.0, 1e-3, 1e4])
def test_huge_logits(size, temperature):
    """Logits far from zero: sums of weights are relative to the maximum, however large it is."""
    x, q = inputs(6, 4099, "fp32", 15, size)
    x[3:] += size * 4
    x[5] = -size
    for kw in (dict(), dict(top_k=9), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0)):
        kw = {"temperature": temperature, **kw}
        tokens, logprobs = api.sample(x, q, **kw)
        check(x, q, tokens, logprobs, **kw)


@pytest.mark.gpu
def test_settings_of_each_row():
    """One value a row, those outside their range among them: they switch the filter off or clamp."""
    n = 24
    x, q = inputs(n, 9001, "bf16", 13, 2.0)
    pick = np.random.default_rng(5)
    nan = float("nan")
    dev = x.device
    kw = dict(
        temperature=torch.tensor(pick.choice([0.0, 0.5, 1.0, 1.7, -1.0, nan], n),
                                 dtype=torch.float32, device=dev),
        top_k=torch.tensor(pick.choice([0, -3, 1, 5, 300, 9001, 50000], n), dtype=torch.int32,
                           device=dev),
        top_p=torch.tensor(pick.choice([1.0, 0.0, 0.5, 0.9, 1.5, nan, -1.0], n),
                           dtype=torch.float32, device=dev),
        min_p=torch.tensor(pick.choice([0.0, 0.1, 1.0, 2.0, nan, -1.0], n), dtype=torch.float32,
                           device=dev))
    tokens, logprobs = api.sample(x, q, **kw)
    check(x, q, tokens, logprobs, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_strides(dtype, shift):
    """Rows inside a wider tensor at odd offsets, one row of noise for all, and a transposed view."""
    big, noise = inputs(5, 3333, dtype, 17)
    x, q = big[:, shift:shift + 3001], noise[:1, shift:shift + 3001].expand(5, 3001)
    tokens, logprobs = api.sample(x, q, temperature=0.9, top_p=0.9)
    check(x, q, tokens, logprobs, temperature=0.9, top_p=0.9)
    xt, qt = big.t().contiguous().t(), noise.t().contiguous().t()
    tokens, logprobs = api.sample(xt, qt, top_k=9)
    check(xt, qt, tokens, logprobs, top_k=9)


@pytest.mark.gpu
def test_noise_that_is_zero_or_not_a_number():
    """A quotient that is NaN or negative loses; one that is infinite wins."""
    x = torch.zeros((4, 40), device="cuda")
    q = torch.ones((4, 40), device="cuda")
    q[0, :30] = float("nan")
    q[0, 33] = 0.5
    q[1, 7] = 0.0
    q[2] = -1.0
    q[2, 5] = 3.0
    q[3] = float("nan")
    tokens, _ = api.sample(x, q)
    assert tokens.tolist() == [33, 7, 5, 0]


@pytest.mark.gpu
def test_same_call_gives_the_same_bits():
    x, q = inputs(64, 50001, "fp16", 23, 0.5)
    a = api.sample(x, q, top_p=0.9, top_k=4000)
    for _ in range(3):
        b = api.sample(x, q, top_p=0.9, top_k=4000)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_frequencies():
    """20000 draws from one row of 6 tokens: counts within 5 standard deviations."""
    n = 20000
    x = torch.tensor([[2.0, 1.0, 0.0, -1.0, float("-inf"), 1.5]], device="cuda").expand(n, 6)
    g = torch.Generator(device="cuda").manual_seed(29)
    q = torch.empty((n, 6), device="cuda").exponential_(generator=g).clamp_(min=1e-20)
    tokens, _ = api.sample(x, q, temperature=0.8, top_k=4)
    count = torch.bincount(tokens, minlength=6).cpu().numpy()
    w = np.exp(np.array([2.0, 1.0, 0.0, -np.inf, -np.inf, 1.5]) / 0.8)
    prob = w / w.sum()
    assert (np.abs(count - n * prob) <= 5 * np.sqrt(n * prob * (1 - prob))).all()


@pytest.mark.gpu
def test_streams_and_out():
    """A call on another stream than the inputs' (after they are ready), into given tensors."""
    x, q = inputs(8, 30001, "fp32", 31)
    want = api.sample(x, q, top_p=0.8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = (torch.empty(8, dtype=torch.int32, device="cuda"), torch.empty(8, device="cuda"))
    got = api.sample(x, q, top_p=0.8, stream=side, out=out)
    side.synchronize()
    assert got[0] is out[0] and torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.gpu
def test_graph_capture():
    x, q = inputs(4, 10000, "bf16", 37)
    want = api.sample(x, q, top_k=30, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = api.sample(x, q, top_k=30, top_p=0.9)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_no_rows_and_refusals():
    x, q = inputs(4, 100, "fp32", 41)
    tokens, logprobs = api.sample(x[:0], q[:0])
    assert tokens.shape == (0,) and logprobs.shape == (0,)
    for kw in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=1.5), dict(min_p=-0.1),
               dict(temperature=float("nan")), dict(top_p=torch.ones(4)),
               dict(top_k=torch.ones(4, device="cuda")),
               dict(min_p=torch.zeros(3, device="cuda"))):
        with pytest.raises(ValueError):
            api.sample(x, q, **kw)
    with pytest.raises(ValueError):
        api.sample(x, q[:, :99])
    with pytest.raises(ValueError):
        api.sample(x, q.double())
    with pytest.raises(ValueError):
        api.sample(x, q, out=(torch.empty(4, device="cuda"), torch.empty(4, device="cuda")))


def test_host_tensors_are_refused():
    with pytest.raises(ValueError):
        api.sample(torch.zeros((2, 8)), torch.ones((2, 8)))
    with pytest.raises(ValueError):
        api.sample(torch.zeros((2, 8), dtype=torch.float64), torch.ones((2, 8)))


def test_abi_argument_errors():
    """Rejected on the host before any CUDA work."""
    def call(x=FAKE, elem=bt.DTYPE_F32, rows=2, vocab=10, xs=10, q=FAKE, qs=10, dt=0, dk=0,
             tok=FAKE, lp=FAKE):
        return bt.sample(x, elem, rows, vocab, xs, q, qs, 1.0, dt, 0, dk, 1.0, 0, 0.0, 0, tok, lp)

    assert call(x=0) == INVALID
    assert call(q=0) == INVALID
    assert call(tok=0) == INVALID
    assert call(lp=0) == INVALID
    assert call(elem=3) == INVALID
    assert call(rows=0) == INVALID
    assert call(vocab=0) == INVALID
    assert call(vocab=bt.MAX_SEG_LEN + 1) == INVALID
    assert call(xs=-1) == INVALID
    assert call(qs=-1) == INVALID
    assert call(x=FAKE + 2) == INVALID
    assert call(q=FAKE + 2) == INVALID
    assert call(dt=FAKE + 2) == INVALID
    assert call(dk=FAKE + 1) == INVALID
    assert call(lp=FAKE + 2) == INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [37, 1000, 32003, 128256])
@pytest.mark.parametrize("settings", [dict(), dict(temperature=0.0), dict(temperature=0.7, top_p=0.9),
                                      dict(top_k=40), dict(top_k=20, top_p=0.95, min_p=0.1)])
def test_confident_rows(dtype, vocab, settings):
    """One token with nearly all weight: its log-probability is the others' weight.  An exponent of up
    to 32 octaves passes through about four roundings of 2^-20, so 1e-5 of the value."""
    n = 9
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn((n, vocab + 3), generator=g, device="cuda").to(DTYPES[dtype])[:, 1:vocab + 1]
    at = torch.tensor([0, 1, 5, vocab // 2, vocab // 3, vocab - 1, vocab - 2, 20, 36], device="cuda")
    lift = np.log(vocab) + torch.tensor([2.5, 4, 6, 8, 2.5, 3, 4, 10, 1.9], device="cuda")
    x[torch.arange(n), at] = lift.to(x.dtype)
    noise = torch.ones((n, vocab), device="cuda")  # the heaviest token wins
    tokens, logprobs = api.sample(x, noise, **settings)
    assert torch.equal(tokens.long(), at)
    t = settings.get("temperature", 1.0) or 1.0
    rows = x.double().cpu().numpy()
    for r in range(n):
        e = np.exp((rows[r] - rows[r, at[r]]) / np.float64(np.float32(t)))
        e[at[r].item()] = 0.0
        want = -np.log1p(e.sum())
        assert abs(logprobs[r].item() - want) <= 1e-5 * abs(want), (r, logprobs[r].item(), want)


@pytest.mark.gpu
def test_outputs_given_for_another_stream_are_kept_for_it(monkeypatch):
    """What a call on another stream reads or writes is not handed out again before it has run."""
    kept = []
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: kept.append((t.data_ptr(), s)))
    x, q = inputs(4, 100, "fp32", 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = (torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(4, device="cuda"))
    p = torch.full((4,), 0.9, device="cuda")
    api.sample(x, q, top_p=p, stream=side, out=out)
    side.synchronize()
    for t in (x, q, p, *out):
        assert (t.data_ptr(), side) in kept


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 5003, 151936])
@pytest.mark.parametrize("rows", [64, 600])
def test_equal_quotients_go_to_the_lowest_index(dtype, vocab, rows):
    """Constant logits with constant noise of many values, and with noise one step lower at two
    places (1 / 1.125 and its neighbour's quotient differ in float32)."""
    x = torch.full((1, vocab), 1.5, device="cuda", dtype=DTYPES[dtype]).expand(rows, vocab)
    q = torch.linspace(0.01, 7.3, rows, device="cuda")[:, None].expand(rows, vocab).contiguous()
    for kw in (dict(), dict(temperature=0.7)):
        tokens, _ = api.sample(x, q, **kw)
        assert (tokens == 0).all(), kw
    r = torch.arange(rows, device="cuda")
    at = (r * 7919 + 3) % (vocab - 1)
    later = torch.minimum(at + 1 + r % 300, torch.tensor(vocab - 1, device="cuda"))
    q.fill_(1.125)
    q[r, at] = q[r, later] = float(np.nextafter(np.float32(1.125), np.float32(0)))
    tokens, _ = api.sample(x, q)
    assert torch.equal(tokens.long(), at)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", [(1, 32003), (40, 5003), (600, 4096)])
def test_nearly_equal_quotients(dtype, n, v):
    """Noise that all but follows the weights: without filters the race is decided as it is behind
    a filter that keeps everything, where each quotient is compared as it is in float32."""
    x, q = inputs(n, v, dtype, 47, 2.0)
    w = torch.exp(x.double() - x.double().amax(1, keepdim=True))
    q = (w * (1 + 1e-6 * torch.randn(n, v, device="cuda", dtype=torch.float64))).float()
    tokens, _ = api.sample(x, q)
    kept, _ = api.sample(x, q, min_p=1e-30)
    assert torch.equal(tokens, kept)


def long_row(kind, v, dtype):
    if kind == "flat":  # one token ahead of all others
        x = torch.full((v,), -0.5, device="cuda")
        x[0] = 0.0
    elif kind == "rising":
        x = torch.linspace(-3.0, 3.0, v, device="cuda")
    else:  # few values in long runs
        x = torch.arange(v, device="cuda").div(v / 5.0).floor().mul(-0.375)
    return x.to(DTYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["flat", "runs", "rising"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,v", [(600, 3000017), (130, 3000017), (2, 2**24 + 5), (1, 2**26)])
def test_sums_of_long_rows(kind, dtype, n, v):
    """Sums over millions of equal or slowly changing weights, at many temperatures, in every pass
    that sums a row: within the bound that holds for every other row."""
    x = long_row(kind, v, dtype)
    best = int(x.argmax())
    t = torch.linspace(0.3, 3.0, n, device="cuda")
    want = []
    for r in range(n):
        z = torch.zeros((), dtype=torch.float64, device="cuda")
        values, counts = torch.unique(x, return_counts=True) if r == 0 else (values, counts)
        e = (values.double() - values[-1].double()) / t[r].double()
        want.append(-torch.log((torch.exp(e) * counts).sum()))
    want = torch.stack(want)
    rows, noise = x.expand(n, v), torch.ones((1, v), device="cuda").expand(n, v)
    settings = [dict(), dict(top_p=0.7), dict(top_k=200)]
    if n * v < 5e8 and kind != "rising":
        settings.append(dict(top_k=3000, top_p=0.99))
    for kw in settings:
        tokens, logprobs = api.sample(rows, noise, temperature=t, **kw)
        assert ((x[tokens.long()] - x[best]).abs() <= 1e-5).all(), kw
        err = (logprobs.double() - want).abs()
        assert (err <= 4e-6 + 2.0**-21 * want.abs()).all(), (kw, err.max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("n,v", [(600, 3000017), (2, 2**24 + 5)])
@pytest.mark.parametrize("p", [0.3, 0.85])
def test_nucleus_of_long_flat_rows(n, v, p):
    """The cut falls among millions of equal tokens: a favoured one 3e-5 of the mass before it is
    kept, a more favoured one as far behind it is not."""
    x = long_row("flat", v, "bf16")
    t = torch.linspace(0.3, 3.0, n, device="cuda")
    w = torch.exp(-0.5 / t.double())
    mass = 1.0 + (v - 1) * w
    p32 = float(np.float32(p))
    inside = ((p32 * (1 - 3e-5) * mass - 1.0) / w).floor().long()
    outside = ((p32 * (1 + 3e-5) * mass - 1.0) / w).ceil().long() + 1
    for r in range(0, n, max(1, n // 12)):
        noise = torch.ones(v, device="cuda")
        noise[inside[r]] = 1e-6
        noise[outside[r]] = 1e-12
        # the row among as many others as the batch has, so that it gets as many blocks
        tokens, _ = api.sample(x.expand(n, v), noise.expand(n, v), temperature=float(t[r]), top_p=p)
        assert (tokens == inside[r]).all(), r


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("n", [7, 300])
def test_same_nucleus_call_gives_the_same_bits(dtype, n):
    """Nuclei of some hundred to some thousand tokens, about the size at which the list ends."""
    x, q = inputs(n, 50001, dtype, 53, 2.0)
    t = torch.linspace(0.6, 1.6, n, device="cuda")
    for p in (0.2, 0.5, 0.8):
        a = api.sample(x, q, temperature=t, top_p=p)
        for _ in range(5):
            b = api.sample(x, q, temperature=t, top_p=p)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
