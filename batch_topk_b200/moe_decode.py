"""One decode step of a small mixture-of-experts model: the selection operators as they are used
together.

    python -m batch_topk_b200.moe_decode [--tokens 32] [--width 1024] [--hidden 512] [--experts 64]
                                         [--k 4] [--vocab 32000] [--layers 2] [--steps 4] [--check]

Each layer routes its tokens (``route``), sorts the assignments by expert (``expert_order``), moves
the tokens' rows there (``dispatch``), runs each expert's two products on its rows, and sums the
results back (``combine``); the head turns the last hidden state into logits (``bt_logits_f16``), and
``sample`` picks the tokens, whose embeddings are the next step's input.  Weights are random; the
command prints the tokens of each step and the time the selection operators take in a step.  --check
compares every layer with the same mathematics in plain torch.
"""
from __future__ import annotations

import argparse

import torch

import batch_topk_b200 as bt
from batch_topk_b200 import torch_api as api


class MoeLayer:
    """Experts e: silu(x @ up[e]) @ down[e], weighted by a sigmoid router with a balance bias."""

    def __init__(self, width, hidden, experts, k, generator, device):
        def make(*shape):
            w = torch.randn(shape, generator=generator, device=device) * shape[-2] ** -0.5
            return w.half()

        self.k, self.experts = k, experts
        self.router = make(width, experts)
        self.bias = torch.randn(experts, generator=generator, device=device) * 0.05
        self.up, self.down = make(experts, width, hidden), make(experts, hidden, width)

    def __call__(self, x):
        weights, experts = api.route(x @ self.router, self.k, score="sigmoid", bias=self.bias)
        plan = api.expert_order(experts, self.experts)
        rows = api.dispatch(x, plan)
        out = torch.zeros_like(rows)
        at = plan.offsets.tolist()
        for e in range(self.experts):
            a, b = at[e], at[e + 1]
            if a < b:
                out[a:b] = torch.nn.functional.silu(rows[a:b] @ self.up[e]) @ self.down[e]
        return x + api.combine(out, plan, weights)

    def plain(self, x):
        """The same layer, every expert on every token."""
        score = torch.sigmoid((x @ self.router).float())
        top = (score + self.bias).topk(self.k, dim=1).indices
        w = score.gather(1, top)
        w = w / w.sum(1, keepdim=True)
        gate = torch.zeros_like(score).scatter_(1, top, w)
        h = torch.nn.functional.silu(torch.einsum("tw,ewh->eth", x, self.up))
        return x + torch.einsum("te,etw->tw", gate, (h @ self.down).float()).half()


class MoeDecoder:
    """Layers, an output head and an embedding, with random weights."""

    def __init__(self, width, hidden, experts, k, vocab, layers, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.layers = [MoeLayer(width, hidden, experts, k, g, device) for _ in range(layers)]
        self.head = (torch.randn((vocab, width), generator=g, device=device) * 2 *
                     width ** -0.5).half()
        self.embed = torch.randn((vocab, width), generator=g, device=device).half()

    def logits(self, x):
        x = (x / x.float().square().mean(1, keepdim=True).sqrt()).half().contiguous()
        out = torch.empty((x.shape[0], self.head.shape[0]), dtype=torch.float16, device=x.device)
        rc = bt.logits_f16(x.data_ptr(), self.head.data_ptr(), x.shape[0], self.head.shape[0],
                           x.shape[1], out.data_ptr(), torch.cuda.current_stream().cuda_stream)
        if rc:
            raise bt.BatchTopkError(rc, "bt_logits_f16")
        return out

    def step(self, tokens, noise, **settings):
        """(next tokens, their log-probabilities) for the tokens of each sequence."""
        x = self.embed[tokens.long()]
        for layer in self.layers:
            x = layer(x)
        return api.sample(self.logits(x), noise, **settings)


def selection_us(model, tokens, noise, reps=50):
    """Microseconds of the selection operators of one layer and of the sampling."""
    layer, x = model.layers[0], model.embed[tokens.long()]
    scores, logits = x @ layer.router, model.logits(x)

    def layer_ops():
        weights, experts = api.route(scores, layer.k, score="sigmoid", bias=layer.bias)
        plan = api.expert_order(experts, layer.experts)
        return api.combine(api.dispatch(x, plan), plan, weights)

    def time(f):
        for _ in range(5):
            f()
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(reps):
            f()
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b) / reps * 1e3

    return time(layer_ops), time(lambda: api.sample(logits, noise, temperature=0.8, top_k=50,
                                                    top_p=0.95))


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, value in (("tokens", 32), ("width", 1024), ("hidden", 512), ("experts", 64), ("k", 4),
                        ("vocab", 32000), ("layers", 2), ("steps", 4), ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--check", action="store_true", help="compare the layers with plain torch")
    a = ap.parse_args()
    if not torch.cuda.is_available():
        raise SystemExit("a CUDA device is required")
    model = MoeDecoder(a.width, a.hidden, a.experts, a.k, a.vocab, a.layers, seed=a.seed)
    g = torch.Generator(device="cuda").manual_seed(a.seed + 1)
    tokens = torch.randint(0, a.vocab, (a.tokens,), generator=g, device="cuda", dtype=torch.int32)
    noise = torch.empty((a.tokens, a.vocab), device="cuda")
    if a.check:
        x = model.embed[tokens.long()]
        for i, layer in enumerate(model.layers):
            got, want = layer(x), layer.plain(x)
            err = ((got - want).float().norm() / want.float().norm()).item()
            print(f"layer {i}: relative difference {err:.1e}")
            if err > 5e-3:
                raise SystemExit(1)
            x = got
    for step in range(a.steps):
        noise.exponential_(generator=g)
        tokens, logprobs = model.step(tokens, noise, temperature=0.8, top_k=50, top_p=0.95)
        print(f"step {step}: tokens {tokens[:8].tolist()} mean log-probability "
              f"{logprobs.mean().item():.3f}")
    layer_us, sample_us = selection_us(model, tokens, noise)
    print(f"route + expert_order + dispatch + combine {layer_us:.1f} us a layer, "
          f"sample {sample_us:.1f} us")


if __name__ == "__main__":
    main()
