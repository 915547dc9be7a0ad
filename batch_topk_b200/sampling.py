"""Sampling a token from each row of logits (tensor-level; ``torch_api`` re-exports it).

    noise = torch.empty(rows, vocab, device="cuda").exponential_()
    tokens, logprobs = sample(logits, noise, temperature=0.8, top_k=50, top_p=0.95)

The filters, their order and their ties are those of ``bt_sample`` in
include/batch_topk_b200.h.  No reference counterpart: the reference ends with the top k
(include/batch_topk.cuh:10-19).
"""
from __future__ import annotations

import torch

from ._lib import tensors


def sample(logits: torch.Tensor, noise: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0,
           min_p=0.0, stream=None, out: tuple | None = None):
    """(tokens int32 [rows], logprobs float32 [rows]) of logits [rows, vocab] (float16, bfloat16
    or float32 on CUDA; rows may be strided) and exponential noise [rows, vocab] (float32; one
    row may be expanded to all).

    Each setting is a number or a tensor [rows] on the logits' device (float32; int32 for top_k).
    temperature 0 takes the best token; top_k 0, top_p 1 and min_p 0 switch their filter off.
    logprobs are the tokens' log-probabilities under softmax(logits / temperature), unfiltered.
    A row without any logit above -inf gives token -1 and log-probability -inf.

    Queued on `stream` (default: the current stream of the logits' device); `out` is a pair of
    tensors to write to.  No gradient: the choice of a token has none."""
    if stream is None:
        return tensors().sample(logits, noise, temperature, top_k, top_p, min_p, out)
    if stream.device != logits.device:
        raise ValueError(f"stream is on {stream.device}, the input on {logits.device}")
    given = out if isinstance(out, tuple) else ()
    for x in (logits, noise, temperature, top_k, top_p, min_p, *given):
        if isinstance(x, torch.Tensor) and x.is_cuda:
            x.record_stream(stream)  # used there: keep its memory until the stream has run
    with torch.cuda.stream(stream):
        return tensors().sample(logits, noise, temperature, top_k, top_p, min_p, out)
