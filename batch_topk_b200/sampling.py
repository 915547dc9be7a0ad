"""Sampling a token from each row of logits (tensor-level; ``torch_api`` re-exports it).

    noise = torch.empty(rows, vocab, device="cuda").exponential_()
    tokens, logprobs = sample(logits, noise, temperature=0.8, top_k=50, top_p=0.95)

The filters, their order and their ties are those of ``bt_sample`` in
include/batch_topk_b200.h.  No reference counterpart: the reference ends with the top k
(include/batch_topk.cuh:10-19).
"""
from __future__ import annotations

import torch

from . import BatchTopkError, ELEM_BF16, ELEM_F16, ELEM_F32, MAX_SEG_LEN, _lib

ELEM = {torch.float16: ELEM_F16, torch.bfloat16: ELEM_BF16, torch.float32: ELEM_F32}


raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream without its wrapper object


def launch(what, entry, device, *args):
    """entry(*args, stream) on `device` and its current stream.  The device guard and the stream
    object cost microseconds, which small calls feel: neither is made when it is not needed."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = entry(*args, raw_stream(index))
    else:
        with torch.cuda.device(device):  # the library launches on the current device
            rc = entry(*args, raw_stream(index))
    if rc != 0:
        raise BatchTopkError(rc, what)


def _setting(name, value, rows, dtype, device, lo, hi):
    """(number, tensor or None) of one setting: a number of its range for the whole batch, or a
    tensor of its dtype with one value for each row."""
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype or value.shape != (rows,) or value.device != device:
            raise ValueError(f"{name} must be a number or a {dtype} tensor [{rows}] on {device}")
        return lo, value.contiguous()
    if not lo <= value <= hi:
        raise ValueError(f"{name} must lie in [{lo}, {hi}], got {value}")
    return value, None


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
    if logits.dtype not in ELEM or logits.dim() != 2 or not logits.is_cuda:
        raise ValueError("logits must be a 2-D float16, bfloat16 or float32 CUDA tensor")
    dev = logits.device
    rows, vocab = logits.shape
    if noise.dtype != torch.float32 or noise.shape != logits.shape or noise.device != dev:
        raise ValueError("noise must be a float32 tensor of the logits' shape on their device")
    if not 1 <= vocab <= MAX_SEG_LEN:
        raise ValueError(f"vocab must lie in [1, {MAX_SEG_LEN}], got {vocab}")
    t, d_t = _setting("temperature", temperature, rows, torch.float32, dev, 0.0, float("inf"))
    k, d_k = _setting("top_k", top_k, rows, torch.int32, dev, 0, 2**31 - 1)
    p, d_p = _setting("top_p", top_p, rows, torch.float32, dev, 0.0, 1.0)
    mp, d_mp = _setting("min_p", min_p, rows, torch.float32, dev, 0.0, 1.0)
    if out is not None:
        tokens, logprobs = out
        if (tokens.dtype != torch.int32 or logprobs.dtype != torch.float32
                or any(o.shape != (rows,) or o.device != dev or not o.is_contiguous() for o in out)):
            raise ValueError(f"out must be contiguous int32 and float32 tensors [{rows}] on {dev}")
    if stream is not None:
        if stream.device != dev:
            raise ValueError(f"stream is on {stream.device}, the input on {dev}")
        for x in (logits, noise, d_t, d_k, d_p, d_mp):
            if x is not None:
                x.record_stream(stream)  # read there: keep its memory until the stream has run
        with torch.cuda.stream(stream):
            return sample(logits, noise, temperature=temperature, top_k=top_k, top_p=top_p,
                          min_p=min_p, out=out)
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    if noise.stride(1) != 1 and vocab > 1:
        noise = noise.contiguous()
    if out is None:
        tokens = torch.empty(rows, dtype=torch.int32, device=dev)
        logprobs = torch.empty(rows, dtype=torch.float32, device=dev)
    if rows:
        launch("sample", _lib.load().bt_sample, dev, logits.data_ptr(), ELEM[logits.dtype], rows,
               vocab, logits.stride(0), noise.data_ptr(), noise.stride(0),
               t, d_t if d_t is None else d_t.data_ptr(),
               k, d_k if d_k is None else d_k.data_ptr(),
               p, d_p if d_p is None else d_p.data_ptr(),
               mp, d_mp if d_mp is None else d_mp.data_ptr(),
               tokens.data_ptr(), logprobs.data_ptr())
    return tokens, logprobs
