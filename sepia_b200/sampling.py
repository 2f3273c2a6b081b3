"""Drawing the next token on the device (include/sepia_cuda.h,
sepia_cuda_sample; csrc/sample.cu)."""
from __future__ import annotations

import contextlib

import torch

from .lib import last_error, load

_F16 = {torch.float32: 0, torch.float16: 1}


def _row(t, name, dtype, n):
    if t.dtype is not dtype or not t.is_cuda or not t.is_contiguous() or t.shape != (n,):
        raise ValueError(f"sepia_b200: sample: {name} must be a contiguous CUDA tensor of {dtype}, one value per row")
    return t.data_ptr()


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, ids=None, prob=None, stream=None):
    """One token per row of logits (float32 or float16 [rows, vocab], any row
    stride) from one uniform number u[row] in [0, 1) each. temperature, top_p,
    min_p (float32) and top_k (int32) hold a value per row; None turns one off.
    Returns (ids int32, prob float32): the tokens and their share of the
    weights that the filters left in; -1 and 0 where a row has no token."""
    f16 = _F16.get(logits.dtype)
    if f16 is None or not logits.is_cuda or logits.dim() != 2:
        raise ValueError("sepia_b200: sample: logits must be a float32 or float16 CUDA tensor [rows, vocab]")
    n, v = logits.shape
    s0, s1 = logits.stride()
    if v > 1 and s1 != 1:
        raise ValueError("sepia_b200: sample: the logits of a row must lie side by side")
    f, i = torch.float32, torch.int32
    if ids is not None:
        _row(ids, "ids", i, n)
    if prob is not None:
        _row(prob, "prob", f, n)
    u_p = _row(u, "u", f, n)
    if ids is None or prob is None:
        # a result's memory belongs to the stream that fills it
        with contextlib.nullcontext() if stream is None else torch.cuda.stream(stream):
            ids = torch.empty_like(u, dtype=i) if ids is None else ids
            prob = torch.empty_like(u) if prob is None else prob
    ids_p, prob_p = ids.data_ptr(), prob.data_ptr()
    st = stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(logits.device.index)
    if not load().sepia_cuda_sample(f16, logits.data_ptr(), s0 if n > 1 else v, n, v, u_p,
                                    None if temperature is None else _row(temperature, "temperature", f, n),
                                    None if top_k is None else _row(top_k, "top_k", i, n),
                                    None if top_p is None else _row(top_p, "top_p", f, n),
                                    None if min_p is None else _row(min_p, "min_p", f, n), ids_p, prob_p, st):
        raise RuntimeError(f"sepia_b200: sample failed: {last_error()}")
    return ids, prob
