"""Drawing the next token on the device (include/sepia_cuda.h,
sepia_cuda_sample; csrc/sample.cu)."""
from __future__ import annotations

import torch

from .lib import last_error, load

_F16 = {torch.float32: 0, torch.float16: 1}


def _row_arg(t, name, dtype, n):
    if t is None:
        return None
    if not (t.is_cuda and t.is_contiguous() and t.dtype == dtype and t.shape == (n,)):
        raise ValueError(f"sepia_b200: sample: {name} must be a contiguous CUDA tensor of {dtype}, one value per row")
    return t.data_ptr()


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, ids=None, prob=None, stream=None):
    """One token per row of logits (float32 or float16 [rows, vocab], any row
    stride) from one uniform number u[row] in [0, 1) each. temperature, top_p,
    min_p (float32) and top_k (int32) hold a value per row; None turns one off.
    Returns (ids int32, prob float32): the tokens and their share of the
    weights that the filters left in; -1 and 0 where a row has no token."""
    if not (logits.is_cuda and logits.dim() == 2 and logits.dtype in _F16):
        raise ValueError("sepia_b200: sample: logits must be a float32 or float16 CUDA tensor [rows, vocab]")
    n, v = logits.shape
    if v > 1 and logits.stride(1) != 1:
        raise ValueError("sepia_b200: sample: the logits of a row must lie side by side")
    dev = logits.device
    if ids is None:
        ids = torch.empty(n, dtype=torch.int32, device=dev)
    if prob is None:
        prob = torch.empty(n, dtype=torch.float32, device=dev)
    st = (stream if stream is not None else torch.cuda.current_stream(dev)).cuda_stream
    f = torch.float32
    if not load().sepia_cuda_sample(_F16[logits.dtype], logits.data_ptr(), logits.stride(0) if n > 1 else v, n, v,
                                    _row_arg(u, "u", f, n), _row_arg(temperature, "temperature", f, n),
                                    _row_arg(top_k, "top_k", torch.int32, n), _row_arg(top_p, "top_p", f, n),
                                    _row_arg(min_p, "min_p", f, n), _row_arg(ids, "ids", torch.int32, n),
                                    _row_arg(prob, "prob", f, n), st):
        raise RuntimeError(f"sepia_b200: sample failed: {last_error()}")
    return ids, prob
