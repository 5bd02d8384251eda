"""Token sampling on torch device tensors: temperature, top-k, top-p and min-p from given
random numbers, for rows of logits such as the last projection of a decode or verify
step leaves (include/k3_hip_sample_abi.h).

The call enqueues gfx950 work on the current torch stream of the current device and
raises K3SpineError with the library's reason on a non-zero status; arguments that do not
fit raise ValueError.  There is no CPU path.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .dense import _check, _ptr, _run
from .moe import _dtype_code


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: torch.Tensor | None = None,
           top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
           min_p: torch.Tensor | None = None, out: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row of logits (fp32 or bfloat16, [rows, vocabulary]) as int32 [rows].

    Tokens are ordered by logit (larger first; lower index first where equal), weighted by
    exp((logit - largest) / temperature) and cut to the shortest of three prefixes: the
    first top_k, the shortest with at least top_p of the top-k ones' weight, and those of
    at least min_p times the largest weight.  The token is the first at which the running
    weight exceeds u times the kept one.  temperature 0 takes the largest logit.

    u: fp32 [rows] in [0, 1); temperature, top_p, min_p: fp32 [rows]; top_k: int32 [rows];
    those left out do not limit (temperature 1).  A row of -inf and NaN alone gives -1.
    The same inputs give the same tokens in any batch."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("logits must be float32 or bfloat16 [rows, vocabulary]")
    _check(logits, logits.dtype, logits.shape, "logits")
    rows, vocab = logits.shape
    _check(u, torch.float32, (rows,), "u")
    for t, dtype, name in ((temperature, torch.float32, "temperature"),
                           (top_k, torch.int32, "top_k"), (top_p, torch.float32, "top_p"),
                           (min_p, torch.float32, "min_p")):
        if t is not None:
            _check(t, dtype, (rows,), name)
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    else:
        _check(out, torch.int32, (rows,), "out")
    d = _lib.K3HipSampleV1(
        _lib.K3_SAMPLE_ABI_V1, C.sizeof(_lib.K3HipSampleV1), _dtype_code(logits), rows, vocab, 0,
        logits.data_ptr(), u.data_ptr(), _ptr(temperature), _ptr(top_k), _ptr(top_p), _ptr(min_p),
        out.data_ptr())
    _run("k3_hip_sample", d, workspace)
    return out
