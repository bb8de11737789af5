"""Token sampling on the device: temperature, top-k, top-p and min-p, one given
uniform number a row.

The reference samples greedily or with temperature and top-k
(``falcon_perception/sampling.py:10-51``) through a chain of tensor operations
and torch's own generator; here one kernel reads the logits and the random
numbers are the caller's, so that a step can be replayed.
"""

from __future__ import annotations

import torch
from torch import Tensor

from . import _lib

_DTYPES = {torch.float32: _lib.FPKV_F32, torch.bfloat16: _lib.FPKV_BF16, torch.float16: _lib.FPKV_F16}


def _per_row(value, name: str, rows: int, dtype: torch.dtype, like: Tensor) -> Tensor | None:
    """A filter setting as the kernel takes it: None, or one ``dtype`` number a row."""
    if value is None:
        return None
    if not isinstance(value, Tensor):
        if dtype == torch.int32:                    # beyond the vocabulary: no limit, as for a tensor of int64
            value = min(max(int(value), 0), like.shape[1])
        return torch.full((rows,), value, dtype=dtype, device=like.device)
    assert value.shape == (rows,), f"{name} must have one entry a row"
    assert value.device == like.device, f"{name} must be on the logits' device"
    if dtype == torch.int32:
        assert value.dtype in (torch.int32, torch.int64), f"{name} must be int32 or int64"
        if value.dtype == torch.int64:
            value = value.clamp(min=0, max=like.shape[1]).to(torch.int32)
    else:
        assert value.dtype == dtype, f"{name} must be float32"
    return value.contiguous()


def sample(logits: Tensor, uniform: Tensor, temperature: Tensor | float | None = None, top_k: Tensor | int | None = None,
           top_p: Tensor | float | None = None, min_p: Tensor | float | None = None) -> tuple[Tensor, Tensor]:
    """One token a row.  ``logits`` (B, V) in fp32, bf16 or fp16 on a CUDA device
    (rows may be strided); ``uniform`` (B,) float32 in [0, 1) (below it or NaN
    counts as 0, beyond it draws the last kept entry).  The settings are
    one number for all rows or one a row: ``temperature`` (<= 0 or subnormal:
    greedy, the lowest index among equal logits), ``top_k`` (<= 0: no limit),
    ``top_p`` (>= 1: no limit), ``min_p`` (<= 0 or subnormal: no limit).

    Entries are ordered by logit, ties by lowest index.  top_k keeps the first k;
    top_p of those the shortest leading run whose probability reaches top_p (at
    least one entry); min_p of those the entries at least min_p times as likely as
    the likeliest.  The token is the first kept one, in vocabulary order, at which
    the running sum of the kept probabilities exceeds ``uniform`` times their sum.

    Returns ``token`` (B,) int64 and ``logprob`` (B,) float32, the logarithm of the
    probability the token was drawn with (0 for greedy rows).  A NaN logit counts
    as -inf; a row of nothing but -inf gives token -1, logprob -inf.  Sums are
    64-bit and weights good to 2e-13, whatever the type of the logits."""
    assert logits.ndim == 2, "logits must be (rows, vocabulary)"
    assert logits.dtype in _DTYPES, "logits must be float32, bfloat16 or float16"
    B, V = logits.shape
    assert V > 0, "the vocabulary is empty"
    assert uniform.shape == (B,) and uniform.dtype == torch.float32, "uniform must be one float32 number a row"
    if not logits.is_cuda:
        raise RuntimeError("fpkv samples only with its CUDA kernel; these logits live on " f"{logits.device}")
    assert uniform.device == logits.device, "uniform must be on the logits' device"
    if torch.cuda.current_device() != logits.device.index:
        with torch.cuda.device(logits.device):
            return sample(logits, uniform, temperature, top_k, top_p, min_p)
    if logits.stride(1) != 1 or (B > 1 and logits.stride(0) < V):
        logits = logits.contiguous()
    uniform = uniform.contiguous()
    temperature = _per_row(temperature, "temperature", B, torch.float32, logits)
    top_k = _per_row(top_k, "top_k", B, torch.int32, logits)
    top_p = _per_row(top_p, "top_p", B, torch.float32, logits)
    min_p = _per_row(min_p, "min_p", B, torch.float32, logits)
    token = torch.empty(B, dtype=torch.int64, device=logits.device)
    logprob = torch.empty(B, dtype=torch.float32, device=logits.device)
    ptr = lambda t: t.data_ptr() if t is not None else None
    _lib.check(_lib.lib.fpkv_sample(
        logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), B, V, uniform.data_ptr(), ptr(temperature), ptr(top_k),
        ptr(top_p), ptr(min_p), token.data_ptr(), logprob.data_ptr(),
        torch._C._cuda_getCurrentRawStream(logits.device.index)), "fpkv_sample")
    return token, logprob
