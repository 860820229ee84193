"""One token per row of logits under temperature, top-k, top-p and min-p, from
given random numbers, in one kernel without a sort.

    e_i = exp((l_i - max l) / T),  Z = sum e          (e = 1 where l is the maximum)
    order: the larger logit first, among equal ones the lower index
    kept:  rank < top_k,  (sum of e ahead) < top_p Z,  e >= min_p;  the first of the order always
    token = the kept token with the largest e_i / noise_i (the lowest index among equal ones),  prob = e_token / Z

Every filter looks at the whole distribution (top-p is not renormalised after
top-k).  ``noise`` holds independent Exp(1) random numbers
(``torch.empty(rows, V).exponential_()``): the token is then drawn with
probability e_i / (sum of the kept e).  Equal calls give equal results.  The
order in which Z is summed follows the number of rows and their alignment, so
that the same row in another batch may have another last bit of ``prob``, and
another token where top_p Z lies within that rounding of a sum of e.  ``prob``
is the token's probability before the filters.  Neither output has a gradient.
"""
from __future__ import annotations

import torch

from . import _native as N

_VOCAB_LIMIT = 2**29


def _option(a, name, value, rows, device, dtypes, cast):
    """A filter's value: one Python number for all rows, or a tensor [rows]; returns the tensor that must stay alive."""
    if not isinstance(value, torch.Tensor):
        try:
            setattr(a, name + "_all", cast(value))
        except (TypeError, ValueError, OverflowError):
            raise TypeError(f"{name} must be a number, a tensor [{rows}] or None, got {value!r}") from None
        return
    if value.ndim != 1 or value.shape[0] != rows or value.dtype not in dtypes or not value.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{rows}] tensor of {' or '.join(map(str, dtypes))}, got "
                         f"{tuple(value.shape)} {value.dtype}")
    if value.device != device:
        raise ValueError("all sampling tensors must share one CUDA device")
    setattr(a, name, value.data_ptr())


def _whole(value):
    """A whole number as 64 bits hold it: what is beyond (a top_k of every token) must not wrap around."""
    return max(-1, min(int(value), 2**62))


def sample(logits, noise, *, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """Draw one token per row; returns ``(token int64 [rows], prob fp32 [rows])``.

    logits [rows, V] bf16 or fp32 and noise [rows, V] fp32 (positive), rows contiguous, any row stride from V up (or 0).
    temperature, top_p, min_p: numbers or fp32 tensors [rows]; top_k: int or int32 / int64 tensor [rows]; None,
    top_k <= 0 or top_p >= 1: no such filter.  temperature below 1e-37 (0, negative): the most likely token, prob 1.
    NaN logits count as -inf and +inf as the largest fp32 value; a row with nothing above -inf gives token -1, prob 0.
    """
    fast = N.host()
    if fast is not None:
        out = fast.sample(logits, noise, temperature, top_k, top_p, min_p, _VOCAB_LIMIT)
        if out is not None:
            return out
    if logits.ndim != 2 or not 1 <= logits.shape[1] <= _VOCAB_LIMIT:
        raise ValueError(f"logits must be [rows, V] with V >= 1, got {tuple(logits.shape)}")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"logits must be bf16 or fp32, got {logits.dtype}")
    if noise.shape != logits.shape or noise.dtype != torch.float32:
        raise ValueError(f"noise must be fp32 {tuple(logits.shape)}, got {tuple(noise.shape)} {noise.dtype}")
    rows, V = logits.shape
    device = logits.device
    if noise.device != device:
        raise ValueError("all sampling tensors must share one CUDA device")
    if V > 1 and (logits.stride(1) != 1 or noise.stride(1) != 1):
        raise ValueError("the rows of logits and noise must be contiguous")
    a = N.KdnSampleArgs()
    a.rows, a.V = rows, V
    _option(a, "temperature", temperature, rows, device, (torch.float32,), float)
    _option(a, "top_k", 0 if top_k is None else top_k, rows, device, (torch.int32, torch.int64), _whole)
    _option(a, "top_p", 1.0 if top_p is None else top_p, rows, device, (torch.float32,), float)
    _option(a, "min_p", 0.0 if min_p is None else min_p, rows, device, (torch.float32,), float)
    if not logits.is_cuda:
        N.require_cuda(logits)
    lib = N.load_library()
    a.logits_bf16 = logits.dtype == torch.bfloat16
    a.top_k_i64 = isinstance(top_k, torch.Tensor) and top_k.dtype == torch.int64
    a.logits, a.noise = logits.data_ptr(), noise.data_ptr()
    a.logits_stride, a.noise_stride = logits.stride(0), noise.stride(0)
    token = noise.new_empty(rows, dtype=torch.int64)
    prob = noise.new_empty(rows)
    a.token, a.prob = token.data_ptr(), prob.data_ptr()
    N.launch(lib.kdn_sample, a, logits, "kdn_sample")
    return token, prob


__all__ = ("sample",)
