"""One token of each row of logits, from given random numbers, on the HIP kernel.

It replaces the sampling inside model.generate (trainer.py:1544-1568, the answers that a non-differentiable objective
scores), and stands next to token_loss, which scores tokens that are given. The random numbers are an input, so that
a run can be repeated, on any number of sequences at once. Work goes to the current stream of the logits'
device; calls may be captured in a graph.
"""
from __future__ import annotations

import operator
from typing import Union

import torch

from .table import dtype_code
from .token_loss import _call, _check_logits, _check_rows, _fail, _no_tangents

MAX_VOCAB = 1 << 20


def _parameter(what: str, name: str, value, lead, device, dtype):
    """(the number for all rows, the tensor of one for each)"""
    if not torch.is_tensor(value):
        try:
            return (operator.index if dtype == torch.int32 else float)(value), None
        except (TypeError, ValueError, OverflowError):
            _fail(what, f"{name} must be a number or a tensor of one for each row, got {value!r}")
    _check_rows(what, name, value, lead, device, (dtype,))
    return 0, _dense(value)


def _dense(t: torch.Tensor) -> torch.Tensor:
    return t if t.dim() == 1 and t.is_contiguous() else t.reshape(-1).contiguous()


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: Union[float, torch.Tensor] = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
                  min_p: Union[float, torch.Tensor] = 0.0) -> torch.Tensor:
    """A token (...) of each row of logits (..., vocab), int64, drawn from softmax(logits / temperature) by uniform (...),
    fp32 from 0 to 1.

    The distribution is restricted to the top_k largest (0: no limit; equal logits in the order of their tokens), of
    these to the fewest, largest first, that hold top_p of their probability, and of these to those of at least min_p
    times the largest one's. The token is the first, in the order of the vocabulary, up to which the sum of what is left
    exceeds uniform of the whole. Temperature 0 takes the largest logit. Each parameter is a number or a tensor (...) of
    one for each row (fp32; top_k int32).

    Weights are computed in 64 bits and summed as whole numbers of 2^-46 of the largest (2^-42 for the longest
    vocabularies): a row's token does not depend on an order of sums, on the other rows, or on the device. Logits of
    -inf are never drawn, those of +inf share the whole. Rows with a NaN or without a logit above -inf give -1, and so
    do rows whose own parameters are NaN or out of range (a number out of range is refused)."""
    what = "sample_tokens"
    _check_logits(what, logits)
    _no_tangents(what, logits, uniform)
    lead, vocab, device = logits.shape[:-1], logits.shape[-1], logits.device
    if vocab > MAX_VOCAB:
        _fail(what, f"at most {MAX_VOCAB} tokens a row, got {vocab}")
    _check_rows(what, "uniform", uniform, lead, device, (torch.float32,))
    t, ts = _parameter(what, "temperature", temperature, lead, device, torch.float32)
    k, ks = _parameter(what, "top_k", top_k, lead, device, torch.int32)
    p, ps = _parameter(what, "top_p", top_p, lead, device, torch.float32)
    m, ms = _parameter(what, "min_p", min_p, lead, device, torch.float32)
    if ts is None and not (t == 0 or 2.0**-63 <= t < 2.0**64):
        _fail(what, f"temperature must be 0, or from 2^-63 up to 2^64, got {t}")
    if ks is None and not 0 <= k < 2**31:
        _fail(what, f"top_k must not be negative, got {k}")
    for name, x, xs in (("top_p", p, ps), ("min_p", m, ms)):
        if xs is None and not 0.0 <= x <= 1.0:
            _fail(what, f"{name} must be 0 to 1, got {x}")
    tokens = torch.empty(lead, dtype=torch.int64, device=device)
    rows = tokens.numel()
    if rows:
        x = logits if logits.dim() == 2 else logits.detach().reshape(-1, vocab)
        u = _dense(uniform)
        _call(device, "dz_sample_tokens", x.data_ptr(), dtype_code(logits.dtype), rows, vocab, x.stride(0), u.data_ptr(), t, k, p, m,
              *(None if a is None else a.data_ptr() for a in (ts, ks, ps, ms)), tokens.data_ptr())
    return tokens

