"""What is read of a model's distributions over the vocabulary, on the HIP kernels.

``token_logprobs``        log probabilities of given tokens, the rows' entropies and their largest
                          alternatives, differentiable in the logits
``topk_distill``          the distance to a teacher of which the largest logits were kept
                          (``token_logprobs(..., top=k)`` records them), differentiable in the logits
``linear_token_logprobs`` log probabilities and entropies straight from the last hidden states and
                          the language-model head, under no_grad: the logits are not stored
``token_logprobs_grad``, ``topk_distill_grad``   value and gradient in one call, for callers that
                          know the rows' weights beforehand (the logits are then read once)

They replace log_softmax, gather and mask of the option loss (trainer.py:1477-1500 and its copy
:497-520). Leading dimensions are rows: logits (..., vocab) go with tokens (...). The vocabulary
dimension has to be contiguous; rows may be strided (``logits[:, :-1]`` is read in place). Results are
fp32: a row's sums are kept in fp32, and rounding them to a 16-bit type would leave a log probability
of -10 with a step of 1/16 (bf16).

Derivatives are reverse-mode, and first order; an operand with a forward-mode tangent is refused.

Work goes to the current stream of the logits' device; tensors made on another stream are the
caller's to order, as with torch's own operators.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn.functional as F

from . import _lib as L
from ._lib import DzError
from .table import _ptr, dtype_code, stream_handle

IGNORE_INDEX = -100  # the masked label of shift_option_labels
MAX_TOP = 128
MAX_TEACHER = 512


class TokenLogprobs(NamedTuple):
    """Per row: the token's log probability, the entropy and, with top > 0, the largest log
    probabilities with their tokens (else None)."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _fail(what: str, why: str):
    raise DzError(f"{what}: {why}")


def _check_logits(what: str, logits: torch.Tensor) -> int:
    if not logits.is_cuda:
        _fail(what, f"logits must live on a GPU, got {logits.device}")
    code = dtype_code(logits.dtype)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        _fail(what, f"logits must be (..., vocab), got {tuple(logits.shape)}")
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        _fail(what, "the vocabulary dimension of the logits must be contiguous")
    return code


def _check_rows(what: str, name: str, t: torch.Tensor, lead, device, dtypes) -> None:
    if t.device != device:
        _fail(what, f"{name} must be on {device}, got {t.device}")
    if t.dtype not in dtypes:
        _fail(what, f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.shape != lead:
        _fail(what, f"{name} must have shape {tuple(lead)}, got {tuple(t.shape)}")


def _no_tangents(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Derivatives are reverse-mode only: results of a dual tensor would lack its tangent without a word.
    (Dual tensors exist only inside a dual level; calls outside of one cost a comparison.)"""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                _fail(what, "forward-mode derivatives are not supported (an operand carries a tangent)")


_INT = (torch.int64, torch.int32)
_F32 = (torch.float32,)


def _rows(t: Optional[torch.Tensor], n: int, inner: int):
    """A tensor of n leading dimensions as (address, batch stride, row stride), and what keeps it alive.
    More than two are made one: a view where the strides allow it, else a copy."""
    if t is None:
        return None, 0, 0, None
    if n > 2:
        t = t.reshape(-1, *t.shape[n:]) if inner else t.reshape(-1)
    s = t.stride()
    if n == 2:
        return t.data_ptr(), s[0], s[1], t
    return t.data_ptr(), 0, s[0] if n else 0, t


def _batch_length(lead) -> Tuple[int, int]:
    return (lead[0], lead[1]) if len(lead) == 2 else (1, lead.numel())


def _call(device, name: str, *args) -> None:
    """The entry point on the device's current stream."""
    if device.index == torch._C._cuda_getDevice():
        L.call(name, *args, stream_handle())
    else:
        with torch.cuda.device(device):
            L.call(name, *args, stream_handle())


def _grad_like(logits: torch.Tensor) -> torch.Tensor:
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


def _score(logits, tokens, top, ignore_index, weights, entropy_weights, grad):
    """One launch over checked operands. grad: a tensor to write, or None."""
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    n = len(lead)
    batch, length = _batch_length(lead)
    lp = logits.new_empty(lead, dtype=torch.float32)
    ent = logits.new_empty(lead, dtype=torch.float32)
    tlp = ttok = None
    if top:
        tlp = logits.new_empty((*lead, top), dtype=torch.float32)
        ttok = logits.new_empty((*lead, top), dtype=torch.int64)
    if batch * length:
        x, x_b, x_l, _x = _rows(logits, n, 1)
        t, t_b, t_l, _t = _rows(tokens, n, 0)
        w, w_b, w_l, _w = _rows(weights, n, 0)
        u, u_b, u_l, _u = _rows(entropy_weights, n, 0)
        g, g_b, g_l, _g = _rows(grad, n, 1)
        _call(logits.device, "dz_token_logprobs", x, dtype_code(logits.dtype), batch, length, vocab, x_b, x_l, t, t_b, t_l,
              ignore_index, top, lp.data_ptr(), ent.data_ptr(), _ptr(tlp), _ptr(ttok), w, w_b, w_l, u, u_b, u_l, g, g_b, g_l)
    return lp, ent, tlp, ttok


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, ignore_index):
        lp, ent, tlp, ttok = _score(logits, tokens, top, ignore_index, None, None, None)
        ctx.save_for_backward(logits, tokens)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(tlp, ttok)
        return lp, ent, tlp, ttok

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_lp, d_ent, _tlp, _ttok):
        logits, tokens = ctx.saved_tensors
        _no_tangents("token_logprobs' backward", d_lp, d_ent)
        if d_lp is None and d_ent is None:
            return None, None, None, None
        grad = _grad_like(logits)
        _score(logits, tokens, 0, ctx.ignore_index, d_lp, d_ent, grad)
        return grad, None, None, None


def _score_checked(what, logits, tokens, top, weights=None, entropy_weights=None):
    _check_logits(what, logits)
    _no_tangents(what, logits, weights, entropy_weights)
    _check_rows(what, "tokens", tokens, logits.shape[:-1], logits.device, _INT)
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        _fail(what, f"top must be 0 to {min(MAX_TOP, logits.shape[-1])}, got {top}")
    return tokens if tokens.dtype == torch.int64 else tokens.long()


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0,
                   ignore_index: int = IGNORE_INDEX) -> TokenLogprobs:
    """log softmax(logits)[tokens] and the entropy of softmax(logits) for every row, with the `top`
    largest log probabilities and their tokens, largest first and equal ones by token.

    Rows whose token is ignore_index are not read: 0, 0, -inf and -1. Another token outside the
    vocabulary gives NaN, and so does a row without a distribution (NaN, +inf, or nothing above -inf).
    Gradients flow to the logits through logprobs and entropy; the alternatives are a report."""
    tokens = _score_checked("token_logprobs", logits, tokens, top)
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, top, ignore_index))
    return TokenLogprobs(*_score(logits, tokens, top, ignore_index, None, None, None))


def token_logprobs_grad(logits: torch.Tensor, tokens: torch.Tensor, weights: Optional[torch.Tensor] = None,
                        entropy_weights: Optional[torch.Tensor] = None, *,
                        ignore_index: int = IGNORE_INDEX) -> Tuple[TokenLogprobs, torch.Tensor]:
    """token_logprobs, and the gradient of sum(weights logprobs) + sum(entropy_weights entropy) with
    respect to the logits, in their dtype. Weights are fp32, shaped like tokens; None stands for zeros.
    Nothing is recorded by autograd."""
    what = "token_logprobs_grad"
    tokens = _score_checked(what, logits, tokens, 0, weights, entropy_weights)
    if weights is None and entropy_weights is None:
        _fail(what, "weights or entropy_weights are needed")
    for name, w in (("weights", weights), ("entropy_weights", entropy_weights)):
        if w is not None:
            _check_rows(what, name, w, logits.shape[:-1], logits.device, _F32)
    with torch.no_grad():
        grad = _grad_like(logits)
        out = _score(logits, tokens, 0, ignore_index, weights, entropy_weights, grad)
    return TokenLogprobs(*out), grad


def _distill(logits, values, tokens, temperature, normalize, weights, grad):
    lead = logits.shape[:-1]
    n = len(lead)
    batch, length = _batch_length(lead)
    loss = logits.new_empty(lead, dtype=torch.float32)
    if batch * length:
        x, x_b, x_l, _x = _rows(logits, n, 1)
        w, w_b, w_l, _w = _rows(weights, n, 0)
        g, g_b, g_l, _g = _rows(grad, n, 1)
        _call(logits.device, "dz_topk_distill", x, dtype_code(logits.dtype), batch, length, logits.shape[-1], x_b, x_l,
              values.data_ptr(), tokens.data_ptr(), values.shape[-1], temperature, int(normalize), loss.data_ptr(), w, w_b, w_l,
              g, g_b, g_l)
    return loss


class _TopkDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, tokens, temperature, normalize):
        ctx.save_for_backward(logits, values, tokens)
        ctx.how = (temperature, normalize)
        return _distill(logits, values, tokens, temperature, normalize, None, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss):
        logits, values, tokens = ctx.saved_tensors
        _no_tangents("topk_distill's backward", d_loss)
        grad = _grad_like(logits)
        _distill(logits, values, tokens, *ctx.how, d_loss, grad)
        return grad, None, None, None, None


def _distill_checked(what, logits, values, tokens, temperature, weights=None):
    _check_logits(what, logits)
    _no_tangents(what, logits, values, weights)
    lead, k = logits.shape[:-1], values.shape[-1] if values.dim() else 0
    if not 1 <= k <= MAX_TEACHER:
        _fail(what, f"a teacher has 1 to {MAX_TEACHER} entries a row, got {k}")
    _check_rows(what, "values", values, (*lead, k), logits.device, (torch.float32, torch.float16, torch.bfloat16))
    _check_rows(what, "tokens", tokens, (*lead, k), logits.device, _INT)
    if not (2.0**-63 <= temperature < 2.0**64):
        _fail(what, f"temperature must be positive and finite, and so its square (2^-63 to 2^64), got {temperature}")
    if values.requires_grad and torch.is_grad_enabled():
        _fail(what, "the teacher's values take no gradient (detach them)")
    return values.detach().float().contiguous(), tokens.long().contiguous()


def topk_distill(logits: torch.Tensor, values: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0,
                 normalize: bool = True) -> torch.Tensor:
    """The distance of softmax(logits / T) to a teacher of which some entries were kept, per row:

        T^2 sum_j w_j (log w_j - log softmax(logits / T)[tokens_j])

    (T from 2^-63 up to 2^64, so that its square is one of fp32.)
    values, tokens: (..., k), the teacher's entries: logits, or log probabilities (both give the same
    with normalize=True, where w = softmax(values / T) over the row's entries; with normalize=False
    w = exp(values), log probabilities at temperature T, and the rest of the teacher's mass is left
    out). A token of -1 is no entry; a row without entries is not read and gives 0. Entries of weight 0
    (a value of -inf) add nothing; a token named twice counts twice. A token outside the vocabulary
    and a value of NaN or +inf give NaN. Gradients flow to the logits."""
    values, tokens = _distill_checked("topk_distill", logits, values, tokens, temperature)
    if logits.requires_grad and torch.is_grad_enabled():
        return _TopkDistill.apply(logits, values, tokens, temperature, normalize)
    return _distill(logits, values, tokens, temperature, normalize, None, None)


def topk_distill_grad(logits: torch.Tensor, values: torch.Tensor, tokens: torch.Tensor, weights: torch.Tensor, *,
                      temperature: float = 1.0, normalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """topk_distill, and the gradient of sum(weights loss) with respect to the logits, in their dtype.
    weights: fp32, one per row. Nothing is recorded by autograd."""
    what = "topk_distill_grad"
    values, tokens = _distill_checked(what, logits, values, tokens, temperature, weights)
    _check_rows(what, "weights", weights, logits.shape[:-1], logits.device, _F32)
    with torch.no_grad():
        grad = _grad_like(logits)
        loss = _distill(logits, values, tokens, temperature, normalize, weights, grad)
    return loss, grad


def linear_token_logprobs(hidden: torch.Tensor, weight: torch.Tensor, tokens: torch.Tensor, *,
                          ignore_index: int = IGNORE_INDEX) -> TokenLogprobs:
    """token_logprobs of the logits hidden @ weight.T, which are not stored (and not rounded: products
    and sums are fp32). hidden (..., width) and weight (vocab, width) of one dtype; the width has to be
    contiguous. Ignored rows give 0 (of many rows, they are not multiplied).

    A parameter requires a gradient: score under torch.no_grad(). Where autograd records (grad mode is
    on, and hidden or weight require a gradient) the logits are F.linear's, stored and rounded to the
    operands' dtype, and token_logprobs takes them from there: a logit of 8 is off by up to 2^-5 in
    bf16, and log probabilities differ by as much from those of the kernel."""
    what = "linear_token_logprobs"
    if not hidden.is_cuda:
        _fail(what, f"hidden must live on a GPU, got {hidden.device}")
    _no_tangents(what, hidden, weight)
    code = dtype_code(hidden.dtype)
    if weight.device != hidden.device or weight.dtype != hidden.dtype:
        _fail(what, f"weight is {weight.dtype} on {weight.device}, hidden {hidden.dtype} on {hidden.device}")
    if hidden.dim() < 1 or weight.dim() != 2 or weight.shape[1] != hidden.shape[-1] or not weight.numel():
        _fail(what, f"hidden (..., width) and weight (vocab, width) do not fit: {tuple(hidden.shape)}, {tuple(weight.shape)}")
    _check_rows(what, "tokens", tokens, hidden.shape[:-1], hidden.device, _INT)
    vocab, width = weight.shape
    if weight.stride(1) != 1 and width > 1:
        _fail(what, "the width of the weight must be contiguous")
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return token_logprobs(F.linear(hidden, weight), tokens, ignore_index=ignore_index)
    lead = tokens.shape
    h = hidden.reshape(-1, width)
    if h.stride(1) != 1 and width > 1:
        h = h.contiguous()
    t = tokens.reshape(-1).long().contiguous()
    lp = hidden.new_empty(lead, dtype=torch.float32)
    ent = hidden.new_empty(lead, dtype=torch.float32)
    rows = h.shape[0]
    if rows:
        need = C.c_int64()
        L.call("dz_linear_token_logprobs_workspace", code, rows, width, vocab, C.byref(need))
        work = torch.empty(need.value, dtype=torch.uint8, device=hidden.device)
        _call(hidden.device, "dz_linear_token_logprobs", h.data_ptr(), weight.data_ptr(), code, rows, width, vocab, h.stride(0),
              weight.stride(0), t.data_ptr(), ignore_index, lp.data_ptr(), ent.data_ptr(), work.data_ptr(), need.value)
    return TokenLogprobs(lp, ent, None, None)
