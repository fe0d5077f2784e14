"""Attention of sequences that share a prompt, and an 8-bit store of keys and values, on the HIP kernels.

``shared_prefix_attention``  groups of sequences that read their group's prompt, once for all of them, and their own
                             keys, causally: the candidates of an example (trainer.py:1524-1542 repeats the prompt for
                             each), questions after one prompt of demonstrations, answers that are drawn token by
                             token, or, without a prompt, whole causal sequences
``KV``                       keys and values
``QuantizedKV``              the same as e4m3 codes, with a power of two for each token and head
``cache_write``              puts new tokens into a QuantizedKV in place
``cache_read``               gives tokens of one as keys and values of a type

Nothing is recorded by autograd: operands that require a gradient are refused where it records, and an operand
with a forward-mode tangent always. Work goes to the current stream of the operands' device; tensors made on another
stream are the caller's to order, as with torch's own operators. Calls may be captured in a graph.
"""
from __future__ import annotations

import ctypes as C
import operator
import struct
from typing import NamedTuple, Optional, Union

import torch
from torch.autograd import forward_ad

from . import _lib as L
from .table import dtype_code
from .token_loss import _call, _fail, _no_tangents

MAX_WIDTH = 128
MAX_SLOT_STRIDE = 1 << 24

CODES = torch.float8_e4m3fn
SCALES = torch.float8_e8m0fnu


class KV(NamedTuple):
    """Keys and values: (..., heads, slots, width), the width contiguous."""

    k: torch.Tensor
    v: torch.Tensor


class QuantizedKV(NamedTuple):
    """Keys and values as e4m3 codes (..., heads, slots, width) and e8m0 scales (..., heads, slots): code * scale."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, *shape: int, device=None) -> "QuantizedKV":
        """A store of the shape (..., heads, slots, width). What it holds before it is written is not defined."""
        codes = [torch.empty(shape, dtype=torch.uint8, device=device).view(CODES) for _ in range(2)]
        scales = [torch.empty(shape[:-1], dtype=torch.uint8, device=device).view(SCALES) for _ in range(2)]
        return cls(*codes, *scales)


_STORE = "2Q8q2Q8q"
_ATTENTION = struct.Struct("2Q8q" + 2 * _STORE + "2Q8qif")
_KEYS_VALUES = struct.Struct(_STORE)
_NOTHING = (0,) * 20
_NO_SCALES = (0,) * 10


def _rows(t: torch.Tensor):
    """(t of four or five dimensions, its strides but for the width's) where the kernels can read t: the width contiguous,
    rows at multiples of 16 bytes (codes: 8), slots near enough; otherwise those of a copy."""
    s = t.stride()
    es = t.element_size()  # (a power of two)
    if len(s) == 5:
        a, b, c, step, last = s
        low = t.data_ptr() | (a | b | c | step) * es
    else:
        a, b, step, last = s
        low = t.data_ptr() | (a | b | step) * es
    if last != 1 or low & (7 if es == 1 else 15) or step >= MAX_SLOT_STRIDE:
        t = t.clone(memory_format=torch.contiguous_format)
        s = t.stride()
    return t, s[:-1]


def _whole(what: str, name: str, x) -> int:
    try:
        return operator.index(x)
    except TypeError:
        _fail(what, f"{name} must be an integer, got {type(x).__name__}")


def _check_operands(what: str, index: int, tensors) -> None:
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t.get_device() != index:
            _fail(what, f"tensors on cuda:{index} and {t.device}")
        if grad and t.requires_grad:
            _fail(what, "nothing is recorded by autograd: call it under torch.no_grad(), or detach the operands")
    if forward_ad._current_level >= 0:
        _no_tangents(what, *tensors)


def _check_store(what: str, name: str, kv, shape, dtype, index: int) -> bool:
    """Checks a KV or QuantizedKV of a shape (its slots are not looked at); whether it is an 8-bit one."""
    bytes_ = len(kv) == 4
    _check_operands(what, index, kv)
    k, v = kv[0], kv[1]
    got = k.shape
    if v.shape != got or len(got) != len(shape) or got[:-2] != shape[:-2] or got[-1] != shape[-1]:
        _fail(what, f"{name} keys and values must be {(*shape[:-2], 'slots', shape[-1])}, got {tuple(got)} and {tuple(v.shape)}")
    want = CODES if bytes_ else dtype
    if k.dtype != want or v.dtype != want:
        _fail(what, f"{name} keys and values must be {want}, got {k.dtype} and {v.dtype}")
    if bytes_:
        for s in kv[2:]:
            if s.shape != got[:-1] or s.dtype != SCALES:
                _fail(what, f"{name} scales must be {SCALES} {tuple(got[:-1])}, got {s.dtype} {tuple(s.shape)}")
    return bytes_


def _check_int32(what: str, name: str, t: Optional[torch.Tensor], shape, index: int):
    if t is None:
        return None
    if t.dtype != torch.int32 or t.get_device() != index or t.shape != shape:
        _fail(what, f"{name} must be torch.int32 {tuple(shape)} on cuda:{index}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def shared_prefix_attention(q: torch.Tensor, own: Union[KV, QuantizedKV, None], prefix: Union[KV, QuantizedKV, None] = None, *,
                            positions: Optional[torch.Tensor] = None, prefix_lengths: Optional[torch.Tensor] = None,
                            scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k) v over the keys that each query sees, in q's dtype.

    q (groups, sequences, heads, length, width): `length` queries of each sequence. prefix (groups, kv_heads, slots,
    width): keys and values that all sequences of a group read; prefix_lengths (groups), int32: how many of them
    (default: all). own (groups, sequences, kv_heads, slots, width): a sequence's own, of which query t sees the
    first positions + t + 1; positions (groups, sequences), int32: how many were there before the call's tokens
    (default: slots - length). Either store may be missing. Lengths outside of their range are taken as the nearest in
    it; a query that sees nothing gives 0. What lies in slots that a query does not see does not matter to it, infinities and
    NaN included.

    Stores are KV, of q's dtype, or both QuantizedKV. heads is a multiple of kv_heads, the width a multiple of 8 up to
    128; scale (default: width ** -0.5) is positive. Products and sums are fp32, and weights are rounded to q's dtype,
    or less, before they multiply values (for bf16 by 2^-8 of each at most, for fp16 by 2^-11 of each and 2^-36 of the
    largest). The result is laid out like q unless `out` is given. The same call gives the same bits; one of other sizes,
    which is cut for the card in another way, may differ in the last ones. Tensors whose rows do not start at multiples of 16
    bytes (codes: 8) are copied first, `out` has to fit."""
    what = "shared_prefix_attention"
    if not q.is_cuda:
        _fail(what, f"q must live on a GPU, got {q.device}")
    index, dtype = q.get_device(), q.dtype
    code = dtype_code(dtype)
    if q.dim() != 5:
        _fail(what, f"q must be (groups, sequences, heads, length, width), got {tuple(q.shape)}")
    groups, sequences, heads, length, width = q.shape
    _check_operands(what, index, (q,) if out is None else (q, out))
    some = own if own is not None else prefix
    if some is None:
        _fail(what, "neither own keys nor a prefix")
    kv_heads = some[0].shape[-3] if some[0].dim() > 2 else 0
    if kv_heads < 1 or heads % kv_heads:
        _fail(what, f"heads ({heads}) is not a multiple of the stores' ({kv_heads})")
    slots = prefix_slots = 0
    if own is not None:
        own_bytes = _check_store(what, "own", own, (groups, sequences, kv_heads, 0, width), dtype, index)
        slots = own[0].shape[3]
    if prefix is not None:
        prefix_bytes = _check_store(what, "prefix", prefix, (groups, kv_heads, 0, width), dtype, index)
        prefix_slots = prefix[0].shape[2]
        if own is not None and own_bytes != prefix_bytes:
            _fail(what, "one of own and prefix is an 8-bit store and the other is not")
    positions = _check_int32(what, "positions", positions, (groups, sequences), index)
    prefix_lengths = _check_int32(what, "prefix_lengths", prefix_lengths, (groups,), index)
    if scale is None:
        scale = width ** -0.5 if width else 1.0
    else:
        try:
            scale = float(scale)
        except (TypeError, ValueError, OverflowError):
            _fail(what, f"scale must be a number, got {scale!r}")
        if not 0.0 < scale <= 2.0**126:
            _fail(what, f"scale must be positive, 2^126 at most, got {scale}")
    if out is None:
        out = torch.empty_like(q)
        if out.stride(-1) != 1 or width * out.element_size() % 16:
            out = torch.empty(q.shape, dtype=dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != dtype:
        _fail(what, f"out must be {dtype} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
    elif out.stride(-1) != 1:
        _fail(what, "the width of out must be contiguous")
    if not q.numel():
        return out
    if not slots and not prefix_slots:
        return out.zero_()
    q, qs = _rows(q)
    own_f = prefix_f = _NOTHING
    if slots:
        k, ks = _rows(own[0])
        v, vs = _rows(own[1])
        own_f = (k.data_ptr(), v.data_ptr(), *ks, *vs, *_NO_SCALES) if not own_bytes else \
            (k.data_ptr(), v.data_ptr(), *ks, *vs, own[2].data_ptr(), own[3].data_ptr(), *own[2].stride(), *own[3].stride())
    if prefix_slots:
        pk, (a, b, c) = _rows(prefix[0])
        pv, (d, e, f) = _rows(prefix[1])
        prefix_f = (pk.data_ptr(), pv.data_ptr(), a, 0, b, c, d, 0, e, f, *_NO_SCALES)
        if prefix_bytes:
            a, b, c = prefix[2].stride()
            d, e, f = prefix[3].stride()
            prefix_f = (*prefix_f[:10], prefix[2].data_ptr(), prefix[3].data_ptr(), a, 0, b, c, d, 0, e, f)
    args = _ATTENTION.pack(q.data_ptr(), out.data_ptr(), *qs, *out.stride()[:4], *own_f, *prefix_f,
                           0 if positions is None else positions.data_ptr(), 0 if prefix_lengths is None else prefix_lengths.data_ptr(),
                           groups, sequences, heads, kv_heads, length, width, slots, prefix_slots, code, scale)
    need = C.c_int64()
    L.call("dz_shared_prefix_attention_workspace", args, C.byref(need))
    need = need.value
    if need:
        work = torch.empty(need, dtype=torch.uint8, device=q.device)
        _call(q.device, "dz_shared_prefix_attention", args, work.data_ptr(), need)
    else:
        _call(q.device, "dz_shared_prefix_attention", args, None, 0)
    return out


def _one_lead(what: str, t: torch.Tensor, n: int):
    """t's strides of (batch, unused, ...) with its first n dimensions taken as one: the batch's is that of the innermost
    of them that has more than one, and each further one steps over all of those inside of it."""
    s = t.stride()
    shape = t.shape
    lead = span = None  # the batch's stride, and what the next dimension has to step over
    for i in range(n - 1, -1, -1):
        if shape[i] == 1:
            continue
        if lead is None:
            lead = span = s[i]
        elif s[i] != span:
            _fail(what, "the cache's leading dimensions must be one by their strides")
        span *= shape[i]
    return lead or 0, 0, s[n], s[n + 1]


def _cache_fields(what: str, cache):
    """(batch, dimensions before the heads, the fields of dz_keys_values)"""
    if not isinstance(cache, QuantizedKV):
        _fail(what, f"the cache must be a QuantizedKV, got {type(cache).__name__}")
    k, v, k_scale, v_scale = cache
    index = k.get_device()
    if index < 0:
        _fail(what, f"the cache must live on a GPU, got {k.device}")
    shape = k.shape
    n = len(shape) - 3
    if n < 0:
        _fail(what, f"the cache must be (..., heads, slots, width), got {tuple(shape)}")
    _check_store(what, "cache", cache, shape, None, index)
    ks, vs, kss, vss = k.stride(), v.stride(), k_scale.stride(), v_scale.stride()
    if ks[-1] != 1 or vs[-1] != 1:
        _fail(what, "the width of the cache must be contiguous")
    if n == 1:
        return shape[0], 1, (k.data_ptr(), v.data_ptr(), ks[0], 0, ks[1], ks[2], vs[0], 0, vs[1], vs[2], k_scale.data_ptr(), v_scale.data_ptr(),
                             kss[0], 0, kss[1], kss[2], vss[0], 0, vss[1], vss[2])
    batch = 1
    for x in shape[:n]:
        batch *= x
    return batch, n, (k.data_ptr(), v.data_ptr(), *_one_lead(what, k, n), *_one_lead(what, v, n), k_scale.data_ptr(), v_scale.data_ptr(),
                      *_one_lead(what, k_scale, n), *_one_lead(what, v_scale, n))


def cache_write(cache: QuantizedKV, k: torch.Tensor, v: torch.Tensor, positions: Union[int, torch.Tensor]) -> None:
    """Puts k and v (..., heads, length, width), fp32, fp16 or bf16, into the cache in place, from slot `positions` on: a
    number for all sequences, or int32 (...), one for each (tokens that fall outside of the cache are left out then).

    A row (one token's head) is kept as code * 2^e: e the least, from -100, that leaves nothing above 448, and codes
    rounded to the nearest e4m3 number, ties to even (e = 0 for a row of zeros). Numbers beyond 240 * 2^8 (fp16) or
    240 * 2^120 (the others), the last before a power of two that the type does not have, are kept as that. A row with an
    infinity or a NaN becomes NaN."""
    what = "cache_write"
    batch, n, fields = _cache_fields(what, cache)
    shape, got = cache.k.shape, k.shape
    heads, slots, width = shape[n:]
    index = cache.k.get_device()
    _check_operands(what, index, (k, v))
    code = dtype_code(k.dtype)
    if got != v.shape or v.dtype != k.dtype or len(got) != n + 3 or got[:-2] != shape[:-2] or got[-1] != width:
        _fail(what, f"k and v must be alike, {(*shape[:-2], 'length', width)}, got {k.dtype} {tuple(got)} and {v.dtype} {tuple(v.shape)}")
    length = got[-2]
    at, position = None, 0
    if torch.is_tensor(positions):
        at = _check_int32(what, "positions", positions, shape[:n], index)
    else:
        position = _whole(what, "positions", positions)
    if not k.numel():
        return
    if at is None and not 0 <= position <= slots - length:
        _fail(what, f"tokens {position} to {position + length} do not fit {slots} slots")
    if n > 1:
        k, v = k.flatten(0, n - 1), v.flatten(0, n - 1)
    elif n == 0:
        k, v = k.unsqueeze(0), v.unsqueeze(0)
    k, (a, b, c) = _rows(k)
    v, (d, e, f) = _rows(v)
    _call(k.device, "dz_cache_write", _KEYS_VALUES.pack(k.data_ptr(), v.data_ptr(), a, 0, b, c, d, 0, e, f, *_NO_SCALES),
          _KEYS_VALUES.pack(*fields), code, batch, heads, length, width, slots, None if at is None else at.data_ptr(), position)


def cache_read(cache: QuantizedKV, length: int, dtype: torch.dtype, start: int = 0) -> KV:
    """Slots start .. start + length - 1 of the cache as keys and values (..., heads, length, width) of a dtype."""
    what = "cache_read"
    batch, n, fields = _cache_fields(what, cache)
    shape = cache.k.shape
    heads, slots, width = shape[n:]
    code = dtype_code(dtype)
    length, start = _whole(what, "length", length), _whole(what, "start", start)
    if length < 0 or start < 0 or start + length > slots:
        _fail(what, f"slots {start} to {start + length} of {slots}")
    shape, device = (*shape[:-2], length, width), cache.k.device
    k, v = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
    if k.numel():
        s = (heads * length * width, 0, length * width, width)
        _call(device, "dz_cache_read", _KEYS_VALUES.pack(*fields), _KEYS_VALUES.pack(k.data_ptr(), v.data_ptr(), *s, *s, *_NO_SCALES), code,
              batch, heads, length, width, slots, start)
    return KV(k, v)
