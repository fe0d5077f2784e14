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
import struct
from typing import NamedTuple, Optional, Tuple, Union

import torch

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


def _fits(t: torch.Tensor, align: int) -> bool:
    """Whether the kernels read t where it is: width contiguous, rows at multiples of `align` bytes, slots near enough."""
    s = t.stride()
    es = t.element_size()
    if s[-1] != 1 or t.data_ptr() % align or s[-2] >= MAX_SLOT_STRIDE:
        return False
    for x in s[:-1]:
        if x * es % align:
            return False
    return True


def _placed(t: torch.Tensor, align: int) -> torch.Tensor:
    return t if _fits(t, align) else t.clone(memory_format=torch.contiguous_format)


def _check_operands(what: str, device, *tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None:
            if t.device != device:
                _fail(what, f"tensors on {device} and {t.device}")
            if t.requires_grad and torch.is_grad_enabled():
                _fail(what, "nothing is recorded by autograd: call it under torch.no_grad(), or detach the operands")
    _no_tangents(what, *tensors)


def _check_store(what: str, name: str, kv, lead: Tuple[int, ...], width: int, dtype, device) -> bool:
    """Checks a KV or QuantizedKV whose leading dimensions (and heads) are `lead`; whether it is an 8-bit one."""
    bytes_ = isinstance(kv, QuantizedKV) or (not isinstance(kv, KV) and len(kv) == 4)
    k, v = kv[0], kv[1]
    _check_operands(what, device, *kv)
    if k.shape != v.shape or k.dim() != len(lead) + 2 or tuple(k.shape[:-2]) != lead or k.shape[-1] != width:
        _fail(what, f"{name} keys and values must be {(*lead, 'slots', width)}, got {tuple(k.shape)} and {tuple(v.shape)}")
    want = CODES if bytes_ else dtype
    if k.dtype != want or v.dtype != want:
        _fail(what, f"{name} keys and values must be {want}, got {k.dtype} and {v.dtype}")
    if bytes_:
        for s in kv[2:]:
            if s.shape != k.shape[:-1] or s.dtype != SCALES:
                _fail(what, f"{name} scales must be {SCALES} {tuple(k.shape[:-1])}, got {s.dtype} {tuple(s.shape)}")
    return bytes_


def _place_store(kv, bytes_: bool):
    """The store's tensors where the kernels can read them (a copy of those that they cannot)."""
    if not bytes_:
        return _placed(kv[0], 16), _placed(kv[1], 16)
    return _placed(kv[0], 8), _placed(kv[1], 8), kv[2], kv[3]


def _packed(kv, four) -> tuple:
    """The store's fields in dz_keys_values' order; `four` makes four strides of a tensor's (without the width's)."""
    k, v = four(kv[0].stride()[:-1]), four(kv[1].stride()[:-1])
    if len(kv) == 2:
        return (kv[0].data_ptr(), kv[1].data_ptr(), *k, *v, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    return (kv[0].data_ptr(), kv[1].data_ptr(), *k, *v, kv[2].data_ptr(), kv[3].data_ptr(), *four(kv[2].stride()), *four(kv[3].stride()))


def _check_int32(what: str, name: str, t: Optional[torch.Tensor], shape, device):
    if t is None:
        return None
    if t.dtype != torch.int32 or t.device != device or tuple(t.shape) != tuple(shape):
        _fail(what, f"{name} must be torch.int32 {tuple(shape)} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
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
    it; a query that sees nothing gives 0. What lies in slots that no query of a sequence sees does not matter.

    Stores are KV, of q's dtype, or both QuantizedKV. heads is a multiple of kv_heads, the width a multiple of 8 up to
    128; scale (default: width ** -0.5) is positive. Products and sums are fp32, and weights are rounded to q's dtype
    before they multiply values. The result is laid out like q unless `out` is given. Tensors whose rows do not
    start at multiples of 16 bytes (codes: 8) are copied first, `out` has to fit."""
    what = "shared_prefix_attention"
    if not q.is_cuda:
        _fail(what, f"q must live on a GPU, got {q.device}")
    device = q.device
    code = dtype_code(q.dtype)
    if q.dim() != 5:
        _fail(what, f"q must be (groups, sequences, heads, length, width), got {tuple(q.shape)}")
    groups, sequences, heads, length, width = q.shape
    _check_operands(what, device, q, out)
    if own is None and prefix is None:
        _fail(what, "neither own keys nor a prefix")
    kv_heads = (own if own is not None else prefix)[0].shape[-3] if (own if own is not None else prefix)[0].dim() > 2 else 0
    if kv_heads < 1 or heads % kv_heads:
        _fail(what, f"heads ({heads}) is not a multiple of the stores' ({kv_heads})")
    slots = prefix_slots = 0
    own_bytes = prefix_bytes = None
    if own is not None:
        own_bytes = _check_store(what, "own", own, (groups, sequences, kv_heads), width, q.dtype, device)
        slots = own[0].shape[-2]
    if prefix is not None:
        prefix_bytes = _check_store(what, "prefix", prefix, (groups, kv_heads), width, q.dtype, device)
        prefix_slots = prefix[0].shape[-2]
    if own_bytes is not None and prefix_bytes is not None and own_bytes != prefix_bytes:
        _fail(what, "one of own and prefix is an 8-bit store and the other is not")
    positions = _check_int32(what, "positions", positions, (groups, sequences), device)
    prefix_lengths = _check_int32(what, "prefix_lengths", prefix_lengths, (groups,), device)
    if out is None:
        out = torch.empty_like(q)
        if not _fits(out, 16):
            out = torch.empty(q.shape, dtype=q.dtype, device=device)
    elif out.shape != q.shape or out.dtype != q.dtype:
        _fail(what, f"out must be {q.dtype} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
    elif out.stride(-1) != 1 and width > 1:
        _fail(what, "the width of out must be contiguous")
    if not q.numel():
        return out
    if not slots and not prefix_slots:
        return out.zero_()
    q = _placed(q, 16)
    own_f = prefix_f = _NOTHING
    if slots:
        own = _place_store(own, own_bytes)
        own_f = _packed(own, tuple)
    if prefix_slots:
        prefix = _place_store(prefix, prefix_bytes)
        prefix_f = _packed(prefix, lambda s: (s[0], 0, s[1], s[2]))
    args = _ATTENTION.pack(q.data_ptr(), out.data_ptr(), *q.stride()[:4], *out.stride()[:4], *own_f, *prefix_f,
                           0 if positions is None else positions.data_ptr(), 0 if prefix_lengths is None else prefix_lengths.data_ptr(),
                           groups, sequences, heads, kv_heads, length, width, slots, prefix_slots, code,
                           width ** -0.5 if scale is None else scale)
    need = C.c_int64()
    L.call("dz_shared_prefix_attention_workspace", args, C.byref(need))
    work = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
    _call(device, "dz_shared_prefix_attention", args, work.data_ptr() if need.value else None, need.value)
    return out


def _cache_operands(what: str, cache):
    if not isinstance(cache, QuantizedKV):
        _fail(what, f"the cache must be a QuantizedKV, got {type(cache).__name__}")
    k = cache.k
    if not k.is_cuda:
        _fail(what, f"the cache must live on a GPU, got {k.device}")
    if k.dim() < 3:
        _fail(what, f"the cache must be (..., heads, slots, width), got {tuple(k.shape)}")
    _check_store(what, "cache", cache, tuple(k.shape[:-2]), k.shape[-1], None, k.device)
    for t in cache[:2]:
        if not _fits(t, 8):
            _fail(what, "the cache's rows must be contiguous and start at multiples of 8 bytes")
    batch = 1
    for n in k.shape[:-3]:
        batch *= n
    try:  # one leading dimension: a view, since the cache is written
        return batch, [t.view(batch, *t.shape[k.dim() - 3:]) for t in cache]
    except RuntimeError:
        _fail(what, "the cache's leading dimensions must be one by their strides")


def cache_write(cache: QuantizedKV, k: torch.Tensor, v: torch.Tensor, positions: Union[int, torch.Tensor]) -> None:
    """Puts k and v (..., heads, length, width), fp32, fp16 or bf16, into the cache in place, from slot `positions` on: a
    number for all sequences, or int32 (...), one for each (tokens that fall outside of the cache are left out then).

    A row (one token's head) is kept as code * 2^e: e the least, from -100, that leaves nothing above 448, and codes
    rounded to the nearest e4m3 number, ties to even. fp16 numbers beyond 61440 are kept as that. A row with an infinity
    or a NaN becomes NaN."""
    what = "cache_write"
    batch, store = _cache_operands(what, cache)
    device = cache.k.device
    heads, slots, width = cache.k.shape[-3:]
    lead = cache.k.shape[:-3]
    _check_operands(what, device, k, v)
    code = dtype_code(k.dtype)
    if k.shape != v.shape or v.dtype != k.dtype or k.dim() != cache.k.dim() or k.shape[:-2] != cache.k.shape[:-2] or k.shape[-1] != width:
        _fail(what, f"k and v must be alike, {(*lead, heads, 'length', width)}, got {k.dtype} {tuple(k.shape)} and {v.dtype} {tuple(v.shape)}")
    length = k.shape[-2]
    at, position = None, 0
    if torch.is_tensor(positions):
        at = _check_int32(what, "positions", positions, lead, device)
    else:
        position = positions
    if not k.numel():
        return
    k, v = (_placed(t.reshape(batch, *t.shape[-3:]), 16) for t in (k, v))
    rows = lambda s: (s[0], 0, s[1], s[2])  # noqa: E731
    _call(device, "dz_cache_write", _KEYS_VALUES.pack(*_packed((k, v), rows)), _KEYS_VALUES.pack(*_packed(store, rows)), code, batch, heads,
          length, width, slots, None if at is None else at.data_ptr(), position)


def cache_read(cache: QuantizedKV, length: int, dtype: torch.dtype, start: int = 0) -> KV:
    """Slots start .. start + length - 1 of the cache as keys and values of a dtype, laid out (..., length, heads, width) and
    seen as (..., heads, length, width)."""
    what = "cache_read"
    batch, store = _cache_operands(what, cache)
    device = cache.k.device
    heads, slots, width = cache.k.shape[-3:]
    code = dtype_code(dtype)
    if length < 0 or start < 0 or start + length > slots:
        _fail(what, f"slots {start} to {start + length} of {slots}")
    kv = [torch.empty(batch, length, heads, width, dtype=dtype, device=device).transpose(1, 2) for _ in range(2)]
    if batch * length:
        rows = lambda s: (s[0], 0, s[1], s[2])  # noqa: E731
        _call(device, "dz_cache_read", _KEYS_VALUES.pack(*_packed(store, rows)), _KEYS_VALUES.pack(*_packed(kv, rows)), code, batch, heads,
              length, width, slots, start)
    lead = cache.k.shape[:-3]
    return KV(*(t if len(lead) == 1 else t.unflatten(0, lead) if lead else t[0] for t in kv))
