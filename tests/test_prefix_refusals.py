"""dizo_amd.prefix_attention and sampling without a GPU: what the C ABI and Python refuse, and the structs' layout."""
import os
import subprocess

import pytest
import torch

from dizo_amd import _lib as L
from dizo_amd import prefix_attention as P
from dizo_amd import sampling as S
from dizo_amd._lib import DzError

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 4096  # a pointer that is not NULL; nothing reads through it


def _refused(name, args, *words):
    lib = L.load()
    rc = getattr(lib, name)(*args)
    msg = lib.dz_last_error().decode()
    assert rc < 0 and all(w in msg for w in words), (rc, msg)


def test_structs_are_packed_as_the_header_has_them(tmp_path):
    src = tmp_path / "s.c"
    src.write_text('#include "dizo_amd.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void) { printf("%zu %zu %zu %zu %zu %zu", '
                   "sizeof(dz_keys_values), sizeof(dz_attention), offsetof(dz_attention, own), offsetof(dz_attention, prefix), "
                   "offsetof(dz_attention, groups), offsetof(dz_attention, scale)); return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    kv = P._KEYS_VALUES.size
    assert got == [kv, P._ATTENTION.size, 80, 80 + kv, 80 + 2 * kv + 16, P._ATTENTION.size - 4]


def _store(k=PTR, v=PTR, ks=0, vs=0, s=(6400, 6400, 640, 64), slot=64):
    s = (*s[:3], slot)
    return (k, v, *s, *s, ks, vs, *((100, 100, 10, 1) * 2))


def _attention(**kw):
    a = dict(q=PTR, out=PTR * 64, q_s=(1280, 640, 320, 64), out_s=(1280, 640, 320, 64), own=_store(), prefix=_store(), positions=0, lengths=0,
             groups=2, sequences=2, heads=2, kv_heads=1, length=5, width=64, slots=10, prefix_slots=10, dtype=L.DZ_DTYPE_F16, scale=0.125)
    assert set(kw) <= set(a)
    a.update(kw)
    return P._ATTENTION.pack(a["q"], a["out"], *a["q_s"], *a["out_s"], *a["own"], *a["prefix"], a["positions"], a["lengths"], a["groups"], a["sequences"],
                             a["heads"], a["kv_heads"], a["length"], a["width"], a["slots"], a["prefix_slots"], a["dtype"], a["scale"])


SHAPE_FAULTS = [
    (dict(dtype=5), ["dtype"]),
    (dict(groups=-1), ["groups"]),
    (dict(sequences=1 << 25), ["sequences"]),
    (dict(heads=0), ["heads"]),
    (dict(kv_heads=0), ["kv_heads"]),
    (dict(heads=3, kv_heads=2), ["multiple"]),
    (dict(length=-5), ["length"]),
    (dict(width=60), ["width", "60"]),
    (dict(width=136), ["width"]),
    (dict(width=0), ["width"]),
    (dict(slots=-1), ["slots"]),
    (dict(slots=0, prefix_slots=0), ["neither"]),
    (dict(scale=0.0), ["scale"]),
    (dict(scale=-1.0), ["scale"]),
    (dict(scale=float("inf")), ["scale"]),
    (dict(scale=float("nan")), ["scale"]),
    (dict(groups=1 << 12, sequences=1 << 12, length=1 << 12), ["queries"]),
    (dict(groups=1 << 20, sequences=1 << 9, heads=1, length=1), ["tiles"]),
    (dict(own=_store(ks=PTR, vs=PTR)), ["8-bit"]),
]


@pytest.mark.parametrize("kw, words", SHAPE_FAULTS)
def test_attention_refuses_shapes(kw, words):
    import ctypes as C

    _refused("dz_shared_prefix_attention", (_attention(**kw), None, 0, None), *words)
    _refused("dz_shared_prefix_attention_workspace", (_attention(**kw), C.byref(C.c_int64())), *words)


@pytest.mark.parametrize("kw, words", [
    (dict(q=0), ["q is NULL"]),
    (dict(q=PTR + 8), ["q", "aligned"]),
    (dict(q_s=(1280, 640, 320, 60)), ["q", "multiple"]),
    (dict(q_s=(-1280, 640, 320, 64)), ["q", "negative"]),
    (dict(q_s=(1 << 60, 640, 320, 64)), ["q", "stride"]),
])
def test_attention_refuses_operands(kw, words):
    _refused("dz_shared_prefix_attention", (_attention(**kw), None, 0, None), *words)


def test_attention_of_nothing_is_no_work():
    for kw in (dict(groups=0), dict(sequences=0), dict(length=0)):
        assert L.load().dz_shared_prefix_attention(_attention(q=0, out=0, **kw), None, 0, None) == 0
    _refused("dz_shared_prefix_attention", (None, None, 0, None), "NULL")


def _cache_args(read, **kw):
    a = dict(kv=P._KEYS_VALUES.pack(*_store()), cache=P._KEYS_VALUES.pack(*_store(k=PTR * 64, v=PTR * 128, ks=PTR * 256, vs=PTR * 512)), dtype=L.DZ_DTYPE_BF16,
             batch=2, heads=2, length=5, width=64, slots=10, positions=None, position=0)
    a.update(kw)
    rest = [a["dtype"], a["batch"], a["heads"], a["length"], a["width"], a["slots"]]
    return [a["cache"], a["kv"], *rest, a["position"], None] if read else [a["kv"], a["cache"], *rest, a["positions"], a["position"], None]


@pytest.mark.parametrize("read", [False, True])
@pytest.mark.parametrize("kw, words", [
    (dict(dtype=9), ["dtype"]),
    (dict(batch=-1), ["batch"]),
    (dict(heads=0), ["heads"]),
    (dict(length=-1), ["length"]),
    (dict(width=4), ["width"]),
    (dict(width=256), ["width"]),
    (dict(slots=0), ["slots"]),
    (dict(position=6), ["fit"]),
    (dict(position=-1), ["fit"]),
    (dict(length=11), ["fit"]),
    (dict(batch=1 << 14, heads=1 << 14), ["rows"]),
    (dict(kv=None), ["NULL"]),
    (dict(cache=None), ["NULL"]),
    (dict(kv=P._KEYS_VALUES.pack(*_store(k=0))), ["NULL"]),
    (dict(kv=P._KEYS_VALUES.pack(*_store(k=PTR + 2))), ["aligned"]),
])
def test_cache_refuses(read, kw, words):
    _refused("dz_cache_read" if read else "dz_cache_write", _cache_args(read, **kw), *words)


def test_cache_calls_of_nothing_are_no_work():
    lib = L.load()
    for kw in (dict(batch=0), dict(length=0)):
        assert lib.dz_cache_write(*_cache_args(False, **kw)) == 0 and lib.dz_cache_read(*_cache_args(True, **kw)) == 0


def _sample_args(**kw):
    a = dict(logits=PTR, dtype=L.DZ_DTYPE_F32, rows=3, vocab=10, stride=10, uniform=PTR, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
             ts=None, ks=None, ps=None, ms=None, tokens=PTR, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, words", [
    (dict(dtype=-1), ["dtype"]),
    (dict(rows=-1), ["row count"]),
    (dict(rows=1 << 22), ["row count"]),
    (dict(vocab=0), ["vocab"]),
    (dict(vocab=(1 << 20) + 1), ["vocab"]),
    (dict(temperature=-0.5), ["temperature"]),
    (dict(temperature=1e-30), ["temperature"]),
    (dict(temperature=float("inf")), ["temperature"]),
    (dict(temperature=float("nan")), ["temperature"]),
    (dict(top_k=-1), ["top_k"]),
    (dict(top_p=1.5), ["top_p"]),
    (dict(top_p=float("nan")), ["top_p"]),
    (dict(min_p=-0.1), ["min_p"]),
    (dict(min_p=2.0), ["min_p"]),
    (dict(logits=None), ["logits", "NULL"]),
    (dict(stride=-10), ["logits", "negative"]),
    (dict(logits=PTR + 2), ["aligned"]),
])
def test_sample_refuses(kw, words):
    _refused("dz_sample_tokens", _sample_args(**kw), *words)


def test_no_rows_is_no_work():
    assert L.load().dz_sample_tokens(*_sample_args(rows=0, logits=None, uniform=None, tokens=None)) == 0


def test_python_wants_a_gpu():
    x = torch.zeros(1, 1, 1, 1, 64)
    with pytest.raises(DzError, match="GPU"):
        P.shared_prefix_attention(x, P.KV(x, x))
    cache = P.QuantizedKV.empty(1, 1, 4, 64)
    assert cache.k.dtype == torch.float8_e4m3fn and cache.k_scale.dtype == torch.float8_e8m0fnu and cache.k_scale.shape == (1, 1, 4)
    with pytest.raises(DzError, match="GPU"):
        P.cache_write(cache, x[0], x[0], 0)
    with pytest.raises(DzError, match="GPU"):
        P.cache_read(cache, 1, torch.float32)
    with pytest.raises(DzError, match="QuantizedKV"):
        P.cache_read(P.KV(x, x), 1, torch.float32)
    with pytest.raises(DzError, match="GPU"):
        S.sample_tokens(torch.zeros(1, 4), torch.zeros(1))
