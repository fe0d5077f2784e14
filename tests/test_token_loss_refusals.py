"""dizo_amd.token_loss without a GPU: what its entry points refuse, at the C ABI and in Python, and the
oracle's gradients against differences of its own values."""
import ctypes as C

import numpy as np
import pytest
import torch

from dizo_amd import _lib as L
from dizo_amd import token_loss as T
from dizo_amd._lib import DzError
from oracle import vocab as O

P = 4096  # a pointer that is not NULL; nothing reads through it


def _refused(name, args, *words):
    lib = L.load()
    rc = getattr(lib, name)(*args)
    msg = lib.dz_last_error().decode()
    assert rc < 0 and all(w in msg for w in words), (rc, msg)


def _score_args(**kw):
    a = dict(logits=P, dtype=L.DZ_DTYPE_F16, batch=2, length=3, vocab=10, lbs=30, lls=10, tokens=P, tbs=3, tls=1, ignore=-100,
             top=0, lp=P, ent=P, tlp=None, ttok=None, w=None, wbs=0, wls=0, u=None, ubs=0, uls=0, g=None, gbs=0, gls=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, words", [
    (dict(dtype=7), ["dtype"]),
    (dict(batch=-1), ["row count"]),
    (dict(batch=1 << 31, length=1 << 31), ["row count"]),
    (dict(batch=1 << 11, length=1 << 11), ["row count", "4194303"]),
    (dict(vocab=0), ["vocab"]),
    (dict(vocab=(1 << 30) + 1), ["vocab"]),
    (dict(top=-1), ["top"]),
    (dict(top=129, vocab=1000), ["top", "128"]),
    (dict(top=11), ["top"]),
    (dict(top=2, g=P), ["exclude"]),
    (dict(logits=None), ["logits", "NULL"]),
    (dict(lls=-10), ["logits", "negative"]),
    (dict(lbs=1 << 60), ["logits", "stride"]),
    (dict(logits=P + 1), ["aligned"]),
])
def test_token_logprobs_refuses(kw, words):
    _refused("dz_token_logprobs", _score_args(**kw), *words)


def test_no_rows_is_no_work():
    lib = L.load()
    assert lib.dz_token_logprobs(*_score_args(batch=0, logits=None, tokens=None, lp=None, ent=None)) == 0
    assert lib.dz_token_logprobs(*_score_args(length=0)) == 0


def _distill_args(**kw):
    a = dict(logits=P, dtype=L.DZ_DTYPE_F16, batch=2, length=3, vocab=10, lbs=30, lls=10, values=P, tokens=P, k=4, temperature=1.0,
             normalize=1, loss=P, w=None, wbs=0, wls=0, g=None, gbs=0, gls=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, words", [
    (dict(dtype=-1), ["dtype"]),
    (dict(k=0), ["entries"]),
    (dict(k=513), ["entries", "512"]),
    (dict(temperature=0.0), ["temperature"]),
    (dict(temperature=-1.0), ["temperature"]),
    (dict(temperature=float("inf")), ["temperature"]),
    (dict(temperature=float("nan")), ["temperature"]),
    (dict(temperature=1e-45), ["temperature"]),
    (dict(vocab=-3), ["vocab"]),
    (dict(logits=None), ["NULL"]),
])
def test_topk_distill_refuses(kw, words):
    _refused("dz_topk_distill", _distill_args(**kw), *words)


def _head_args(**kw):
    a = dict(hidden=P, weight=P, dtype=L.DZ_DTYPE_F16, rows=4, width=8, vocab=10, hs=8, ws=8, tokens=P, ignore=-100, lp=P, ent=P,
             work=P, bytes=1 << 20, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw, words", [
    (dict(dtype=3), ["dtype"]),
    (dict(rows=-1), ["row count"]),
    (dict(width=0), ["width"]),
    (dict(vocab=0), ["vocab"]),
    (dict(hidden=None), ["hidden", "NULL"]),
    (dict(hs=-8), ["negative"]),
])
def test_linear_token_logprobs_refuses(kw, words):
    _refused("dz_linear_token_logprobs", _head_args(**kw), *words)


def test_workspace_query():
    lib = L.load()
    n = C.c_int64(-1)
    assert lib.dz_linear_token_logprobs_workspace(L.DZ_DTYPE_F16, 0, 64, 100, C.byref(n)) == 0 and n.value == 0
    sizes = []
    for rows in (1, 100, 5000):
        assert lib.dz_linear_token_logprobs_workspace(L.DZ_DTYPE_F16, rows, 64, 50272, C.byref(n)) == 0
        sizes.append(n.value)
    assert 0 < sizes[0] < sizes[1] < sizes[2]
    _refused("dz_linear_token_logprobs_workspace", [L.DZ_DTYPE_F16, 1, 64, 100, None], "NULL")


def test_host_tensors_are_refused():
    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(DzError, match="GPU"):
        T.token_logprobs(x, t)
    with pytest.raises(DzError, match="GPU"):
        T.token_logprobs_grad(x, t, torch.ones(3))
    with pytest.raises(DzError, match="GPU"):
        T.topk_distill(x, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64))
    with pytest.raises(DzError, match="GPU"):
        T.topk_distill_grad(x, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64), torch.ones(3))
    with pytest.raises(DzError, match="GPU"):
        T.linear_token_logprobs(x, torch.zeros(9, 8), t)


def _difference(f, x, h=1e-5):
    d = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        d[i] = (f(a) - f(b)) / (2 * h)
    return d


def test_oracle_gradients_are_the_values_differences():
    r = np.random.default_rng(0)
    x = r.standard_normal((4, 9)) * 2
    tokens, w, u = np.array([3, -100, 0, 8]), r.standard_normal(4), r.standard_normal(4)

    def score(y):
        lp, ent, _, _ = O.token_logprobs(y, tokens)
        return (w * lp + u * ent).sum()

    # central differences: h^2 f''' / 6 + 2^-53 |f| / h, both below 1e-9 here
    np.testing.assert_allclose(O.token_logprobs_grad(x, tokens, w, u), _difference(score, x), atol=1e-8)
    values, at = r.standard_normal((4, 3)), np.array([[1, 5, 8], [-1, -1, -1], [2, 2, 0], [4, -1, 7]])
    for tau, norm in ((1.0, True), (2.5, True), (0.7, False)):
        got = O.topk_distill(x, values, at, tau, norm, w)[1]
        want = _difference(lambda y: (w * O.topk_distill(y, values, at, tau, norm)[0]).sum(), x)
        np.testing.assert_allclose(got, want, atol=1e-8)
