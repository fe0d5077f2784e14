"""dizo_amd.token_loss on the GPU against the definitions in 64 bits (oracle/vocab.py): types, layouts,
vocabularies from one token to one past 2^17, masked columns, rows without a distribution, ties,
gradients, streams, captured graphs and offsets past 32 bits.

Tolerances. Sums are fp32 with e = 2^-24 a rounding. A row's sum of 2^y is a sum of positive terms added in
at most v / 256 + 60 steps, each term off by at most a few e (1 + |y|); log probabilities are a difference
of that sum's logarithm and of y, each off by its size times a few e. Hence

  logprobs, alternatives   e (4 |lp| + 4 ln v + v / 256 + 60)
  entropy                  e (v / 256 + 60) (1 + ln v)
  distillation             T^2 e (v / 256 + 60 + k + 4 max |t| / T) (1 + sum w (|ln w| + |ln q|))
  gradients                half a step of their type, plus e (v / 256 + 100) times the sizes of their terms, and half
                           the type's smallest number
  head                     those of logprobs and entropy, plus twice the logits' own: products of width d, summed in
                           fp32: 16 e sqrt(d) |h * w|_2 (partial sums grow as a walk; a rounding of each step)
"""
import math

import numpy as np
import pytest
import torch

from dizo_amd import _lib as L
from dizo_amd import token_loss as T
from dizo_amd._lib import DzError
from dizo_amd.table import dtype_code, stream_handle
from oracle import vocab as O

pytestmark = pytest.mark.gpu

E = 2.0**-24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SMALLEST = {torch.float32: 2.0**-126, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126}
IDS = ["f32", "f16", "bf16"]


def f64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, tol, what=""):
    """|got - want| <= tol where want is finite; NaN and infinities have to be the same."""
    got, want, tol = np.broadcast_arrays(np.asarray(got, dtype=np.float64), want, tol)
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what + " (NaN)")
    odd = ~fine & ~np.isnan(want)
    np.testing.assert_array_equal(got[odd], want[odd], err_msg=what + " (infinite)")
    off = np.abs(got[fine] - want[fine]) - tol[fine]
    if off.size and not off.max() <= 0:
        i = int(np.argmax(off))
        raise AssertionError(f"{what}: off by {np.abs(got[fine] - want[fine])[i]:.3g} at {want[fine][i]:.6g}, allowed {tol[fine][i]:.3g}")


def same(a, b):
    """Equal bits, any NaN like another."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def lp_tol(lp, v):
    return E * (4 * np.nan_to_num(np.abs(lp), posinf=0, neginf=0) + 4 * math.log(v) + v / 256 + 60)


def ent_tol(v):
    return E * (v / 256 + 60) * (1 + math.log(v))


def check_score(logits, tokens, top=0, ignore=-100, out=None):
    """token_logprobs of (..., v) logits against the oracle."""
    if out is None:
        out = T.token_logprobs(logits, tokens, top=top, ignore_index=ignore)
    v = logits.shape[-1]
    x, t = f64(logits).reshape(-1, v), tokens.cpu().numpy().reshape(-1)
    lp, ent, tlp, ttok = O.token_logprobs(x, t, top, ignore)
    assert out.logprobs.shape == tokens.shape and out.logprobs.dtype == torch.float32
    close(f64(out.logprobs).reshape(-1), lp, lp_tol(lp, v), "logprobs")
    close(f64(out.entropy).reshape(-1), ent, ent_tol(v), "entropy")
    if top:
        assert out.top_tokens.dtype == torch.int64 and out.top_tokens.shape == (*tokens.shape, top)
        np.testing.assert_array_equal(out.top_tokens.cpu().numpy().reshape(-1, top), ttok)
        close(f64(out.top_logprobs).reshape(-1, top), tlp, lp_tol(tlp, v), "top_logprobs")
    else:
        assert out.top_logprobs is None and out.top_tokens is None
    return out


def score_grad_tol(x, t, w, u, dtype, ignore=-100):
    """(the oracle's gradient, how far it may be off)"""
    n, v = x.shape
    want = O.token_logprobs_grad(x, t, w, u, ignore)
    logq = np.nan_to_num(O.log_softmax(x), nan=0.0, neginf=0.0)
    q = np.exp(O.log_softmax(x))
    q = np.nan_to_num(q)
    h = math.log(v)
    terms = q * (np.abs(w)[:, None] + np.abs(u)[:, None] * (np.abs(logq) + h)) * (v / 256 + 100 + 4 * np.abs(logq))
    own = np.zeros((n, v))
    for r in range(n):
        if 0 <= t[r] < v:
            own[r, t[r]] = 4 * abs(w[r])
    return want, torch.finfo(dtype).eps / 2 * np.abs(np.nan_to_num(want)) + E * (terms + own) + SMALLEST[dtype]


def distill_tol(x, values, at, tau, norm, w, dtype):
    n, v = x.shape
    k = at.shape[1]
    loss, grad = O.topk_distill(x, values, at, tau, norm, w)
    logq = O.log_softmax(x / tau)
    q = np.nan_to_num(np.exp(logq))
    ltol, gtol = np.zeros(n), np.zeros((n, v))
    for r in range(n):
        tw, tl = O.teacher_weights(values[r], at[r], v, tau, norm)
        there = (at[r] >= 0) & (at[r] < v) & (np.nan_to_num(tw) > 0)
        tw, tl, ids = tw[there], tl[there], at[r][there]
        steps = v / 256 + 60 + k + 4 * np.abs(np.nan_to_num(values[r][there])).max(initial=0) / tau
        size = (tw * (np.abs(tl) + np.abs(np.nan_to_num(logq[r][ids], neginf=0)))).sum()
        ltol[r] = tau * tau * E * steps * (1 + size)
        gtol[r] = q[r] * max(1.0, tw.sum()) * (steps + 100 + 4 * np.abs(np.nan_to_num(logq[r], neginf=0)))
        np.add.at(gtol[r], ids, tw * (steps + 100))
    gtol *= E * tau * np.abs(w)[:, None]
    return loss, ltol, grad, gtol + torch.finfo(dtype).eps / 2 * np.abs(np.nan_to_num(grad)) + SMALLEST[dtype]


def check_distill(logits, values, at, tau=1.0, norm=True, weights=None):
    v, k = logits.shape[-1], at.shape[-1]
    lead = logits.shape[:-1]
    if weights is None:
        weights = torch.linspace(-1.0, 1.5, max(1, math.prod(lead)), device="cuda")[:math.prod(lead)].reshape(lead)
    loss, ltol, grad, gtol = distill_tol(f64(logits).reshape(-1, v), f64(values).reshape(-1, k), at.cpu().numpy().reshape(-1, k), tau, norm,
                                         f64(weights).reshape(-1), logits.dtype)
    got = T.topk_distill(logits, values, at, temperature=tau, normalize=norm)
    assert got.shape == lead and got.dtype == torch.float32
    close(f64(got).reshape(-1), loss, ltol, "loss")
    got2, g = T.topk_distill_grad(logits, values, at, weights, temperature=tau, normalize=norm)
    close(f64(got2).reshape(-1), loss, ltol, "loss of the call with a gradient")
    assert g.dtype == logits.dtype and g.shape == logits.shape
    close(f64(g).reshape(-1, v), grad, gtol, "gradient")


def rows(n, v, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, v, generator=g) * spread).to(dtype).cuda()


def some_tokens(n, v, seed, ignored=True):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, v, (n,), generator=g)
    if ignored and n > 1:
        t[torch.rand(n, generator=g) < 0.25] = -100
    return t.cuda()


VOCABS = [1, 2, 7, 63, 255, 256, 257, 1000, 4099, 8192, 32771, 50272, 65541, 131072 + 13, 270001]


# ---------------------------------------------------------- token_logprobs --
@pytest.mark.parametrize("v", VOCABS)
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_token_logprobs(dtype, v):
    n = 13 if v < 5000 else 5
    x, t = rows(n, v, dtype, v), some_tokens(n, v, v + 1)
    check_score(x, t)
    check_score(x, t, top=min(v, 20))
    check_score(x, t, top=min(v, 128))


@pytest.mark.parametrize("v", VOCABS)
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_token_logprobs_grad(dtype, v):
    n = 9 if v < 5000 else 4
    x, t = rows(n, v, dtype, v + 2), some_tokens(n, v, v + 3)
    w, u = torch.linspace(-1, 1.3, n).cuda(), torch.linspace(0.5, -0.4, n).cuda()
    for a, b in ((w, u), (w, None), (None, u)):
        out, g = T.token_logprobs_grad(x, t, a, b)
        check_score(x, t, out=out)
        zero = np.zeros(n)
        want, tol = score_grad_tol(f64(x), t.cpu().numpy(), zero if a is None else f64(a), zero if b is None else f64(b), dtype)
        close(f64(g), want, tol, "gradient")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_token_logprobs_layouts(dtype):
    """Views are read in place: shifted, strided and offset rows, one row, no row, three leading dimensions."""
    for v in (250, 257, 4099):
        full = rows(4 * 6, v, dtype, 5).view(4, 6, v)
        t = some_tokens(24, v, 6).view(4, 6)
        w = torch.rand(4, 6, generator=torch.Generator().manual_seed(1)).cuda()
        wide = rows(7, 3 * v + 5, dtype, 8)
        views = [(full[:, :-1], t[:, 1:], w[:, 1:]), (full[:, 1:4], t[:, :3], w[:, :3]), (full.transpose(0, 1), t.t(), w.t()),
                 (full[::2, ::3], t[::2, ::3], w[::2, ::3]), (wide[:, 3:3 + v], t.view(-1)[:7], w.view(-1)[:7]),
                 (wide[2, 1:1 + v], t[0, 0], w[0, 0]), (full[:0], t[:0], w[:0]), (full[:, :0], t[:, :0], w[:, :0]),
                 (full.view(2, 2, 6, v), t.view(2, 2, 6), w.view(2, 2, 6)), (full.view(2, 2, 6, v)[:, :, 1:], t.view(2, 2, 6)[:, :, 1:], w.view(2, 2, 6)[:, :, 1:]),
                 (full[1:2].expand(3, 6, v), t[:3], w[:1].expand(3, 6))]
        for x, tok, wt in views:
            check_score(x, tok, top=5)
            out, g = T.token_logprobs_grad(x, tok, wt, wt)
            assert g.shape == x.shape
            want, tol = score_grad_tol(f64(x).reshape(-1, v), tok.cpu().numpy().reshape(-1), f64(wt).reshape(-1), f64(wt).reshape(-1), dtype)
            close(f64(g).reshape(-1, v), want, tol, "gradient")


def test_token_types_and_ignore_index():
    x, t = rows(6, 100, torch.float16, 1), some_tokens(6, 100, 2, ignored=False)
    check_score(x, t.int(), top=3)
    t[2] = 0
    out = check_score(x, t, top=3, ignore=0)
    assert out.logprobs[2] == 0 and out.top_tokens[2].tolist() == [-1] * 3
    t[4] = -100  # not the ignore index here: a token outside the vocabulary
    out = check_score(x, t, ignore=0)
    assert out.logprobs[4].isnan() and not out.entropy[4].isnan()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("v", [9, 1000, 50272])
def test_masked_columns_and_rows(dtype, v):
    """-inf, the type's lowest value, NaN and +inf: what takes no part, what takes a uniform part, and what makes a row NaN."""
    low = torch.finfo(dtype).min
    x = rows(12, v, dtype, 3)
    x[0, v // 2:] = -math.inf
    x[1, : v // 2] = low
    x[2] = low  # a uniform distribution
    x[3] = -math.inf  # none
    x[4, v // 3] = math.nan
    x[5, v - 1] = math.inf
    x[6] = -math.inf
    x[6, v // 2] = 1.5  # one token alone: log probability 0, entropy 0
    x[7] = 0.25  # ties everywhere
    x[8] = torch.finfo(dtype).max  # a uniform distribution again
    x[9, ::2] = math.nan
    x[10] = low
    x[10, v // 4] = -math.inf
    x[11, v // 2] = torch.finfo(dtype).max
    t = torch.tensor([0, v - 1, 1, 1, 0, 0, v // 2, 2, 3, -100, 0, v // 2]).cuda()
    for top in (0, 5):
        check_score(x, t, top=top)
    out = check_score(x, torch.where(t >= 0, torch.full_like(t, v - 1), t))  # a masked token's: -inf
    assert out.logprobs[0] == -math.inf
    w = torch.linspace(0.5, 1.5, 12).cuda()
    _, g = T.token_logprobs_grad(x, t, w, w)
    want, tol = score_grad_tol(f64(x), t.cpu().numpy(), f64(w), f64(w), dtype)
    close(f64(g), want, tol, "gradient")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_alternatives_with_ties_and_adverse_orders(dtype):
    """Equal logits by their token; large logits side by side, in runs, and in ascending and descending order; -0 and +0."""
    v = 20011
    g = torch.Generator().manual_seed(9)
    few = torch.randint(-3, 4, (v,), generator=g).float()
    up = torch.arange(v).float() / 512
    run = torch.full((v,), -5.0)
    run[7000:7000 + 4096] = 3.0
    comb = torch.full((v,), -2.0)
    comb[::2048] = 1.0
    blocks = -torch.rand(v, generator=g)
    for s in range(0, v - 40, 1024):  # many large ones in few lanes
        blocks[s:s + 32] = 4 + torch.rand(32, generator=g)
    zeros = torch.zeros(v)
    zeros[::3] = -0.0
    only = torch.full((v,), -math.inf)
    only[[5, 17, 19999]] = torch.tensor([1.0, 1.0, 2.0])
    x = torch.stack([few, up, -up, run, comb, blocks, zeros, only, torch.full((v,), 7.0), up.flip(0)]).to(dtype).cuda()
    t = torch.zeros(x.shape[0], dtype=torch.int64).cuda()
    for top in (1, 2, 17, 64, 128):
        check_score(x, t, top=top)
    y = x[:, :130].contiguous()
    for top in (127, 128):
        check_score(y, t, top=top)
    z = x[:, :60].contiguous()
    check_score(z, t, top=60)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_token_logprobs_autograd(dtype):
    v = 1003
    x = rows(10, v, dtype, 4).view(2, 5, v)
    t = some_tokens(10, v, 5).view(2, 5)
    a, b = torch.linspace(-1, 1, 10).cuda().view(2, 5), torch.linspace(0.2, -0.3, 10).cuda().view(2, 5)
    leaf = x.clone().requires_grad_(True)
    out = T.token_logprobs(leaf[:, 1:], t[:, 1:], top=3)
    assert out.logprobs.requires_grad and out.entropy.requires_grad and not out.top_logprobs.requires_grad
    (a[:, 1:] * out.logprobs + b[:, 1:] * out.entropy).sum().backward()
    _, want = T.token_logprobs_grad(x[:, 1:], t[:, 1:], a[:, 1:], b[:, 1:])
    assert torch.equal(leaf.grad[:, 1:], want) and not leaf.grad[:, 0].any()
    # one output alone, through an expanded upstream gradient
    leaf = x.clone().requires_grad_(True)
    T.token_logprobs(leaf, t).logprobs.sum().backward()
    _, want = T.token_logprobs_grad(x, t, torch.ones(2, 5, device="cuda"))
    assert torch.equal(leaf.grad, want)
    with torch.no_grad():
        assert not T.token_logprobs(leaf, t).logprobs.requires_grad


def test_gradients_are_the_values_differences():
    """Central differences of the kernel's own fp32 values with h = 2^-6: h^2 |f'''| / 6 <= 4e-5 |weights|, and the
    values' error over h: 2^6 * 2 * 80 e < 7e-4 (v small: about 80 roundings)."""
    v = 11
    x, t = rows(4, v, torch.float32, 1, 1.0), torch.tensor([0, 5, -100, 10]).cuda()
    w, u = torch.tensor([1.0, -0.5, 1.0, 0.7]).cuda(), torch.tensor([0.0, 0.8, 1.0, -0.6]).cuda()
    val, at = rows(4, 3, torch.float32, 2, 1.0), torch.tensor([[1, 2, 3], [0, 0, 9], [-1, -1, -1], [10, -1, 4]]).cuda()

    def score(y):
        o = T.token_logprobs(y, t)
        return w * o.logprobs + u * o.entropy

    for f, g in ((score, T.token_logprobs_grad(x, t, w, u)[1]),
                 (lambda y: w * T.topk_distill(y, val, at, temperature=1.5), T.topk_distill_grad(x, val, at, w, temperature=1.5)[1])):
        h = 2.0**-6
        for i in range(v):
            d = torch.zeros(v, device="cuda")
            d[i] = h
            np.testing.assert_allclose(f64(g[:, i]), f64(f(x + d) - f(x - d)) / (2 * h), atol=1e-3)


# ------------------------------------------------------------ topk_distill --
def teacher(x, k, seed, ragged=True):
    g = torch.Generator().manual_seed(seed)
    t = x.detach().float().cpu().reshape(-1, x.shape[-1]) + torch.randn(x.reshape(-1, x.shape[-1]).shape, generator=g)
    val, at = t.topk(k, -1)
    if ragged and at.shape[0] > 2:
        at[1] = -1
        at[2, k // 2:] = -1
        val[1], val[2, k // 2:] = math.nan, -math.inf  # what stands where there is no entry does not count
        if k < 2:
            at[2] = 0
    lead = x.shape[:-1]
    return val.view(*lead, k).cuda(), at.view(*lead, k).cuda()


@pytest.mark.parametrize("v", VOCABS)
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_topk_distill(dtype, v):
    n = 7 if v < 5000 else 4
    x = rows(n, v, dtype, v + 4)
    for k, tau, norm in ((1, 1.0, True), (min(v, 20), 2.0, True), (min(v, 64), 0.6, True), (min(v, 5), 1.3, False), (min(v, 512), 1.0, True)):
        val, at = teacher(x, k, v + k)
        if not norm:
            val = val - val.logsumexp(-1, keepdim=True) - 0.2
        check_distill(x, val, at, tau, norm)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_topk_distill_layouts(dtype):
    for v in (250, 257):
        full = rows(24, v, dtype, 5).view(4, 6, v)
        val, at = teacher(full, 6, 7)
        w = torch.rand(4, 6, generator=torch.Generator().manual_seed(1)).cuda()
        for s in ((slice(None), slice(0, -1)), (slice(0, None, 2), slice(1, 6, 3)), (slice(1, 2), slice(None)), (slice(0, 0), slice(None)), (0, 3)):
            check_distill(full[s], val[s], at[s], 1.5, True, w[s])
        check_distill(full.transpose(0, 1), val.transpose(0, 1), at.transpose(0, 1), 1.0, True, w.t())
        check_distill(full.view(2, 2, 6, v), val.view(2, 2, 6, 6).to(torch.bfloat16), at.view(2, 2, 6, 6).int(), 1.0, True, w.view(2, 2, 6))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_topk_distill_edges(dtype):
    """Duplicates, weights of zero, tokens outside the vocabulary, masked student logits, rows without a distribution."""
    v = 600
    x = rows(14, v, dtype, 3)
    val, at = teacher(x, 5, 4, ragged=False)
    at[0] = at[0, 0]  # one token five times
    at[1, 3] = at[1, 1]
    val[2, 1:] = -math.inf
    at[3, 2] = v  # outside
    at[4, 0] = -7
    val[5, 1] = math.nan
    val[6, 1] = math.inf
    val[7] = -math.inf  # entries, but no weight
    x[8, at[8, 0]] = -math.inf  # the teacher's best is impossible for the student: an infinite loss
    x[9, at[9, 4]] = -math.inf
    val[9, 4] = -math.inf  # impossible for both: adds nothing
    x[10] = -math.inf
    x[11, 5] = math.nan
    x[12] = torch.finfo(dtype).min
    at[13] = -1
    x[13] = math.nan  # not read
    check_distill(x, val, at, 1.0)
    check_distill(x, val, at, 3.0)
    check_distill(x, val - 40.0, at, 1.0, norm=False)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_topk_distill_autograd(dtype):
    v = 1003
    x = rows(10, v, dtype, 4).view(2, 5, v)
    val, at = teacher(x, 8, 5)
    w = torch.linspace(-1, 1, 10).cuda().view(2, 5)
    leaf = x.clone().requires_grad_(True)
    (w * T.topk_distill(leaf, val, at, temperature=2.0)).sum().backward()
    assert torch.equal(leaf.grad, T.topk_distill_grad(x, val, at, w, temperature=2.0)[1])
    leaf = x.clone().requires_grad_(True)
    T.topk_distill(leaf, val, at).mean().backward()
    assert torch.equal(leaf.grad, T.topk_distill_grad(x, val, at, torch.full((2, 5), 0.1, device="cuda"))[1])


def test_recorded_alternatives_are_a_teacher():
    """A model distilled from its own recorded alternatives, all of them: the distance is 0, and so is the gradient."""
    v = 100
    x = rows(6, v, torch.bfloat16, 1)
    rec = T.token_logprobs(x, torch.zeros(6, dtype=torch.int64, device="cuda"), top=v)
    loss, g = T.topk_distill_grad(x, rec.top_logprobs, rec.top_tokens, torch.ones(6, device="cuda"))
    close(f64(loss), np.zeros(6), np.full(6, E * 300 * 10))
    close(f64(g), np.zeros((6, v)), np.full((6, v), E * 300))


# --------------------------------------------------- linear_token_logprobs --
def check_head(h, w, t, ignore=-100, out=None):
    d, v = h.shape[-1], w.shape[0]
    if out is None:
        out = T.linear_token_logprobs(h, w, t, ignore_index=ignore)
    hh, ww, tt = f64(h).reshape(-1, d), f64(w), t.cpu().numpy().reshape(-1)
    dead = tt == ignore
    x = np.where(dead[:, None], 0.0, np.where(dead[:, None], 0.0, hh) @ ww.T)
    lp, ent, _, _ = O.token_logprobs(x, tt, 0, ignore)
    off = 2 * 16 * E * math.sqrt(d) * np.sqrt((np.nan_to_num(hh, nan=0, posinf=0, neginf=0)**2) @ (ww**2).T).max(-1)
    assert out.logprobs.shape == t.shape and out.top_tokens is None
    close(f64(out.logprobs).reshape(-1), lp, lp_tol(lp, v) + off, "logprobs")
    close(f64(out.entropy).reshape(-1), ent, ent_tol(v) + off * (1 + math.log(v)), "entropy")
    return out


def head(n, d, v, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, d, generator=g).to(dtype).cuda(), (torch.randn(v, d, generator=g) * 2.5 / math.sqrt(d)).to(dtype).cuda()


@pytest.mark.parametrize("n, d, v", [(1, 1, 1), (1, 64, 50), (2, 8, 64), (5, 40, 65), (16, 100, 1000), (17, 257, 129), (64, 64, 4099), (65, 1024, 130),
                                     (130, 72, 513), (200, 768, 1003), (257, 520, 2048), (1, 5120, 999), (33, 33, 33), (1100, 65, 70), (300, 136, 700)])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_token_logprobs(dtype, n, d, v):
    h, w = head(n, d, v, dtype, n + d + v)
    check_head(h, w, some_tokens(n, v, 3))
    check_head(h, w, some_tokens(n, v, 4, ignored=False).int())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_token_logprobs_layouts(dtype):
    h, w = head(24, 200, 300, dtype, 1)
    t = some_tokens(24, 300, 2)
    wide = torch.zeros(300, 211, dtype=dtype, device="cuda")
    wide[:, 5:205] = w
    for hh, tt in ((h.view(4, 6, 200)[:, 1:], t.view(4, 6)[:, 1:]), (h.view(2, 2, 6, 200), t.view(2, 2, 6)), (h[3], t[3]), (h[:0], t[:0]),
                   (h[::5], t[::5]), (h.t().contiguous().t(), t)):
        check_head(hh, w, tt)
        check_head(hh, wide[:, 5:205], tt)
        check_head(hh, w[::3], tt.clamp(max=99))
    few = torch.full((24,), -100, device="cuda")
    check_head(h, w, few)  # nothing asked for
    few[23] = 7
    check_head(h, w, few)
    few[11] = 300  # outside the vocabulary
    out = check_head(h, w, few)
    assert out.logprobs[11].isnan() and not out.entropy[11].isnan()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_bad_hidden_states_stay_in_their_rows(dtype):
    h, w = head(40, 96, 200, dtype, 6)
    t = some_tokens(40, 200, 2, ignored=False)
    clean = T.linear_token_logprobs(h, w, t)
    h[3, 5] = math.nan
    h[20] = math.inf
    h[21] = math.nan
    t2 = t.clone()
    t2[21] = -100  # ignored: not computed
    out = T.linear_token_logprobs(h, w, t2)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[3, 20, 21]] = False
    assert torch.equal(out.logprobs[keep], clean.logprobs[keep]) and torch.equal(out.entropy[keep], clean.entropy[keep])
    assert out.logprobs[[3, 20]].isnan().all() and out.logprobs[21] == 0 and out.entropy[21] == 0


def test_linear_token_logprobs_where_autograd_records():
    h, w = head(10, 64, 100, torch.float32, 6)
    t = some_tokens(10, 100, 2)
    want = T.linear_token_logprobs(h, w, t).logprobs
    h.requires_grad_(True)
    got = T.linear_token_logprobs(h, w, t)
    assert got.logprobs.requires_grad
    np.testing.assert_allclose(f64(got.logprobs), f64(want), atol=1e-4)
    got.logprobs.sum().backward()
    x = (h.detach() @ w.t()).requires_grad_(True)
    T.token_logprobs(x, t).logprobs.sum().backward()
    np.testing.assert_allclose(f64(h.grad), f64(x.grad @ w), atol=1e-4)


# ---------------------------------------------------------------- in common --
def test_results_do_not_change_from_call_to_call():
    """The same bits every time (no atomics in a sum), whatever was computed before."""
    x, t = rows(40, 50272, torch.float16, 1), some_tokens(40, 50272, 2)
    h, w = head(100, 256, 5000, torch.bfloat16, 3)
    th = some_tokens(100, 5000, 4)
    val, at = teacher(x, 16, 5)
    ones = torch.ones(40, device="cuda")

    def everything():
        return [*T.token_logprobs(x, t, top=33), *T.token_logprobs_grad(x, t, ones, ones)[0][:2], T.token_logprobs_grad(x, t, ones, ones)[1],
                *T.topk_distill_grad(x, val, at, ones), *T.linear_token_logprobs(h, w, th)[:2]]

    first = everything()
    T.token_logprobs(rows(300, 1000, torch.float32, 6), some_tokens(300, 1000, 7), top=5)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, everything()))


def test_other_streams():
    x, t = rows(64, 4099, torch.float16, 1), some_tokens(64, 4099, 2)
    h, w = head(64, 256, 5000, torch.float16, 3)
    want = T.token_logprobs(x, t, top=4), T.linear_token_logprobs(h, w, t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = T.token_logprobs(x, t, top=4), T.linear_token_logprobs(h, w, t)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for p, q in zip(want, got) for a, b in zip(p, q) if a is not None)


def test_captured_calls_replay():
    """Every call in one captured graph; each replay sees what its inputs hold by then."""
    x, t = rows(12, 4099, torch.bfloat16, 1), some_tokens(12, 4099, 2)
    h, w = head(12, 96, 4099, torch.bfloat16, 3)
    val, at = teacher(x, 9, 4)
    wt = torch.linspace(0.5, 1, 12).cuda()

    def calls():
        return [*T.token_logprobs(x, t, top=7), *T.token_logprobs_grad(x, t, wt, wt)[0][:2], T.token_logprobs_grad(x, t, wt, wt)[1],
                T.topk_distill(x, val, at), *T.topk_distill_grad(x, val, at, wt), *T.linear_token_logprobs(h, w, t)[:2]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for i in range(4):
        x.copy_(rows(12, 4099, torch.bfloat16, 10 + i))
        h.copy_(head(12, 96, 1, torch.bfloat16, 20 + i)[0])
        t.copy_(some_tokens(12, 4099, 30 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, calls())), i


def test_rows_past_two_to_the_32nd_element():
    """Offsets in 64 bits: the second sequence starts past 2^32 elements."""
    v, far = 1001, 2**32 + 24
    buf = torch.empty(far + 2 * v, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((2, 2, v), (far, v, 1))
    x.copy_(rows(4, v, torch.bfloat16, 1).view(2, 2, v))
    t = some_tokens(4, v, 2, ignored=False).view(2, 2)
    check_score(x, t, top=9)
    val, at = teacher(x, 4, 3, ragged=False)
    check_distill(x, val, at)
    del buf, x
    wide = torch.empty(3 * 2**30 + 64, dtype=torch.bfloat16, device="cuda")  # head rows 2^29 elements apart
    w = wide.as_strided((6, 64), (2**29 + 8, 1))
    h, w0 = head(5, 64, 6, torch.bfloat16, 4)
    w.copy_(w0)
    check_head(h, w, torch.tensor([0, 5, 3, -100, 2]).cuda())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("v", [1, 9, 250, 257, 1001])
def test_nothing_is_written_outside_the_gradient(dtype, v):
    """Through the C ABI: gradient rows at strides and offsets other than the logits', with marks all around."""
    x, t = rows(6, v, dtype, 1), some_tokens(6, v, 2)
    w = torch.linspace(0.5, 1, 6).cuda()
    val, at = teacher(x, 1, 3)
    lp, ent, loss = (torch.empty(6, device="cuda") for _ in range(3))
    _, want = T.token_logprobs_grad(x, t, w)
    _, want2 = T.topk_distill_grad(x, val, at, w)
    for offset, stride in ((0, v + 3), (5, v), (3, v + 8), (8, v + 8)):
        buf = torch.full((offset + 6 * stride + 16,), 7.0, dtype=dtype, device="cuda")
        g = buf.as_strided((6, v), (stride, 1), offset)
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask.as_strided((6, v), (stride, 1), offset).fill_(False)
        L.call("dz_token_logprobs", x.data_ptr(), dtype_code(dtype), 1, 6, v, 0, v, t.data_ptr(), 0, 1, -100, 0, lp.data_ptr(), ent.data_ptr(),
               None, None, w.data_ptr(), 0, 1, None, 0, 0, g.data_ptr(), 0, stride, stream_handle())
        assert same(g, want) and (buf[mask] == 7.0).all()
        buf.fill_(7.0)
        L.call("dz_topk_distill", x.data_ptr(), dtype_code(dtype), 1, 6, v, 0, v, val.data_ptr(), at.data_ptr(), 1, 1.0, 1, loss.data_ptr(),
               w.data_ptr(), 0, 1, g.data_ptr(), 0, stride, stream_handle())
        assert same(g, want2) and (buf[mask] == 7.0).all()


def test_refusals():
    x, t = rows(4, 16, torch.float16, 1), torch.zeros(4, dtype=torch.int64, device="cuda")
    val, at = torch.zeros(4, 2, device="cuda"), torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    w = torch.ones(4, device="cuda")
    for call, word in (
        (lambda: T.token_logprobs(x.double(), t), "dtype"),
        (lambda: T.token_logprobs(x.t(), torch.zeros(16, dtype=torch.int64, device="cuda")), "contiguous"),
        (lambda: T.token_logprobs(x, t[:3]), "shape"),
        (lambda: T.token_logprobs(x, t.float()), "int64"),
        (lambda: T.token_logprobs(x, t.cpu()), "must be on"),
        (lambda: T.token_logprobs(x, t, top=17), "top"),
        (lambda: T.token_logprobs(x, t, top=-1), "top"),
        (lambda: T.token_logprobs_grad(x, t), "weights"),
        (lambda: T.token_logprobs_grad(x, t, w.half()), "float32"),
        (lambda: T.token_logprobs_grad(x, t, w[:2]), "shape"),
        (lambda: T.topk_distill(x, val, at, temperature=0.0), "temperature"),
        (lambda: T.topk_distill(x, val[:, :0], at[:, :0]), "entries"),
        (lambda: T.topk_distill(x, val, at[:, :1]), "shape"),
        (lambda: T.topk_distill(x, val.requires_grad_(True), at), "gradient"),
        (lambda: T.topk_distill_grad(x, val.detach(), at, w.cpu()), "must be on"),
        (lambda: T.linear_token_logprobs(x, x.float(), t), "weight is"),
        (lambda: T.linear_token_logprobs(x, x[:, :8], t), "fit"),
        (lambda: T.linear_token_logprobs(x, x.t()[:, :4].contiguous().t(), t), "fit|contiguous"),
    ):
        with pytest.raises(DzError, match=word):
            call()
    # at the C ABI: a range that leaves its allocation, rows that overlap, a workspace that is too small
    n = x.numel()
    ok = [x.data_ptr(), L.DZ_DTYPE_F16, 1, 4, 16, 0, 16, t.data_ptr(), 0, 1, -100, 0, w.data_ptr(), w.data_ptr(), None, None, w.data_ptr(), 0, 1,
          None, 0, 0, x.data_ptr(), 0, 16, stream_handle()]
    far, overlap = list(ok), list(ok)
    far[6] = 1 << 40
    with pytest.raises(DzError, match="logits range exceeds"):
        L.call("dz_token_logprobs", *far)
    overlap[24] = 8
    with pytest.raises(DzError, match="overlap"):
        L.call("dz_token_logprobs", *overlap)
    with pytest.raises(DzError, match="are needed"):
        L.call("dz_linear_token_logprobs", x.data_ptr(), x.data_ptr(), L.DZ_DTYPE_F16, 4, 16, 4, 16, 16, t.data_ptr(), -100, w.data_ptr(), w.data_ptr(),
               x.data_ptr(), n, stream_handle())


# ------------------------------------------------- lengths of every variant --
HELD = [8 * 2048, 8 * 2048 + 8, 8 * 4096 + 3, 8 * 512 * 13, 8 * 512 * 13 + 9, 8 * 8192 + 1, 8 * 1024 * 13 + 5, 8 * 16384, 8 * 16384 + 7, 8 * 32768 + 4099]


@pytest.mark.parametrize("v", HELD)
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_rows_at_the_borders_of_what_a_workgroup_holds(dtype, v):
    """Lengths at and past the sizes between which the kernels change, in 16-bit types and in fp32; more rows than one
    workgroup a compute unit, and fewer."""
    if dtype == torch.float32:
        v = v // 2 + v % 2
    x, t = rows(3, v, dtype, v), torch.tensor([v - 1, -100, v // 2]).cuda()
    x[2, : v // 3] = -math.inf
    check_score(x, t, top=50)
    check_score(x, t)
    w, u = torch.tensor([0.7, 1.0, -1.2]).cuda(), torch.tensor([0.1, 1.0, 0.3]).cuda()
    _, g = T.token_logprobs_grad(x, t, w, u)
    want, tol = score_grad_tol(f64(x), t.cpu().numpy(), f64(w), f64(u), dtype)
    close(f64(g), want, tol, "gradient")
    val, at = teacher(x.clamp(min=-30), 7, v, ragged=False)
    check_distill(x.clamp(min=-30), val, at, 1.5)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("n", [255, 256, 257, 700])
def test_many_and_few_rows_agree(dtype, n):
    """The rule on the number of rows changes the kernel, not the results beyond rounding: rows of 9,000 tokens, twice over."""
    x, t = rows(n, 9001, dtype, 3), some_tokens(n, 9001, 4)
    check_score(x, t)
    few, many = T.token_logprobs(x[:5], t[:5]), T.token_logprobs(x, t)
    tol = lp_tol(f64(few.logprobs), 9001)
    close(f64(many.logprobs[:5]), f64(few.logprobs), 2 * tol)


def test_a_rising_maximum_moves_the_statistics():
    """Logits that rise along the row by far more than the 8 binary orders that the running maximum may lag behind."""
    v = 40000
    ramp = torch.arange(v).float()
    x = torch.stack([ramp / 64, ramp / 4096, -ramp / 64, torch.where(ramp < v - 3, -500.0, ramp - v), ramp.remainder(4096) / 8 - 100]).cuda()
    t = torch.tensor([v - 1, v - 2, 0, v - 2, 4095]).cuda()
    for dtype in TYPES:
        check_score(x.to(dtype), t)
        check_score(x.to(dtype), t, top=64)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_a_gradient_may_be_written_over_its_logits(dtype):
    for v in (7, 1001, 40000, 150001):
        x, t = rows(4, v, dtype, v), some_tokens(4, v, 1)
        val, at = teacher(x, 3, 2, ragged=False)
        w = torch.linspace(0.5, 1.5, 4).cuda()
        _, want = T.token_logprobs_grad(x, t, w, w)
        _, want2 = T.topk_distill_grad(x, val, at, w)
        out, y = torch.empty(8, device="cuda"), x.clone()
        L.call("dz_token_logprobs", y.data_ptr(), dtype_code(dtype), 1, 4, v, 0, v, t.data_ptr(), 0, 1, -100, 0, out.data_ptr(), out[4:].data_ptr(),
               None, None, w.data_ptr(), 0, 1, w.data_ptr(), 0, 1, y.data_ptr(), 0, v, stream_handle())
        assert torch.equal(y, want)
        y = x.clone()
        L.call("dz_topk_distill", y.data_ptr(), dtype_code(dtype), 1, 4, v, 0, v, val.data_ptr(), at.data_ptr(), 3, 1.0, 1, out.data_ptr(),
               w.data_ptr(), 0, 1, y.data_ptr(), 0, v, stream_handle())
        assert torch.equal(y, want2)
        big = torch.empty(5 * v, dtype=dtype, device="cuda")
        with pytest.raises(DzError, match="overlap"):
            L.call("dz_topk_distill", big.data_ptr(), dtype_code(dtype), 1, 4, v, 0, v, val.data_ptr(), at.data_ptr(), 3, 1.0, 1, out.data_ptr(),
                   w.data_ptr(), 0, 1, big[v:].data_ptr(), 0, v, stream_handle())


@pytest.mark.parametrize("n, d, v", [(1, 64, 33000), (31, 72, 32800), (33, 136, 33001), (64, 64, 33000), (65, 64, 33000), (128, 200, 32800), (129, 64, 33000),
                                     (300, 136, 17000), (520, 8, 12000), (257, 1000, 16500)])
@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_token_logprobs_in_large_tiles(dtype, odd, n, d, v):
    """Enough tiles for every compute unit, and more than one for some; widths that do and do not fill 16 bytes."""
    h, w = head(n, d + odd, v, dtype, n + d + v)
    t = some_tokens(n, v, 3)
    t[-1] = v - 1
    check_head(h, w, t)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_bad_head_rows_count_where_they_are(dtype):
    """A head row of NaN makes every row a NaN; one that gives -inf takes no part; +inf makes a NaN."""
    for n, d, v in ((20, 96, 200), (90, 64, 33000)):
        h, w = head(n, d, v, dtype, 6)
        h = h.abs() + 0.5
        t = some_tokens(n, v, 2)
        w[7] = -math.inf
        out = T.linear_token_logprobs(h, w, t)
        x = h.double().cpu() @ w.double().cpu().nan_to_num(neginf=0.0).T
        x[:, 7] = -math.inf
        lp, ent, _, _ = O.token_logprobs(x.numpy(), t.cpu().numpy())
        off = 2 * 16 * E * math.sqrt(d) * float((h.double().square() @ w.double().nan_to_num(neginf=0.0).square().T).max().sqrt())
        close(f64(out.logprobs), lp, lp_tol(lp, v) + off, "logprobs")
        close(f64(out.entropy), ent, ent_tol(v) + off * (1 + math.log(v)), "entropy")
        for bad in (math.nan, math.inf):
            w[9, 3] = bad
            out = T.linear_token_logprobs(h, w, t)
            live = t != -100
            assert out.logprobs[live].isnan().all() and out.entropy[live].isnan().all() and (out.logprobs[~live] == 0).all()


def test_head_and_hidden_rows_gigabytes_apart():
    """Offsets between 2^31 and 2^32 bytes inside a tile: 64 head rows, and then 60 hidden states, 33,000,000 elements apart."""
    far = 33_000_000
    buf = torch.empty(63 * far + 64, dtype=torch.bfloat16, device="cuda")
    h, w0 = head(60, 64, 64, torch.bfloat16, 4)
    t = some_tokens(60, 64, 5)
    w = buf.as_strided((64, 64), (far, 1))
    w.copy_(w0)
    want = check_head(h, w, t)
    assert torch.equal(want.logprobs, T.linear_token_logprobs(h, w0, t).logprobs)
    x = buf.as_strided((60, 64), (far, 1))
    x.copy_(h)
    assert torch.equal(T.linear_token_logprobs(x, w0, t).logprobs, want.logprobs)
