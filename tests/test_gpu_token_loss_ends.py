"""dizo_amd.token_loss on the GPU at the ends of what its operands can hold."""
import math

import numpy as np
import pytest
import torch

from dizo_amd import token_loss as T
from oracle import vocab as O

pytestmark = pytest.mark.gpu


def rows(n, v, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, v, generator=g) * spread).to(dtype).cuda()


@pytest.mark.parametrize("exponent", [20, 30, 40, 60, 100])
@pytest.mark.parametrize("v", [50, 9001])
def test_large_entropy_weights_beside_masked_columns(v, exponent):
    """The gradient is linear in the weights, and a weight that is a power of two changes no rounding: it has the bits
    of the gradient of weight 1, scaled. A masked column's is 0 whatever the weight is."""
    x = rows(4, v, torch.float32, v)
    x[:, v // 3:] = -math.inf
    x[1, : v // 3] = torch.finfo(torch.float32).min  # uniform over them
    x[2, 1:] = torch.finfo(torch.float32).min  # one token alone, the others impossible at any distance
    x[3, : v // 3] -= 1000.0 * torch.arange(v // 3, device="cuda") / v
    t = torch.tensor([0, 1, 0, 3], device="cuda")
    u = torch.tensor([1.0, -1.0, 1.0, 0.5], device="cuda")
    _, one = T.token_logprobs_grad(x, t, None, u)
    _, g = T.token_logprobs_grad(x, t, None, u * 2.0**exponent)
    assert torch.equal(g, one * 2.0**exponent)
    assert not g[:, v // 3:].any() and not g.isnan().any()


@pytest.mark.parametrize("tau", [0.25, 0.5, 0.7, 1.0, 3.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_teacher_values_at_the_limits_of_fp32(dtype, tau):
    """Entries masked by the type's lowest value, and its largest: a row of equal ones is uniform at every temperature,
    and the lowest have weight 0 beside others.

    Differences to the largest value are 0, exact or past every exponent here, so that a weight is off by
    (2 k + 10) e; the loss T^2 sum w (ln w - ln q) by T^2 e (v / 256 + 60 + 2 k + 4 max |x| / T) (1 + sum w (|ln w| + |ln q|)),
    a gradient by T e (v / 256 + 100 + 2 k + 4 max |x| / T) (q + w)."""
    v, k = 500, 6
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = rows(7, v, torch.float32, 3)
    at = torch.stack([torch.randperm(v, generator=torch.Generator().manual_seed(i))[:k] for i in range(7)]).cuda()
    val = torch.zeros(7, k, dtype=dtype, device="cuda")
    val[0] = low
    val[1] = high
    val[2, 1:] = low
    val[3] = low
    val[3, 2] = high
    val[4] = low
    val[4, 3:] = -math.inf
    val[5, ::2] = high
    val[6] = low
    at[6, 1:] = -1
    w = torch.linspace(0.5, 1.5, 7, device="cuda")
    loss, grad = T.topk_distill_grad(x, val, at, w, temperature=tau)
    x64, val64, at64, w64 = (t.double().cpu().numpy() for t in (x, val, at, w))
    at64 = at64.astype(np.int64)
    want, want_grad = O.topk_distill(x64, val64, at64, tau, True, w64)
    assert np.isfinite(want).all()
    logq = O.log_softmax(x64 / tau)
    e, steps = 2.0**-24, v / 256 + 60 + 2 * k + 4 * np.abs(x64).max() / tau
    for r in range(7):
        tw, tl = O.teacher_weights(val64[r], at64[r], v, tau, True)
        there = tw > 0
        size = (tw[there] * (np.abs(tl[there]) + np.abs(logq[r][at64[r][there]]))).sum()
        assert abs(float(loss[r]) - want[r]) <= tau * tau * e * steps * (1 + size), r
        term = np.exp(logq[r])
        np.add.at(term, at64[r][there], tw[there])
        assert (np.abs(grad[r].double().cpu().numpy() - want_grad[r]) <= tau * w64[r] * e * (steps + 40) * term + 2.0**-126).all(), r
    assert torch.equal(T.topk_distill(x, val, at, temperature=tau).isnan(), torch.zeros(7, dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("tau", [0.3, 0.5, 0.9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_masked_student_logits_that_a_temperature_takes_past_fp32(dtype, tau):
    """A student's logits at the type's lowest value, of which a teacher's entries name some: their log probabilities
    divided by a temperature below 1 are no numbers of fp32, the distance is. Within T^2 e (v / 256 + 60 + k + 4 max |t| / T)
    (1 + sum w (|ln w| + |ln q|)); a masked logit of -inf stays an infinite distance."""
    v, k = 700, 5
    x = rows(6, v, dtype, 5)
    g = torch.Generator().manual_seed(6)
    at = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(6)]).cuda()
    val = (torch.randn(6, k, generator=g) * 4).cuda()
    low = torch.finfo(dtype).min
    x[0, at[0, 2]] = low
    x[1, at[1]] = low
    x[2, : v // 2] = low
    val[3, 4] = -40 * tau  # little weight, and a large distance for it
    x[3, at[3, 4]] = low
    x[4, at[4, 1]] = -math.inf
    x[5, at[5, 0]], x[5, at[5, 1]] = low, -math.inf
    x64, val64, at64 = x.double().cpu().numpy(), val.double().cpu().numpy(), at.cpu().numpy()
    want, _ = O.topk_distill(x64, val64, at64, tau)
    assert np.isfinite(want[:4]).all() and (want[:2] > 1e20).all() and np.isinf(want[4:]).all()
    logq = O.log_softmax(x64 / tau)
    w = torch.ones(6, device="cuda")
    for got in (T.topk_distill(x, val, at, temperature=tau), T.topk_distill_grad(x, val, at, w, temperature=tau)[0]):
        got = got.double().cpu().numpy()
        for r in range(4):
            tw, tl = O.teacher_weights(val64[r], at64[r], v, tau, True)
            size = (tw * (np.abs(tl) + np.abs(logq[r][at64[r]]))).sum()
            steps = v / 256 + 60 + k + 4 * np.abs(val64[r]).max() / tau
            assert abs(got[r] - want[r]) <= tau * tau * 2.0**-24 * steps * (1 + size), (r, got[r], want[r])
        assert np.isposinf(got[4:]).all()


@pytest.mark.parametrize("tau", [0.5, 1.0, 1.7])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_student_logits_at_both_ends_of_their_type(dtype, tau):
    """The largest logit at the type's largest value and a named one at its lowest, whose difference is no number of fp32:
    the distance is one where the weight is small. Its size is w (max - min) T, off by the weight's (2 k + 10 + 4 max |t| / T) e."""
    v, k = 300, 4
    x = rows(2, v, dtype, 5)
    at = torch.tensor([[1, 2, 3, 4], [5, 6, 7, 8]], device="cuda")
    val = torch.tensor([[0.0, 0.0, 0.0, -20 * tau], [3.0, -9 * tau, 1.0, -30 * tau]], device="cuda")
    x[0, 1:4], x[0, 4] = torch.finfo(dtype).max, torch.finfo(dtype).min
    x[1, 5:8], x[1, 8] = torch.finfo(dtype).max, torch.finfo(dtype).min
    want, _ = O.topk_distill(x.double().cpu().numpy(), val.double().cpu().numpy(), at.cpu().numpy(), tau)
    for got in (T.topk_distill(x, val, at, temperature=tau), T.topk_distill_grad(x, val, at, torch.ones(2, device="cuda"), temperature=tau)[0]):
        tol = want * 2.0**-24 * (2 * k + 10 + 4 * val.abs().amax(-1).double().cpu().numpy() / tau + 10)
        assert (np.abs(got.double().cpu().numpy() - want) <= tol).all(), (got.tolist(), want.tolist())
