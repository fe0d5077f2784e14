"""dizo_amd.sampling on the GPU against its definition in 64 bits (oracle.prefix)."""
import math

import pytest
import torch

from dizo_amd.sampling import sample_tokens
from oracle import prefix as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def rows_of(seed, rows, vocab, dtype, std=3.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g, device=DEV) * std).to(DT[dtype]), torch.rand(rows, generator=g, device=DEV)


def check(x, u, **how):
    got = sample_tokens(x, u, **how)
    per_row = {k: (v.tolist() if torch.is_tensor(v) else [v] * x.shape[0]) for k, v in how.items()}
    want = [O.sample(x[i], float(u[i]), **{k: v[i] for k, v in per_row.items()}) for i in range(x.shape[0])]
    assert got.dtype == torch.int64 and got.tolist() == want


HOW = [
    {}, dict(temperature=0.7), dict(temperature=0.0), dict(top_k=1), dict(top_k=5), dict(top_k=50, temperature=1.5), dict(top_p=0.9),
    dict(top_p=0.5, temperature=2.0), dict(min_p=0.1), dict(top_k=20, top_p=0.8, min_p=0.05, temperature=0.8), dict(top_p=0.0), dict(min_p=1.0),
    dict(top_k=100000), dict(top_k=3, top_p=0.999),
]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 1000, 8193, 50257])
def test_distributions(vocab, dtype):
    for i, how in enumerate(HOW):
        x, u = rows_of(vocab + i, 3, vocab, dtype)
        check(x, u, **how)


@pytest.mark.parametrize("how", HOW, ids=str)
def test_equal_logits_go_by_their_token(how):
    x = torch.zeros(6, 3001, device=DEV, dtype=torch.float16)
    x[1, ::3] = 1.0
    x[2, 7:] = -1.0
    x[3] = torch.arange(3001, device=DEV).remainder(5).half()
    x[4, 1::2] = -0.0  # equals 0
    x[5, 1500:] = 3.0
    check(x, torch.tensor([0.0, 0.25, 0.999, 0.5, 0.123, 1.0], device=DEV), **how)


def test_parameters_of_each_row():
    x, u = rows_of(3, 6, 999, "fp32")
    check(x, u, temperature=torch.tensor([1.0, 0.0, 0.5, 2.0, 1.0, 1.0], device=DEV),
          top_k=torch.tensor([0, 5, 10, 1, 0, 2], dtype=torch.int32, device=DEV),
          top_p=torch.tensor([0.9, 1.0, 0.5, 0.3, 1.0, 0.0], device=DEV), min_p=torch.tensor([0.0, 0.1, 0.0, 0.2, 0.5, 1.0], device=DEV))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_rows_with_infinities_and_without_a_distribution(dtype):
    x, _ = rows_of(5, 8, 300, dtype)
    x[0, 10] = math.nan
    x[1] = -math.inf
    x[2, 40] = math.inf
    x[3, [50, 60, 70]] = math.inf
    x[4, 5:] = -math.inf
    x[5] = torch.finfo(x.dtype).min
    x[6, :299] = -math.inf
    x[7, 100:] = torch.finfo(x.dtype).min
    u = torch.tensor([0.5, 0.5, 0.9, 0.5, 0.5, 0.5, 0.0, 1.0], device=DEV)
    for how in ({}, dict(top_k=2), dict(top_p=0.6), dict(min_p=0.5), dict(top_k=299, top_p=0.99)):
        check(x, u, **how)
    assert sample_tokens(x, u)[:3].tolist() == [-1, -1, 40]
    bad = torch.full((8,), 0.5, device=DEV)
    bad[4] = math.nan
    assert sample_tokens(x, bad)[4] == -1 and sample_tokens(x, u, temperature=bad)[4] == -1


def test_strided_rows_and_leading_dimensions():
    x, u = rows_of(9, 12, 501, "bf16")
    y = torch.zeros(3, 5, 501, device=DEV, dtype=x.dtype)
    y[:, 1:] = x.view(3, 4, 501)
    assert torch.equal(sample_tokens(y[:, 1:], u.view(3, 4), top_p=0.9), sample_tokens(x, u, top_p=0.9).view(3, 4))
    last = y[:, -1]
    assert torch.equal(sample_tokens(last, u[:3]), sample_tokens(last.contiguous(), u[:3]))
    assert sample_tokens(x[:0], u[:0]).shape == (0,)


def test_frequencies():
    # 4,096 evenly spaced numbers: a token of probability p is drawn p 4096 times, give or take one at each border
    x = torch.tensor([0.0, 1.0, 2.0, -math.inf, 0.5], device=DEV)
    n = 4096
    got = sample_tokens(x.expand(n, 5), (torch.arange(n, device=DEV) + 0.5) / n)
    p = torch.softmax(x.double(), 0) * n
    assert ((torch.bincount(got, minlength=5).double() - p).abs() <= 1).all()


@pytest.mark.parametrize("how", [dict(top_p=0.3), dict(top_p=0.75, top_k=1500), dict(min_p=0.03), dict(top_k=700), dict(top_k=1200, top_p=0.5)], ids=str)
def test_logits_around_zero_where_numbers_lie_close(how):
    """A row's largest is 1 and nearly all of the others are within 1e-5 of 0: a bin's end is 1 - (32 n + 31) T ln 2 / 1024, at 0 to
    within 1e-16 by the temperature, where fp32 has more numbers than a search of the nearest ones covers."""
    g = torch.Generator(device=DEV)
    g.manual_seed(8)
    e = torch.rand(4, 3001, generator=g, device=DEV) * 35 - 40
    x = torch.pow(10.0, e) * torch.where(torch.rand(4, 3001, generator=g, device=DEV) < 0.5, -1.0, 1.0)
    x[:, ::5] = 0.0
    x[:, 17] = 1.0
    u = torch.tensor([0.1, 0.4, 0.7, 0.95], device=DEV)
    for n in (3, 10, 11):
        check(x, u, temperature=1024 / ((32 * n + 31) * math.log(2)), **how)


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-3, 1e4, 1e19, 3e38])
@pytest.mark.parametrize("how", [dict(), dict(top_p=0.6), dict(top_k=40, top_p=0.9), dict(top_k=2000), dict(min_p=0.2)], ids=str)
def test_logits_of_any_size(scale, how):
    x, u = rows_of(9, 4, 2500, "fp32", std=1.0)
    x = (x / 5).clamp(-1, 1) * scale
    for t in (0.05, 1.0, 30.0):
        if 2.0**-63 <= t * scale < 2.0**64:
            check(x, u, temperature=t * scale, **how)
    check(x[:1], u[:1], temperature=1.0, **how)  # all alike, or one alone
