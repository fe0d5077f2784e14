"""The products of many fp32 rows are taken of three bf16 parts a number; two of the nine products of the parts are
left out at up to 2^-25 of the number's each. Operands where they are that large, of one sign along the width."""
import pytest
import torch

from dizo_amd import token_loss as T

pytestmark = pytest.mark.gpu

E = 2.0**-24
N, V = 100, 33000  # the fewest rows and tokens that the parts are taken of


@pytest.mark.parametrize("d", [64, 768, 1000])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_operands_whose_parts_are_largest(d, sign):
    """One token's logit is a sum of d equal products, S together; the others' are 0. Its log probability is off by what
    is left out (2^-24 of S), by the roundings of the sum (6 d / 32 matrix products, of four steps each at most, every one off by
    at most e S), and by the statistics' (e (4 |lp| + 4 ln v + v / 256 + 60))."""
    worst = 1 + 2.0**-8 - 2.0**-17
    scale = 2.0**-7
    h = torch.full((N, d), worst, device="cuda")
    h[1::2] *= 2.0**-3
    w = torch.zeros(V, d, device="cuda")
    w[V - 5] = sign * worst * scale
    t = torch.full((N,), V - 5, device="cuda")
    t[::3] = 17
    out = T.linear_token_logprobs(h, w, t)
    x = h.double() @ w.double().t().contiguous()
    logq = x - x.logsumexp(-1, keepdim=True)
    lp = logq.gather(-1, t.unsqueeze(-1)).squeeze(-1)
    size = x[:, V - 5].abs()
    tol = E * size * (1 + 24 * d / 32 + 24) + E * (4 * lp.abs() + 4 * 10.41 + V / 256 + 60)
    assert ((out.logprobs.double() - lp).abs() <= tol).all()


def test_parts_of_numbers_of_every_size():
    """Numbers of 24 bits from 2^-40 to 2^40, whose products are of one size: logits of hidden states scaled by column
    against a head scaled the other way by the same powers of two are those of the operands unscaled, to the bit."""
    g = torch.Generator(device="cuda").manual_seed(1)
    d = 768
    h = torch.randn(N, d, generator=g, device="cuda")
    w = torch.randn(V, d, generator=g, device="cuda") * (2.0 / d**0.5)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    by = torch.tensor([2.0**k for k in range(-40, 41)], device="cuda")[torch.randint(0, 81, (d,), generator=g, device="cuda")]  # (a power taken on the GPU may be off)
    a, b = T.linear_token_logprobs(h, w, t), T.linear_token_logprobs(h * by, w / by, t)
    assert torch.equal(a.logprobs, b.logprobs) and torch.equal(a.entropy, b.entropy)
