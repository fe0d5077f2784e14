"""linear_token_logprobs of operands that require a gradient: under no_grad the logits are neither stored nor rounded;
where autograd records they are F.linear's, rounded to the operands' type."""
import math

import pytest
import torch

from dizo_amd import token_loss as T

pytestmark = pytest.mark.gpu

E = 2.0**-24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def operands(n, d, v, dtype):
    g = torch.Generator(device="cuda").manual_seed(n + d)
    h = torch.randn(n, d, generator=g, device="cuda").to(dtype)
    w = torch.randn(v, d, generator=g, device="cuda").mul_(2.5 / math.sqrt(d)).to(dtype)
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    t[3] = -100
    return h, w, t


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_no_grad_takes_the_kernel_for_parameters(dtype):
    h, w, t = operands(20, 128, 3000, dtype)
    want = T.linear_token_logprobs(h, w, t)
    h.requires_grad_(True)
    weight = torch.nn.Parameter(w)
    with torch.no_grad():
        got = T.linear_token_logprobs(h, weight, t)
    assert torch.equal(got.logprobs, want.logprobs) and torch.equal(got.entropy, want.entropy) and not got.logprobs.requires_grad


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_values_and_gradients_where_autograd_records(dtype):
    """With r half a step of the type and M the largest logit's size: a logit is off by a = r M + 16 e sqrt(d) |h * w|_2 (its
    rounding, its sum), a log probability by 2 a + e (4 |lp| + 4 ln v + v / 256 + 60). q is off by 2 a of itself and
    the logits' gradient is rounded (r, and the type's smallest number), so that the gradient of h, whose terms are (o - q) w,
    is off by (2 a + r + 16 e sqrt(v)) sum |o - q| |w| + half a smallest number times sum |w|, and rounded (r); the head's in the same way."""
    n, d, v = 20, 128, 3000
    h, w, t = operands(n, d, v, dtype)
    h.requires_grad_(True)
    w.requires_grad_(True)
    out = T.linear_token_logprobs(h, w, t)
    c = torch.linspace(0.5, 1.5, n, device="cuda")
    (c * out.logprobs).sum().backward()
    hd, wd = h.detach().double(), w.detach().double()
    x = hd @ wd.t().contiguous()
    logq = x - x.logsumexp(-1, keepdim=True)
    live = t != -100
    at = t.clamp(min=0).unsqueeze(-1)
    lp = torch.where(live, logq.gather(-1, at).squeeze(-1), 0.0)
    r = torch.finfo(dtype).eps / 2
    smallest = {torch.float32: 2.0**-126, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-126}[dtype]
    a = r * x.abs().amax(-1) + 16 * E * math.sqrt(d) * (hd.square() @ wd.square().t().contiguous()).amax(-1).sqrt()
    assert ((out.logprobs.double() - lp).abs() <= 2 * a + E * (4 * lp.abs() + 4 * math.log(v) + v / 256 + 60)).all()
    g = torch.zeros_like(x).scatter_(-1, at, 1.0) - logq.exp()
    g = torch.where(live.unsqueeze(-1), c.double().unsqueeze(-1) * g, 0.0)
    size = torch.where(live.unsqueeze(-1), g.abs(), 0.0)
    for got, want, terms, plain, k in ((h.grad, g @ wd, (2 * a + r + 16 * E * math.sqrt(v)).unsqueeze(-1) * (size @ wd.abs()), wd.abs().sum(0), v),
                                       (w.grad, g.t().contiguous() @ hd, ((2 * a + r + 16 * E * math.sqrt(n)).unsqueeze(-1) * size).t().contiguous() @ hd.abs(),
                                        hd.abs().sum(0), n)):
        tol = terms + smallest * plain + r * want.abs() + smallest
        assert got.dtype == dtype and ((got.double() - want).abs() <= tol).all(), float(((got.double() - want).abs() - tol).max())
