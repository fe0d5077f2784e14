"""dizo_amd.token_loss on the GPU at the ends of what its operands can hold."""
import math

import pytest
import torch

from dizo_amd import token_loss as T

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
