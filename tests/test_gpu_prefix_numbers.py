"""dizo_amd.prefix_attention and sampling on the GPU: numbers that do not fit where they go are refused, and not taken as others."""
import numpy as np
import pytest
import torch

from dizo_amd import prefix_attention as P
from dizo_amd._lib import DzError
from dizo_amd.sampling import sample_tokens
from test_gpu_prefix_attention import inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("at", [2**32, 2**64, 2**64 + 1, -(2**63), 10**30, 6, -1])
def test_positions_past_64_bits_are_not_wrapped(at):
    cache = P.QuantizedKV.empty(2, 1, 8, 16, device=DEV)
    for x in cache:
        x.view(torch.uint8).fill_(0x55)
    k = torch.randn(2, 1, 3, 16, device=DEV)
    with pytest.raises(DzError, match="fit"):
        P.cache_write(cache, k, k, at)
    with pytest.raises(DzError, match="slots"):
        P.cache_read(cache, 3, torch.float32, start=at)
    assert all((x.view(torch.uint8) == 0x55).all() for x in cache)


@pytest.mark.parametrize("scale", ["one", [], 1e39, 10**400, float("nan"), float("inf"), 0, -1, 2.0**127, 1e-300], ids=lambda x: str(x)[:8])
def test_scales(scale):
    q, own, pre = inputs(1, "bf16", 1, 2, 2, 1, 3, 5, 4, 64)
    with pytest.raises(DzError, match="scale"):
        P.shared_prefix_attention(q, own, pre, scale=scale)


def test_scales_of_other_types():
    q, own, pre = inputs(1, "bf16", 1, 2, 2, 1, 3, 5, 4, 64)
    want = P.shared_prefix_attention(q, own, pre, scale=0.25)
    for scale in (np.float32(0.25), np.float64(0.25), torch.tensor(0.25)):
        assert torch.equal(P.shared_prefix_attention(q, own, pre, scale=scale), want)
    assert torch.equal(P.shared_prefix_attention(q, own, pre, scale=1), P.shared_prefix_attention(q, own, pre, scale=1.0))


@pytest.mark.parametrize("how", [dict(temperature=10**400), dict(top_p=10**400), dict(min_p=-(10**400)), dict(top_k=2**31), dict(top_k=2**32 + 1)], ids=lambda h: next(iter(h)))
def test_parameters_that_no_number_of_theirs_holds(how):
    with pytest.raises(DzError, match=next(iter(how))):
        sample_tokens(torch.randn(2, 50, device=DEV), torch.rand(2, device=DEV), **how)
