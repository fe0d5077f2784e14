"""dizo_amd.prefix_attention on the GPU: what many keys of small weights have in a result."""
import math

import pytest
import torch

from dizo_amd import prefix_attention as P
from oracle import prefix as O
from test_gpu_prefix_attention import DT, bound, inputs, stored, values

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("width", [64, 72])
@pytest.mark.parametrize("nats", [8.0, 12.0, 18.0, 22.0])
@pytest.mark.parametrize("length, keys", [(1, 1 << 20), (1, 1 << 17), (24, 1 << 17), (130, 1 << 16), (17920, 1 << 16)])  # the last: no two workgroups share a row's keys
@pytest.mark.parametrize("dtype, bits", [("fp16", 16), ("fp16", 8), ("bf16", 16), ("fp32", 16)])
def test_a_key_above_many_others(dtype, bits, length, keys, nats, width):
    """One key is `nats` above all others, whose values are about 1, and its own are 0: the result is what the others weigh,
    T / (1 + T) with T = keys e^-nats."""
    g = torch.Generator(device=DEV)
    g.manual_seed(width)
    at = {1: keys // 3, 24: 5, 130: keys - 7, 17920: 2}[length]
    k = torch.zeros(1, 1, keys, width, dtype=DT[dtype], device=DEV)
    k[0, 0, at, 0] = nats
    v = (1 + torch.randn(1, 1, keys, width, generator=g, device=DEV) / 8).to(DT[dtype])
    v[0, 0, at] = 0.0
    q = torch.zeros(1, 1, 1, length, width, dtype=DT[dtype], device=DEV)
    q[..., 0] = 1.0
    store = P.KV(k, v) if bits == 16 else stored(P.KV(k, v))
    got = P.shared_prefix_attention(q, None, store, scale=1.0).cpu().double()
    out, spread, reach = O.attend(q[:, :, :, :1], None, values(store), None, None, 1.0)  # (the rows are alike)
    # a 16-bit weight's half step, and of a fp16 one 2^-36 of the largest
    most = bound(dtype, out, spread, reach, keys, width, bits) + (keys * 2.0**-36 * float(v.max()) if dtype == "fp16" else 0.0)
    assert (most < out / 4).all() or math.exp(nats) * 64 > keys  # it says something
    far = (got - out).abs()
    assert (far <= most).all(), f"{float((far / most).max())} times the bound"


@pytest.mark.parametrize("shape", [
    (2, 3, 4, 2, 1, 7, 5, 128),      # codes in whole chunks of 16, by waves with keys for themselves
    (1, 9, 3, 3, 2, 33, 100, 80),
    (1, 2, 2, 1, 50, 70, 129, 96),
    (1, 2, 2, 1, 40, 70, 3000, 64),  # prompts in several parts
    (2, 3, 4, 2, 1, 7, 5, 120),      # half a chunk at the end
    (1, 2, 2, 1, 100, 130, 129, 64),  # tiles that waves share
], ids=str)
@pytest.mark.parametrize("std", [1.0, 4.0])
def test_fp16_queries_keep_their_bits_beside_8_bit_stores(shape, std):
    """However the codes lie: fp16's half step for the weights, and not bf16's."""
    q, own, pre = inputs(sum(shape), "fp16", *shape, bits=8, std=std)
    got = P.shared_prefix_attention(q, own, pre).cpu().double()
    out, spread, reach = O.attend(q, values(own), values(pre), None, None, shape[-1] ** -0.5)
    far = (got - out).abs()
    most = bound("fp16", out, spread, reach, shape[5] + shape[6], shape[-1], 16)
    assert (far <= most).all(), f"{float((far / most).max())} times the bound"
