"""dizo_amd.prefix_attention on the GPU at the ends of its types."""
import math

import pytest
import torch

from dizo_amd import prefix_attention as P
from oracle import prefix as O
from test_gpu_prefix_attention import DT, bound, check, inputs, stored, values

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = [
    (1, 3, 2, 1, 2, 30, 9, 64),      # waves with keys for themselves
    (1, 2, 2, 1, 70, 90, 65, 80),    # tiles that waves share
    (1, 2, 2, 1, 70, 90, 65, 128),
    (1, 3, 2, 1, 2, 30, 1500, 112),  # a prompt in several parts
    (1, 2, 2, 1, 3, 20, 1500, 72),   # codes that do not lie in whole chunks
    (1, 2, 2, 1, 100, 100, 1500, 64),
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype, most", [("fp32", 3e38), ("bf16", 3e38), ("fp16", 6e4)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_means_of_values_near_a_types_largest(shape, dtype, most, bits):
    """Sums of such values are beyond fp32; what they weigh to is not."""
    q, own, pre = inputs(3, dtype, *shape)
    for v in (own.v, pre.v):
        v.copy_((torch.rand(v.shape, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV) / 4 + 0.75) * most)
        v[..., 3::7] = 0.5
    own.v[:, -1, :, 1] *= -1
    if bits == 8:
        own, pre = stored(own), stored(pre)
    check(dtype, q, own, pre)


CODE_SHAPES = [
    (1, 3, 2, 1, 2, 30, 9, 128),     # whole chunks, by waves with keys for themselves
    (1, 2, 2, 1, 70, 90, 65, 64),    # converted on the way, tiles that waves share
    (1, 3, 2, 1, 2, 30, 1500, 112),  # a prompt in several parts
    (1, 2, 2, 1, 3, 20, 300, 72),    # half a chunk at the end
]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", CODE_SHAPES, ids=str)
@pytest.mark.parametrize("most", [0, 1, 5, 26, 40])
def test_scales_of_the_least_powers(most, shape, dtype):
    """Stores that were not filled by cache_write: a slot's values are code 2^(s - 127) for every s from 0 on."""
    q, own, pre = inputs(5, dtype, *shape, bits=8)
    g = torch.Generator(device=DEV).manual_seed(6)
    for store in (own, pre):
        s = store.v_scale.view(torch.uint8)
        s.copy_(torch.randint(0, most + 1, s.shape, generator=g, device=DEV))
    width, keys = shape[-1], shape[5] + shape[6]
    got = P.shared_prefix_attention(q, own, pre).cpu().double()
    out, spread, reach = O.attend(q, values(own), values(pre), None, None, width ** -0.5)
    # Below 2^-126 a bf16 number has steps of 2^-133 and an fp32 one of 2^-149: half of the first for a value that is converted on the way and
    # for the result, of the second for each product; or, for a weight that has its value's power, half of the first next to 2^16 for
    # the largest weight, of codes up to 448.
    lost = 2 * 2.0**-134 + keys * (2.0**-150 + 448 * 2.0**-134 * 2.0**-16)
    far, most_far = (got - out).abs(), bound(dtype, out, spread, reach, keys, width, 8) + lost
    assert (far <= most_far).all(), f"{float((far / most_far).max())} times the bound"
    assert (most_far < spread).all()  # it says something


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", CODE_SHAPES, ids=str)
@pytest.mark.parametrize("which", ["v_scale", "k_scale"])
def test_a_scale_of_255_is_nan(which, shape, dtype):
    q, own, pre = inputs(7, dtype, *shape, bits=8)
    slots, heads = shape[5], shape[2] // shape[3]
    scale = getattr(own, which).view(torch.uint8)
    scale[0, -1, 0, slots - 1] = 255  # seen by the last sequence's last token, by the first key head's queries
    got = P.shared_prefix_attention(q, own, pre).cpu().double()
    assert torch.isnan(got[0, -1, :heads, -1]).all()
    scale[0, -1, 0, slots - 1] = 127
    out, spread, reach = O.attend(q, values(own), values(pre), None, None, shape[-1] ** -0.5)
    far, most = (got - out).abs(), bound(dtype, out, spread, reach, slots + shape[6], shape[-1], 8)
    far[0, -1, :heads, -1] = 0.0
    assert (far <= most).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_reading_scales_of_every_kind(dtype):
    cache = P.QuantizedKV.empty(1, 256, 16, device=DEV)
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes.view(torch.uint8).copy_(torch.arange(256 * 16, device=DEV).view(1, 256, 16) * 37 % 256)
        scales.view(torch.uint8).copy_(torch.arange(256, device=DEV).view(1, 256))
    codes = O.CODE_VALUES[cache.k.view(torch.uint8).cpu().long()]
    power = torch.exp2(torch.arange(256, dtype=torch.float64) - 127)
    power[255] = math.nan
    want = (codes * power.view(1, 256, 1)).float().to(DT[dtype])  # (exact in fp32, but for what is beyond it)
    for got in P.cache_read(cache, 256, DT[dtype]):
        got = got.cpu()
        assert ((got == want) | (torch.isnan(got) & torch.isnan(want))).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_the_largest_numbers_are_kept(dtype):
    """The nearest code of a number above 248 2^120 stands for 2^128, which is none of fp32 or bf16."""
    top = torch.finfo(DT[dtype]).max
    k = torch.ones(1, 9, 16, dtype=DT[dtype], device=DEV)
    for i, x in enumerate((1.0, 0.99, 0.98, 0.97, 0.9375, 0.93, 0.9, 0.875, 0.5)):
        k[0, i, 3] = x * top
        k[0, i, 4] = -x * top
    cache = P.QuantizedKV.empty(1, 9, 16, device=DEV)
    P.cache_write(cache, k, -k, 0)
    got = P.cache_read(cache, 9, DT[dtype])
    most = 240.0 * 2.0 ** (8 if dtype == "fp16" else 120)
    kept = k.cpu().double().clamp(-most, most)
    far = (got.k.cpu().double() - kept).abs()
    # half a step of a code: 2^-4 of the value, or 2^-10 of 2^e
    assert (far <= torch.maximum(kept.abs() * 2.0**-4, torch.tensor(2.0**-10 * most / 240, dtype=torch.float64))).all()
    assert torch.equal(got.v, -got.k) and torch.isfinite(got.k).all()
