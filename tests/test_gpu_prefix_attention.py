"""dizo_amd.prefix_attention on the GPU against its definition in 64 bits (oracle.prefix)."""
import math

import numpy as np
import pytest
import torch

from dizo_amd import prefix_attention as P
from oracle import prefix as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"fp32": 2.0**-24, "fp16": 2.0**-11, "bf16": 2.0**-8}


def bound(dtype, out, spread, reach, keys, width, bits):
    """How far a result may be from the definition. Roundings: the result's (half a step of it); the weights', each half a step of
    a 16-bit type (bf16 with an 8-bit store, since a weight carries its value's power of two then), of sum w |v|; the scores', (width + 4) sums and products in fp32 of sum |q k|, which a weight shows as
    a relative error and twice that once it is divided by the sum; exp2's few units; keys sums and products of w v in fp32. An
    fp16 result below 2^-14 rounds in steps of 2^-24."""
    half = HALF_STEP[dtype]
    weights = 0 if dtype == "fp32" else HALF_STEP["bf16"] if bits == 8 else half
    scores = 2 * (width + 8) * 2.0**-24 * reach.unsqueeze(-1) + 2.0**-20
    floor = 2.0**-25 if dtype == "fp16" else 0.0
    return half * out.abs() + spread * (weights + scores + (keys + 64) * 2.0**-24) * (1 + weights) + floor


def inputs(seed, dtype, groups, sequences, heads, kv_heads, length, slots, prefix, width, bits=16, std=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def made(*shape):
        x = torch.randn(*shape[:-3], shape[-2], shape[-3], shape[-1], generator=g, device=DEV) * std
        return x.to(DT[dtype]).transpose(-3, -2)

    q = made(groups, sequences, heads, length, width)
    own = P.KV(made(groups, sequences, kv_heads, slots, width), made(groups, sequences, kv_heads, slots, width)) if slots else None
    pre = P.KV(made(groups, kv_heads, prefix, width), made(groups, kv_heads, prefix, width)) if prefix else None
    if bits == 8:
        own, pre = (None if s is None else stored(s) for s in (own, pre))
    return q, own, pre


def stored(kv):
    cache = P.QuantizedKV.empty(*kv.k.shape, device=DEV)
    P.cache_write(cache, kv.k, kv.v, 0)
    return cache


def values(store):
    if store is None or len(store) == 2:
        return store
    return [c.double() * s.double().unsqueeze(-1) for c, s in zip(store[:2], store[2:])]


def check(dtype, q, own, pre, positions=None, prefix_lengths=None, scale=None, got=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    if got is None:
        got = P.shared_prefix_attention(q, own, pre, positions=positions, prefix_lengths=prefix_lengths, scale=scale)
    assert got.shape == q.shape and got.dtype == q.dtype
    out, spread, reach = O.attend(q, values(own), values(pre), positions, prefix_lengths, scale)
    keys = (own[0].shape[-2] if own else 0) + (pre[0].shape[-2] if pre else 0)
    far = (got.cpu().double() - out).abs()
    most = bound(dtype, out, spread, reach, keys, q.shape[-1], 8 if len(own or pre) == 4 else 16)
    assert torch.isfinite(got).all()
    assert (far <= most).all(), f"{float((far / most.clamp(min=1e-300)).max())} times the bound"
    return got


SHAPES = [
    # groups, sequences, heads, kv_heads, length, slots, prefix, width
    (1, 1, 1, 1, 1, 1, 0, 64),      # one token, one key
    (1, 1, 1, 1, 1, 0, 1, 64),      # one key of a prompt, none of its own
    (2, 3, 4, 2, 1, 7, 5, 128),     # single tokens, shared key heads
    (1, 9, 3, 3, 1, 33, 100, 80),   # a width between the tiles', slots past one tile
    (2, 2, 2, 2, 6, 6, 61, 128),    # candidates
    (1, 5, 4, 1, 7, 40, 64, 64),    # 28 rows a sequence: tiles of one sequence each
    (1, 3, 2, 2, 33, 33, 65, 64),   # one row more than the smallest tile has
    (1, 2, 2, 1, 100, 130, 129, 96),  # 200 rows a sequence: tiles inside of it
    (1, 1, 2, 2, 257, 257, 0, 80),  # a causal sequence
    (3, 1, 1, 1, 129, 129, 1, 8),   # the narrowest head
    (1, 40, 1, 1, 1, 3, 700, 72),   # more sequences than a tile has rows
    (1, 2, 1, 1, 2, 2, 1500, 104),  # a prompt over several workgroups
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(shape, bits, dtype):
    q, own, pre = inputs(sum(shape), dtype, *shape, bits=bits)
    check(dtype, q, own, pre)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("shape", [SHAPES[2], SHAPES[5], SHAPES[7]], ids=str)
def test_positions_and_prefix_lengths(shape, bits):
    groups, sequences, _, _, length, slots, prefix, _ = shape
    q, own, pre = inputs(7, "fp16", *shape, bits=bits)
    r = np.random.default_rng(3)
    # before the first slot, past the last one, and in between
    positions = torch.from_numpy(r.integers(-length - 1, slots + 2, (groups, sequences))).int().to(DEV)
    lengths = torch.from_numpy(r.integers(0, prefix + 1, groups)).int().to(DEV)
    check("fp16", q, own, pre, positions, lengths)
    lengths = torch.tensor([-3, prefix + 9][:groups], dtype=torch.int32, device=DEV)
    check("fp16", q, own, pre, positions, lengths)


@pytest.mark.parametrize("bits", [16, 8])
def test_queries_that_see_nothing_give_zero(bits):
    q, own, pre = inputs(1, "bf16", 2, 3, 2, 2, 4, 9, 5, 64, bits=bits)
    positions = torch.tensor([[-4, -2, 0], [-100, 3, -4]], dtype=torch.int32, device=DEV)
    got = check("bf16", q, own, pre, positions, torch.tensor([0, 0], dtype=torch.int32, device=DEV))
    assert (got[0, 0] == 0).all() and (got[0, 1, :, :1] == 0).all() and (got[1, 0] == 0).all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("length, slots", [(1, 40), (40, 200)])
def test_slots_that_no_query_sees_do_not_matter(length, slots, bits):
    q, own, pre = inputs(5, "fp16", 1, 4, 2, 2, length, slots, 70, 64, bits=bits)
    positions = torch.tensor([[0, 3, slots - length - 1, 17 if length == 1 else 30]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([37], dtype=torch.int32, device=DEV)
    want = P.shared_prefix_attention(q, own, pre, positions=positions, prefix_lengths=lengths)
    for x in own[:2]:
        for n in range(4):
            x[:, n, :, int(positions[0, n]) + length:].view(torch.uint8).fill_(255)  # NaN of all three types, and of codes
    for x in pre[:2]:
        x[:, :, 37:].view(torch.uint8).fill_(255)
    assert torch.equal(P.shared_prefix_attention(q, own, pre, positions=positions, prefix_lengths=lengths), want)


def test_large_scores_and_their_differences():
    # scores of some thousands: the weights of the largest are far from those of the next
    q, own, pre = inputs(2, "bf16", 1, 3, 2, 2, 5, 40, 90, 128, std=16.0)
    check("bf16", q, own, pre, scale=0.5)
    q, own, pre = inputs(3, "fp32", 1, 3, 2, 2, 5, 40, 90, 128, std=1e-3)
    check("fp32", q, own, pre, scale=1.0)


def test_strided_misaligned_and_transposed_operands():
    q, own, pre = inputs(4, "fp16", 1, 3, 2, 2, 5, 20, 33, 64)
    want = P.shared_prefix_attention(q, own, pre)
    flat = torch.zeros(q.numel() + 1, dtype=q.dtype, device=DEV)[1:]
    odd = flat.view(q.shape)  # rows at multiples of 2 bytes
    odd.copy_(q)
    wide = [torch.zeros(*x.shape[:-1], 80, dtype=x.dtype, device=DEV)[..., 5:69] for x in own]
    for w, x in zip(wide, own):
        w.copy_(x)
    heads_last = [x.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2) for x in pre]  # the width is not contiguous
    assert torch.equal(P.shared_prefix_attention(odd, P.KV(*wide), P.KV(*heads_last)), want)
    room = torch.full((1, 5, 3, 2, 72), 7.0, dtype=q.dtype, device=DEV)
    out = room.permute(0, 2, 3, 1, 4)[..., :64]
    assert P.shared_prefix_attention(q, own, pre, out=out) is out
    assert torch.equal(out, want) and (room[..., 64:] == 7).all()


def test_results_do_not_depend_on_the_batch_around_them():
    q, own, pre = inputs(6, "fp16", 2, 5, 2, 2, 3, 50, 200, 64)
    both = P.shared_prefix_attention(q, own, pre)
    one = P.shared_prefix_attention(q[1:], P.KV(own.k[1:], own.v[1:]), P.KV(pre.k[1:], pre.v[1:]))
    assert torch.equal(both[1:], one)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("width", [8, 64, 80, 128])
def test_cache_write_and_read(dtype, width):
    g = torch.Generator(device=DEV)
    g.manual_seed(width)
    k, v = (torch.randn(3, 5, 4, width, generator=g, device=DEV).mul(s).to(DT[dtype]).transpose(1, 2) for s in (1.0, 30.0))
    k[0, 0, 0] = 0.0
    k[0, 1, 0] = torch.linspace(-1, 1, width) * (6e4 if dtype == "fp16" else 3e38)
    k[0, 2, 0, 0] = math.nan
    k[0, 3, 0, 1] = math.inf
    k[1, 0, 0] = 448.0
    k[1, 1, 0] = 449.0 if dtype != "bf16" else 450.0
    k[1, 2, 0] = torch.linspace(0, 1, width) * (6e-8 if dtype == "fp16" else 1e-38)
    if dtype == "fp16":
        k[1, 3, 0, :3] = torch.tensor([65504.0, -65504.0, 63000.0])
    cache = P.QuantizedKV.empty(3, 4, 9, width, device=DEV)
    for x in cache:
        x.view(torch.uint8).fill_(0x55)
    positions = torch.tensor([0, 4, 2], dtype=torch.int32, device=DEV)
    P.cache_write(cache, k, v, positions)
    for x, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        want, e = O.quantize(x, dtype == "fp16")
        for b, at in enumerate(positions.tolist()):
            inside = slice(at, at + 5)
            got = O.CODE_VALUES[codes[b, :, inside].contiguous().view(torch.uint8).cpu().long()]
            assert torch.equal(got.nan_to_num(1e9), want[b].nan_to_num(1e9))
            assert torch.equal(scales[b, :, inside].float().cpu().double(), e[b])
            rest = torch.ones(9, dtype=torch.bool)
            rest[inside] = False
            assert (codes[b].view(torch.uint8)[:, rest] == 0x55).all() and (scales[b].view(torch.uint8)[:, rest] == 0x55).all()
    # what reading gives: code 2^e, which every type but fp16's subnormals holds exactly, and those too (the codes came from it)
    kr, vr = P.cache_read(cache, 9, DT[dtype])
    for got, codes, scales in ((kr, cache.k, cache.k_scale), (vr, cache.v, cache.v_scale)):
        b, at = 1, 4
        want = O.CODE_VALUES[codes[b, :, at:at + 5].contiguous().view(torch.uint8).cpu().long()] * scales[b, :, at:at + 5].cpu().double().unsqueeze(-1)
        assert torch.equal(got[b, :, at:at + 5].cpu().double(), want)
        part = P.cache_read(cache, 2, DT[dtype], start=5)
        assert torch.equal(part.k.nan_to_num(1e4), kr[:, :, 5:7].nan_to_num(1e4))


def test_cache_write_leaves_out_what_does_not_fit():
    k = torch.ones(2, 1, 4, 64, device=DEV, dtype=torch.float16)
    cache = P.QuantizedKV.empty(2, 1, 6, 64, device=DEV)
    for x in cache:
        x.view(torch.uint8).fill_(0x55)
    P.cache_write(cache, k, k, torch.tensor([-2, 4], dtype=torch.int32, device=DEV))
    there = torch.tensor([[True, True, False, False, False, False], [False, False, False, False, True, True]], device=DEV)
    codes = cache.k.view(torch.uint8)[:, 0]
    assert ((codes != 0x55).all(-1) == there).all() and ((codes == 0x55).all(-1) == ~there).all()
