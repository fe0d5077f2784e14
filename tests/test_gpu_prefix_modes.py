"""Candidates and answers that share a prompt: captured graphs, streams, refusals that need operands, many workgroups, and offsets
past 32 bits."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from dizo_amd import _lib as L
from dizo_amd import prefix_attention as P
from dizo_amd._lib import DzError
from dizo_amd.sampling import sample_tokens
from dizo_amd.table import stream_handle
from test_gpu_prefix_attention import check, inputs, stored

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("shape", [
    (1, 1, 523, 523, 1, 2, 700, 16),   # 66 items an XCD: 64 at a time, and two in two parts each
    (1, 1, 131, 131, 33, 33, 1100, 24),  # 17 larger tiles an XCD
    (1, 1, 9, 9, 33, 33, 1100, 24),    # 2, in four parts
    (1, 2, 270, 270, 40, 50, 600, 40),  # 34, of which two are in two parts
    (2, 3, 4, 2, 12, 20, 600, 64),     # 24 rows a sequence: waves take keys for themselves
    (1, 1, 520, 520, 24, 24, 40, 16),  # the same, two waves an item
    (1, 1, 1100, 1100, 20, 20, 30, 24),  # one wave an item
    (1, 1, 2060, 2060, 1, 2, 700, 16),  # the same, 258 an XCD: 256 at a time, and two in two parts each
    (1, 1, 520, 520, 24, 24, 1000, 16),  # many keys: shared tiles
    (1, 3, 100, 100, 40, 50, 1000, 24),  # shared tiles of three sequences
    (1, 2, 2, 1, 60, 70, 300, 104),    # shared tiles of wide heads
    (1, 2, 4, 2, 40, 60, 100, 64),     # 80 rows in tiles of 32
    (1, 1, 2, 2, 300, 310, 20, 112),   # codes of wide heads in tiles of 32, 16 bits in shared ones
    (2, 66, 4, 4, 1, 20, 300, 64),     # several tiles of sequences, with keys of their own
    (1, 2, 8, 2, 40, 77, 513, 128),    # 160 rows a sequence
], ids=str)
def test_many_workgroups_and_parts(shape, bits):
    q, own, pre = inputs(11, "fp16", *shape, bits=bits)
    positions = torch.from_numpy(np.random.default_rng(1).integers(0, shape[5] - shape[4] + 1, shape[:2])).int().to(DEV)
    check("fp16", q, own, pre, positions)


def test_captured_calls_see_what_their_operands_hold():
    q, own, pre = inputs(3, "bf16", 1, 4, 2, 2, 1, 30, 1200, 64)
    qb, ob, pb = q, stored(own), stored(pre)
    positions = torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    lengths = torch.tensor([900], dtype=torch.int32, device=DEV)
    logits, u = torch.randn(6, 5000, device=DEV), torch.rand(6, device=DEV)
    k = torch.randn(1, 4, 2, 1, 64, device=DEV).bfloat16()
    where = torch.zeros(1, 4, dtype=torch.int32, device=DEV)

    def run():
        P.cache_write(ob, k, k, where)
        return (P.shared_prefix_attention(q, own, pre, positions=positions, prefix_lengths=lengths), P.shared_prefix_attention(qb, ob, pb, positions=positions),
                *P.cache_read(ob, 30, torch.bfloat16), sample_tokens(logits, u, top_k=40, top_p=0.9), sample_tokens(logits, u, top_p=0.7, min_p=0.01))

    run()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(run())
    for i in range(5):
        q.normal_()
        k.normal_()
        logits.normal_()
        u.uniform_()
        positions.fill_(3 * i)
        where.copy_(positions)
        lengths.fill_(1200 - 250 * i)
        graphs[i % 2].replay()
        got = [x.clone() for x in outs[i % 2]]
        want = run()  # (what is written is the same)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.float().nan_to_num(7.0), b.float().nan_to_num(7.0))


def test_work_goes_to_the_current_stream():
    q, own, pre = inputs(4, "fp16", 1, 3, 2, 2, 2, 30, 2000, 64)
    logits, u = torch.randn(3, 40000, device=DEV), torch.rand(3, device=DEV)
    want = (P.shared_prefix_attention(q, own, pre), sample_tokens(logits, u, top_p=0.9))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    held = torch.zeros_like(q)
    with torch.cuda.stream(s):
        for _ in range(50):  # the copy comes after work on the same stream
            held.normal_()
        held.copy_(q)
        got = (P.shared_prefix_attention(held, own, pre), sample_tokens(logits, u, top_p=0.9))
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_calls_at_once_have_workspaces_of_their_own():
    a, b = inputs(5, "fp16", 1, 4, 2, 2, 1, 8, 9000, 64), inputs(6, "fp16", 1, 4, 2, 2, 1, 8, 9000, 64)
    want = [P.shared_prefix_attention(*x) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(P.shared_prefix_attention(*x))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_refusals_of_operands():
    q, own, pre = inputs(7, "fp16", 2, 3, 4, 2, 2, 5, 6, 64)
    call = P.shared_prefix_attention
    for bad, words in (
            (lambda: call(q[0], own), "groups, sequences"),
            (lambda: call(q, None), "neither"),
            (lambda: call(q, P.KV(own.k[:, :2], own.v[:, :2])), "own"),
            (lambda: call(q, P.KV(own.k, own.v[..., :3, :])), "own"),
            (lambda: call(q, own, P.KV(pre.k.bfloat16(), pre.v.bfloat16())), "prefix"),
            (lambda: call(q, stored(own), pre), "8-bit"),
            (lambda: call(q, own, pre, positions=torch.zeros(2, 3, device=DEV)), "positions"),
            (lambda: call(q, own, pre, positions=torch.zeros(2, 3, dtype=torch.int32)), "positions"),
            (lambda: call(q, own, pre, prefix_lengths=torch.zeros(3, dtype=torch.int32, device=DEV)), "prefix_lengths"),
            (lambda: call(q, own, pre, scale=-1.0), "scale"),
            (lambda: call(q, own, pre, out=q), "overlap"),
            (lambda: call(q, own, pre, out=torch.empty(1, 3, 4, 2, 64, device=DEV, dtype=q.dtype).expand_as(q)), "overlap"),
            (lambda: call(q, own, pre, out=torch.empty_like(q).bfloat16()), "out"),
            (lambda: call(q[:, :, :3], own, pre), "multiple"),
            (lambda: call(q.clone().requires_grad_(), own, pre), "autograd"),
            (lambda: call(q[..., :60], P.KV(*(x[..., :60] for x in own))), "width"),
            (lambda: call(q.double(), own), "dtype")):
        with pytest.raises(DzError, match=words):
            bad()
    with torch.no_grad():
        call(q.clone().requires_grad_(), own, pre)
    cache = stored(own)
    k = own.k.contiguous()
    for bad, words in (
            (lambda: P.cache_write(cache, k, k, 1), "fit"),
            (lambda: P.cache_write(cache, k[0], k[0], 0), "alike"),
            (lambda: P.cache_write(cache, k, k.bfloat16(), 0), "alike"),
            (lambda: P.cache_write(cache, k, k, torch.zeros(3, dtype=torch.int32, device=DEV)), "positions"),
            (lambda: P.cache_write(P.QuantizedKV(cache.k, cache.k, cache.k_scale, cache.v_scale)._replace(k=cache.k[:1].expand_as(cache.k)), k, k, 0), "leading dimensions"),
            (lambda: P.cache_read(cache, 6, torch.float16), "slots"),
            (lambda: P.cache_read(cache, 2, torch.float16, start=-1), "slots"),
            (lambda: P.cache_read(cache, 2, torch.float64), "dtype")):
        with pytest.raises(DzError, match=words):
            bad()
    x, u = torch.randn(3, 50, device=DEV), torch.rand(3, device=DEV)
    for bad, words in (
            (lambda: sample_tokens(x, u[:2]), "uniform"),
            (lambda: sample_tokens(x, u.double()), "uniform"),
            (lambda: sample_tokens(x, u, top_k=-1), "top_k"),
            (lambda: sample_tokens(x, u, top_p=1.01), "top_p"),
            (lambda: sample_tokens(x, u, temperature=-1.0), "temperature"),
            (lambda: sample_tokens(x, u, top_k=torch.zeros(3, device=DEV)), "top_k"),
            (lambda: sample_tokens(x.t(), u[:1].expand(50)), "contiguous")):
        with pytest.raises(DzError, match=words):
            bad()


def test_a_refused_call_leaves_no_error_behind():
    host = np.zeros(4096, dtype=np.float32)
    q, own, pre = inputs(8, "fp32", 1, 1, 1, 1, 1, 4, 4, 64)
    want = P.shared_prefix_attention(q, own, pre)
    with pytest.raises(DzError, match="not device memory"):
        L.call("dz_sample_tokens", host.ctypes.data, L.DZ_DTYPE_F32, 1, 16, 16, q.data_ptr(), 1.0, 0, 1.0, 0.0, None, None, None, None, q.data_ptr(), stream_handle())
    assert torch.equal(P.shared_prefix_attention(q, own, pre), want)


def test_a_workspace_that_is_too_small_is_refused():
    q, own, pre = inputs(9, "fp16", 1, 1, 1, 1, 1, 4, 4096, 64)
    s = lambda t: tuple(t.stride()[:-1])  # noqa: E731
    pk, pv = ((x.stride(0), 0, *x.stride()[1:3]) for x in pre)
    out = torch.empty_like(q)
    args = P._ATTENTION.pack(q.data_ptr(), out.data_ptr(), *s(q), *s(out), own.k.data_ptr(), own.v.data_ptr(), *s(own.k), *s(own.v), *(0,) * 10, pre.k.data_ptr(),
                             pre.v.data_ptr(), *pk, *pv, *(0,) * 10, 0, 0, 1, 1, 1, 1, 1, 64, 4, 4096, L.DZ_DTYPE_F16, 0.125)
    need = C.c_int64()
    L.call("dz_shared_prefix_attention_workspace", args, C.byref(need))
    assert need.value > 0
    work = torch.empty(need.value, dtype=torch.uint8, device=DEV)
    with pytest.raises(DzError, match="workspace"):
        L.call("dz_shared_prefix_attention", args, work.data_ptr(), need.value - 1, stream_handle())
    with pytest.raises(DzError, match="workspace"):
        L.call("dz_shared_prefix_attention", args, None, need.value, stream_handle())
    L.call("dz_shared_prefix_attention", args, work.data_ptr(), need.value, stream_handle())
    assert torch.equal(out, P.shared_prefix_attention(q, own, pre))


def test_offsets_past_32_bits():
    # 2^24 slots of 256 bytes: all keys are 0 but the last but one, which the query meets
    slots = 1 << 24
    k, v = (torch.zeros(1, 1, 1, slots, 128, dtype=torch.float16, device=DEV) for _ in range(2))
    q = torch.ones(1, 1, 1, 1, 128, dtype=torch.float16, device=DEV)
    k[..., slots - 2, :] = 4.0
    v[..., slots - 2, :] = torch.arange(128, device=DEV).half()
    v[..., slots - 1, :] = 1000.0
    positions = torch.tensor([[slots - 2]], dtype=torch.int32, device=DEV)
    got = P.shared_prefix_attention(q, P.KV(k, v), positions=positions)[0, 0, 0, 0].cpu().double()
    # scores of 512 / sqrt(128) = 45.25 and of 0: what the others weigh together is 2^24 exp(-45.25) = 4e-13
    assert torch.equal(got, torch.arange(128, dtype=torch.float64))
    got = P.shared_prefix_attention(q, None, P.KV(k[0], v[0]), prefix_lengths=torch.tensor([slots - 1], dtype=torch.int32, device=DEV))
    assert torch.equal(got[0, 0, 0, 0].cpu().double(), torch.arange(128, dtype=torch.float64))
    del k, v
    cache = P.QuantizedKV.empty(2, 1, slots, 128, device=DEV)
    x = torch.randn(2, 1, 3, 128, device=DEV).half()
    P.cache_write(cache, x, x, slots - 3)
    small = P.QuantizedKV.empty(2, 1, 3, 128, device=DEV)
    P.cache_write(small, x, x, 0)
    assert torch.equal(P.cache_read(cache, 3, torch.float16, start=slots - 3).v, P.cache_read(small, 3, torch.float16).v)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shape", [
    (1, 3, 2, 2, 3, 40, 9, 64),      # a tile of rows of three sequences
    (1, 2, 2, 1, 70, 90, 65, 80),    # tiles of 128 rows of one
    (1, 40, 1, 1, 1, 3, 0, 16),      # 32 sequences in a tile
    (1, 3, 2, 1, 2, 30, 1500, 104),  # a prompt in several parts
    (1, 2, 600, 600, 2, 6, 20, 16),  # two waves an item
    (1, 2, 1100, 1100, 2, 6, 20, 80),  # one
], ids=str)
def test_what_is_not_finite_reaches_those_that_see_it(shape, dtype, bits):
    q, own, pre = inputs(10, dtype, *shape, bits=bits)
    sequences, length, slots = shape[1], shape[4], shape[5]
    positions = torch.full((1, sequences), slots - length, dtype=torch.int32, device=DEV)
    want = P.shared_prefix_attention(q, own, pre, positions=positions)
    heads = shape[2] // shape[3]  # the query heads of key head 0
    see = (0, -1, slice(0, heads), -1)  # those see the last sequence's last key

    def attend(x, column, store):
        """With one slot's keys or values set: the results, where those that see it are taken from `want` once looked at."""
        held = store[0, -1, 0, slots - 1].clone()
        to = store[0, -1, 0, slots - 1]
        (to.view(torch.uint8) if bits == 8 else to)[column] = x
        got = P.shared_prefix_attention(q, own, pre, positions=positions)
        to.view(torch.uint8).copy_(held.view(torch.uint8))
        seen = got[see][..., column].clone()
        got[see][..., column] = want[see][..., column]
        check(dtype, q, own, pre, positions, got=got)
        return seen

    assert torch.isnan(attend(0x7F if bits == 8 else math.nan, 3, own.v)).all()
    if bits == 16:
        assert (attend(-math.inf, 5, own.v) == -math.inf).all()
        every = slice(None)
        assert torch.isnan(attend(math.nan, every, own.v)).all()
        assert torch.isnan(attend(math.inf, every, own.k)).all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("shape", [
    (1, 3, 40, 1, 1, 20, 70, 64),   # 40 rows of one token
    (2, 2, 160, 1, 1, 9, 33, 80),   # 160: two tiles
    (1, 2, 36, 1, 5, 7, 600, 128),  # tiles that end inside of a token's heads
], ids=str)
def test_many_query_heads_of_one_key_head(shape, bits):
    q, own, pre = inputs(12, "bf16", *shape, bits=bits)
    check("bf16", q, own, pre)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 3, 2, 1, 2, 30, 0, 72), (1, 2, 2, 2, 40, 60, 0, 64), (1, 3, 2, 1, 2, 30, 1500, 104)], ids=str)
def test_scores_of_minus_infinity(shape, dtype):
    q, own, pre = inputs(13, dtype, *shape)
    q = q.abs() + 0.125
    prefix = shape[6]

    def is_value(got, v):
        """Where one key is left, with a score s: its weight is w = 2^x, x what is lost as s log2(e) scale is rounded, and the answer
        (w v) (1 / w) with three roundings in fp32, of 2^-24 each. Rounded to 16 bits that is v; w is 1 in 16 bits."""
        v = v.unsqueeze(1).repeat_interleave(shape[2] // shape[3], 0).expand_as(got)
        return ((got - v).abs() <= (4 * 2.0**-24 if dtype == "fp32" else 0) * v.abs()).all()

    want = P.shared_prefix_attention(q, own, pre)
    held = own.k[0, 0].clone()
    own.k[0, 0] = -math.inf
    if prefix:
        pre.k[0] = -math.inf
        assert torch.isnan(P.shared_prefix_attention(q, own, pre)[0, 0]).all()  # 0 / 0
        pre.k[0, :, 700] = 0.0
        got = P.shared_prefix_attention(q, own, pre)
        assert is_value(got[0, 0], pre.v[0, :, 700])
        return
    got = P.shared_prefix_attention(q, own, None)
    assert torch.isnan(got[0, 0]).all()
    assert torch.equal(got[0, 1:], want[0, 1:])
    own.k[0, 0, :, 3] = held[:, 3]
    got = P.shared_prefix_attention(q, own, None)
    assert is_value(got[0, 0], own.v[0, 0, :, 3])


def test_numbers_of_other_types():
    cache = P.QuantizedKV.empty(2, 1, 8, 16, device=DEV)
    x = torch.randn(2, 1, 1, 16, device=DEV)
    P.cache_write(cache, x, x, np.int64(3))
    assert torch.equal(P.cache_read(cache, np.int32(1), torch.float32, start=np.int64(3)).k, P.cache_read(cache, 1, torch.float32, start=3).k)
    logits, u = torch.randn(2, 50, device=DEV), torch.rand(2, device=DEV)
    assert torch.equal(sample_tokens(logits, u, top_k=np.int64(4), temperature=np.float32(0.5)), sample_tokens(logits, u, top_k=4, temperature=0.5))
    for call in (lambda: P.cache_write(cache, x, x, 1.5), lambda: P.cache_read(cache, 1.0, torch.float32), lambda: P.cache_read(cache, 1, torch.float32, start=None),
                 lambda: sample_tokens(logits, u, top_k=2.5), lambda: sample_tokens(logits, u, temperature="one"), lambda: sample_tokens(logits, u, top_p=None)):
        with pytest.raises(DzError, match="must be"):
            call()


@pytest.mark.parametrize("shape", [(1, 2, 2, 1, 3, 40, 300, 128), (1, 1, 4, 2, 80, 100, 70, 112), (2, 20, 16, 16, 2, 9, 33, 64)], ids=str)
def test_codes_whose_rows_start_at_multiples_of_8_bytes(shape):
    q, own, pre = inputs(14, "bf16", *shape, bits=8)
    width = shape[-1]

    def moved(x):
        """The same codes 8 bytes into rows of 16 more."""
        to = torch.zeros(*x.shape[:-1], width + 16, dtype=torch.uint8, device=DEV)
        to[..., 8:8 + width] = x.view(torch.uint8)
        return to.view(P.CODES)[..., 8:8 + width]

    own8, pre8 = (P.QuantizedKV(moved(s.k), moved(s.v), s.k_scale, s.v_scale) for s in (own, pre))
    assert own8.k.data_ptr() % 16 == 8
    check("bf16", q, own8, pre8)
    check("bf16", q, own8, pre)
