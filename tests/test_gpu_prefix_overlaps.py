"""dizo_amd.prefix_attention and sampling on the GPU: stores that lie in one another, and calls whose outputs lie in their inputs."""
import pytest
import torch

from dizo_amd import _lib as L
from dizo_amd import prefix_attention as P
from dizo_amd._lib import DzError
from dizo_amd.table import stream_handle

pytestmark = pytest.mark.gpu
DEV = "cuda"
B, H, S, W = 3, 2, 5, 16


def room(n):
    return torch.full((n,), 0x55, dtype=torch.uint8, device=DEV)


def store(buffer, k, v, ks, vs):
    """A store in a buffer: (offset, strides) of each part."""
    def part(at, kind, shape):
        return buffer.as_strided(shape, at[1], at[0]).view(kind)
    return P.QuantizedKV(part(k, P.CODES, (B, H, S, W)), part(v, P.CODES, (B, H, S, W)), part(ks, P.SCALES, (B, H, S)), part(vs, P.SCALES, (B, H, S)))


N = B * H * S * W
ROW = 2 * W + 8  # [keys | values | scales] of a token's head
BLOCK = 2 * H * S * W + 2 * H * S + 4  # a sequence's keys, values and scales
LAYOUTS = {
    "one after another": ((0, (H * S * W, S * W, W, 1)), (N, (H * S * W, S * W, W, 1)), (2 * N, (H * S, S, 1)), (2 * N + 50, (H * S, S, 1))),
    "rows in turn": ((0, (H * S * ROW, S * ROW, ROW, 1)), (W, (H * S * ROW, S * ROW, ROW, 1)), (2 * W, (H * S * ROW, S * ROW, ROW)),
                     (2 * W + 1, (H * S * ROW, S * ROW, ROW))),
    "values first": ((W, (H * S * ROW, S * ROW, ROW, 1)), (0, (H * S * ROW, S * ROW, ROW, 1)), (2 * W + 7, (H * S * ROW, S * ROW, ROW)),
                     (2 * W, (H * S * ROW, S * ROW, ROW))),
    "a block a sequence": ((0, (BLOCK, S * W, W, 1)), (H * S * W, (BLOCK, W, H * W, 1)), (2 * H * S * W, (BLOCK, S, 1)), (2 * H * S * W + H * S, (BLOCK, 1, H))),
    "heads in turn": ((0, (2 * H * S * W, 2 * S * W, W, 1)), (S * W, (2 * H * S * W, 2 * S * W, W, 1)), (2 * N, (2 * H * S, 2 * S, 1)), (2 * N + S, (2 * H * S, 2 * S, 1))),
}


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
def test_stores_whose_parts_lie_among_each_other(layout):
    cache = store(room(4 * N), *LAYOUTS[layout])
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(B, H, S, W, generator=g, device=DEV) for _ in range(2))
    P.cache_write(cache, k, v, 0)
    want = P.QuantizedKV.empty(B, H, S, W, device=DEV)
    P.cache_write(want, k, v, 0)
    for x, y in zip(cache, want):
        assert torch.equal(x.contiguous().view(torch.uint8), y.view(torch.uint8))


FLAT = (H * S * W, S * W, W, 1)


@pytest.mark.parametrize("k, v, ks, vs", [
    ((0, FLAT), (0, FLAT), (2 * N, (H * S, S, 1)), (2 * N + 50, (H * S, S, 1))),              # keys and values are one
    ((0, FLAT), (W, FLAT), (2 * N, (H * S, S, 1)), (2 * N + 50, (H * S, S, 1))),              # a slot apart
    ((0, FLAT), (N - 8, FLAT), (2 * N, (H * S, S, 1)), (2 * N + 50, (H * S, S, 1))),          # half a row
    ((0, FLAT), (N, FLAT), (2 * N, (H * S, S, 1)), (2 * N, (H * S, S, 1))),                   # one scale for both
    ((0, FLAT), (N, FLAT), (2 * N, (H * S, S, 1)), (2 * N - 1, (H * S, S, 1))),               # a scale in the values
    ((0, (H * S * ROW, S * ROW, ROW, 1)), (W - 8, (H * S * ROW, S * ROW, ROW, 1)), (2 * W, (H * S * ROW, S * ROW, ROW)), (2 * W + 1, (H * S * ROW, S * ROW, ROW))),
    ((0, FLAT), (8, (H * S * W, S * W, W, 1)), (2 * N, (H * S, S, 1)), (2 * N + 50, (H * S, S, 1))),
])
def test_stores_whose_parts_overlap_are_refused(k, v, ks, vs):
    buffer = room(4 * N)
    cache = store(buffer, k, v, ks, vs)
    x = torch.randn(B, H, S, W, device=DEV)
    with pytest.raises(DzError, match="overlap"):
        P.cache_write(cache, x, x, 0)
    assert (buffer == 0x55).all()
    P.cache_read(cache, S, torch.float32)  # reads may


def test_positions_in_a_store_are_refused():
    cache = P.QuantizedKV.empty(B, H, S, W, device=DEV)
    x = torch.randn(B, H, 1, W, device=DEV)
    with pytest.raises(DzError, match="positions"):
        P.cache_write(cache, x, x, cache.k.view(torch.uint8).view(-1)[:4 * B].view(torch.int32))


def test_outputs_in_inputs_are_refused():
    q = torch.zeros(1, 2, 1, 1, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(1, 2, 1, 4, 64, dtype=torch.bfloat16, device=DEV)
    out = torch.zeros_like(q)
    ints = out.view(-1)[:4].view(torch.int32)
    with pytest.raises(DzError, match="out overlaps positions"):
        P.shared_prefix_attention(q, P.KV(k, k), positions=ints.view(1, 2), out=out)
    with pytest.raises(DzError, match="out overlaps prefix_lengths"):
        P.shared_prefix_attention(q, None, P.KV(k[:, 0], k[:, 0]), prefix_lengths=ints[:1], out=out)
    x = torch.zeros(4, 16, device=DEV)
    u = torch.zeros(16, device=DEV)
    for logits, uniform, ts, tokens in ((x, u, None, x), (x, u, None, u), (x, u, u[4:], u[6:])):
        with pytest.raises(DzError, match="tokens overlap"):
            L.call("dz_sample_tokens", logits.data_ptr(), L.DZ_DTYPE_F32, 4, 16, 16, uniform.data_ptr(), 1.0, 0, 1.0, 0.0, None if ts is None else ts.data_ptr(),
                   None, None, None, tokens.data_ptr(), stream_handle())
