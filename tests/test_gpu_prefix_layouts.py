"""dizo_amd.prefix_attention on the GPU: caches whose leading dimensions lie apart."""
import pytest
import torch

from dizo_amd import prefix_attention as P

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("lead, take", [
    ((2, 1, 5), lambda x: x[:1, :, :3]),    # (1, 1, 3) of more
    ((2, 1, 3), lambda x: x),
    ((3, 1, 2), lambda x: x[:, :, :1].permute(1, 2, 0, *range(3, x.dim()))),  # every second sequence
    ((4, 5), lambda x: x[:, 1:2]),          # (4, 1), five sequences apart
], ids=["slice", "whole", "permuted", "column"])
def test_a_view_of_a_cache_is_written_and_read_in_its_place(lead, take):
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    cache = P.QuantizedKV.empty(*lead, 2, 6, 16, device=DEV)
    for x in cache:
        x.view(torch.uint8).fill_(0x55)
    part = P.QuantizedKV(*map(take, cache))
    shape = part.k.shape
    k, v = (torch.randn(*shape[:-2], 4, 16, generator=g, device=DEV) for _ in range(2))
    P.cache_write(part, k, v, 1)
    want = P.QuantizedKV.empty(*shape, device=DEV)
    for x in want:
        x.view(torch.uint8).fill_(0x55)
    P.cache_write(want, k, v, 1)
    whole = P.QuantizedKV(*(torch.full(x.shape, 0x55, dtype=torch.uint8, device=DEV) for x in cache))
    for x, y in zip(whole, want):
        take(x).copy_(y.view(torch.uint8))
    assert all(torch.equal(x.view(torch.uint8), y) for x, y in zip(cache, whole))
    for x, y in zip(P.cache_read(part, 4, torch.float32, start=1), P.cache_read(want, 4, torch.float32, start=1)):
        assert torch.equal(x, y)
