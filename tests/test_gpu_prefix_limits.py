"""dizo_amd.prefix_attention on the GPU at the ends of its types."""
import math

import pytest
import torch

from dizo_amd import prefix_attention as P
from oracle import prefix as O
from test_gpu_prefix_attention import bound, check, inputs, stored, values

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
