"""dizo_amd.sampling on the GPU: parameters of one row that are out of range, next to rows whose are not."""
import math

import pytest
import torch

from dizo_amd.sampling import sample_tokens
from oracle import prefix as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TINY = 2.0**-149
GOOD = {"temperature": [0.5, 0.0, 1.0, 2.0**-63], "top_k": [0, 3, 2**31 - 1, 700], "top_p": [0.5, 0.0, 1.0, TINY], "min_p": [0.1, 0.0, 1.0, TINY]}
BAD = {"temperature": [-1.0, -TINY, 2.0**-64, 2.0**64, math.inf, math.nan], "top_k": [-1, -(2**31)],
       "top_p": [-0.5, -TINY, 1.0 + 2.0**-23, math.inf, -math.inf, math.nan], "min_p": [-0.5, -TINY, 1.0 + 2.0**-23, math.inf, -math.inf, math.nan]}


@pytest.mark.parametrize("others", [{}, dict(temperature=0.0), dict(top_k=40, top_p=0.9), dict(top_p=0.8, min_p=0.02)], ids=str)
@pytest.mark.parametrize("name", sorted(BAD))
@pytest.mark.parametrize("vocab", [5, 3001])
def test_rows_whose_parameters_are_out_of_range_give_no_token(vocab, name, others):
    values = [v for pair in zip(GOOD[name] * 2, BAD[name] + GOOD[name]) for v in pair]
    n = len(values)
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x, u = torch.randn(n, vocab, generator=g, device=DEV) * 3, torch.rand(n, generator=g, device=DEV)
    others = {k: v for k, v in others.items() if k != name}
    kind = torch.int32 if name == "top_k" else torch.float32
    of_row = torch.tensor(values, dtype=kind, device=DEV)
    got = sample_tokens(x, u, **{name: of_row}, **others)
    for i, v in enumerate(values):
        if v in GOOD[name]:
            assert got[i] == O.sample(x[i], float(u[i]), **{name: of_row[i].item()}, **others)
        else:
            assert got[i] == -1
