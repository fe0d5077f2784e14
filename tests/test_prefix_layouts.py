"""dizo_amd.prefix_attention without a GPU: a cache's leading dimensions as one, by their strides."""
import itertools

import pytest
import torch

from dizo_amd import prefix_attention as P
from dizo_amd._lib import DzError

# shape and strides of the leading dimensions, in rows of the rest
LEADS = [
    ((2, 1, 3), (5, 5, 1)),     # a slice of the last of (2, 1, 5)
    ((2, 1, 3), (2, 6, 1)),     # the outer one inside
    ((2, 1, 3), (1, 1, 2)),     # (3, 2, 1) permuted
    ((2, 1, 3), (3, 3, 1)),
    ((2, 1, 3), (3, 99, 1)),    # a stride that nothing steps by
    ((1, 2, 1, 3, 1), (7, 3, 2, 1, 50)),
    ((1, 2, 1, 3, 1), (7, 4, 2, 1, 50)),
    ((2, 2, 2), (8, 2, 1)),
    ((2, 2, 2), (8, 4, 2)),
    ((2, 2, 2), (4, 2, 1)),
    ((3, 1), (0, 1)),           # the same rows for all
    ((3, 2), (0, 1)),
    ((3, 2), (1, 0)),
    ((3, 2), (0, 0)),
    ((1, 1), (4, 9)),
    ((4, 1), (7, 1)),
    ((1, 4), (3, 7)),
]


def starts(lead, strides, unit):
    return [sum(i * s * unit for i, s in zip(at, strides)) for at in itertools.product(*map(range, lead))]


@pytest.mark.parametrize("lead, strides", LEADS, ids=str)
@pytest.mark.parametrize("rest", [(2, 4, 8), (2, 4)], ids=["codes", "scales"])
def test_leading_dimensions_are_one_where_their_strides_are(lead, strides, rest):
    unit = 64
    room = torch.empty(unit * 200, dtype=torch.uint8)
    inner = (32, 8, 1) if len(rest) == 3 else (4, 1)
    t = room.as_strided((*lead, *rest), (*(s * unit for s in strides), *inner))
    want = starts(lead, strides, unit)
    steps = {b - a for a, b in zip(want, want[1:])}
    if len(steps) <= 1:  # the sequences are as far from each other throughout
        batch, _, head, slot = P._one_lead("test", t, len(lead))
        assert [i * batch for i in range(len(want))] == want and (head, slot) == t.stride()[len(lead):len(lead) + 2]
    else:
        with pytest.raises(DzError, match="leading dimensions"):
            P._one_lead("test", t, len(lead))


def test_the_layouts_above_are_of_both_kinds():
    ways = [len({b - a for a, b in zip(w, w[1:])}) <= 1 for w in (starts(lead, s, 1) for lead, s in LEADS)]
    assert 5 <= sum(ways) <= len(ways) - 5
