"""The host's model of the attention's split of rows, on the CPU: its own
numbers, and that the lengths the GPU tests of each split use do reach it."""

import pytest

from tests import cache8_split as sp
from tests import cache8_split_cases as cases

CUS = 256


def test_split_by_hand():
    # two rows of 3 segments of 64 at one tile: 100 -> 128, 0, 5 -> 64 tokens
    (a,) = sp.split([100, 0, 5], 2, 4, 16, 8, 128, CUS)
    assert (a.few, a.seg) == (1, 64)
    assert a.rows == [(0, 0, 0, 2), (0, 1, 2, 2), (2, 0, 4, 1), (2, 1, 5, 1)]
    assert a.inside == 0 and a.both == 0 and set(a.in_seg.values()) == {1}
    # equal segments: 300 rows of 1000 tokens over 2048, 147 + 1 -> 160 tokens
    (a,) = sp.split([1000] * 300, 1, 4, 16, 63, 128, CUS)
    assert (a.few, a.seg, a.nseg) == (0, 160, 2048)
    assert a.rows[1] == (1, 0, 6, 7) and a.in_seg[6] == 2
    # 17 q heads a kv head: two rows
    assert sp.tiles_of(16) == 1 and sp.tiles_of(17) == 2 and sp.tiles_of(33) == 3


@pytest.mark.parametrize("name", cases.CASES)
def test_cases_reach_their_split(name):
    c = cases.CASES[name]
    cases.check_reached(c, sp.split(c.lens, c.hkv, c.group, c.page, c.width, c.d, CUS))
