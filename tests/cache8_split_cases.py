"""Calls of attention_decode_paged_int8 that reach its splits of many tokens:
equal segments over all rows, and segments of 128 tokens of one row."""

import dataclasses
import random


def ragged(seed, rows=40, long=20011):
    """Rows of 0, 1 and a few tokens, of multiples of a segment and one more or
    less, of thousands, one much longer than the others; none at the start, in
    a run in the middle and at the end."""
    r = random.Random(seed)
    some = [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 192, 256, 257, 384, 960, 1024, 4096]
    lens = [r.choice(some) if r.random() < 0.5 else r.randint(1, 3000) for _ in range(rows)]
    lens[0] = lens[1] = lens[-1] = 0
    lens[10:14] = [0] * 4
    lens[rows // 2] = long
    return lens


def short(seed, rows, hi):
    r = random.Random(seed)
    return [r.randint(0, hi) for _ in range(rows)]


@dataclasses.dataclass
class Case:
    d: int
    hkv: int
    group: int
    page: int
    lens: list
    few: int                 # of the first launch
    dtypes: str = "bf16"     # names, in one string
    several: bool = False    # a segment of several rows, whole rows inside
    at_end: bool = False     # rows that end with a segment
    many: bool = False       # four heads a workgroup in the combine, some of > 32 pieces
    holes: bool = False      # table entries outside the pool
    whole: bool = False      # lens not given: every row of the table

    @property
    def width(self):
        return max(1, -(-max(self.lens) // self.page))


CASES = {
    "ragged_128": Case(128, 8, 4, 16, ragged(1), 0, "bf16 f16 f32", True, many=True),
    "ragged_64": Case(64, 8, 4, 24, ragged(2), 0, "bf16 f16 f32", True, many=True),
    "ragged_256": Case(256, 4, 8, 32, ragged(3), 0, "bf16 f32", True, many=True),
    "ragged_96": Case(96, 8, 5, 5, ragged(4), 0, "bf16 f16 f32", True),
    "ragged_192": Case(192, 4, 3, 16, ragged(5), 0, "f16 f32", True),
    "ragged_16": Case(16, 8, 2, 16, ragged(6), 0, "f32", True),
    "ragged_48": Case(48, 8, 1, 64, ragged(7), 0, "f16", True),
    "holes_128": Case(128, 8, 4, 16, ragged(8), 0, "bf16 f32", True, holes=True),
    "holes_64": Case(64, 8, 5, 7, ragged(9), 0, "f16", True, holes=True),
    "holes_240": Case(240, 4, 2, 16, ragged(10), 0, "f32", True, holes=True),
    # several tiles of q heads a kv head
    "tiles_128": Case(128, 4, 20, 64, ragged(11), 0, "f16 f32", True, many=True),
    "tiles_64": Case(64, 3, 33, 16, ragged(12), 0, "bf16", True),
    "tiles_80": Case(80, 4, 17, 16, ragged(13), 0, "f32", True),
    # many short rows: several whole ones in each segment
    "short_64": Case(64, 8, 2, 16, short(14, 700, 200), 0, "bf16 f32", True),
    "short_128": Case(128, 8, 1, 16, short(15, 700, 150), 0, "f16 f32", True),
    "short_112": Case(112, 8, 2, 5, short(16, 700, 150), 0, "f32", True),
    # every row a whole number of segments (16 x 8 rows of 15 x 192 tokens)
    "ends_64": Case(64, 8, 2, 16, [2880] * 16, 0, "f32", at_end=True),
    "ends_128": Case(128, 8, 2, 16, [2880] * 16, 0, "bf16 f32", at_end=True),
    # more sequences than a launch has
    "launches_64": Case(64, 4, 2, 16, short(17, 1400, 200), 0, "f32", True),
    "launches_96": Case(96, 4, 2, 16, short(18, 1100, 200), 0, "bf16", True),
    "whole_128": Case(128, 8, 4, 24, [1536] * 32, 0, "bf16", whole=True),
    # segments of 128 tokens of one row
    "few2_64": Case(64, 3, 15, 16, ragged(19), 2, "bf16 f32", many=True),
    "few2_128": Case(128, 2, 16, 24, ragged(20), 2, "f16 f32", many=True),
    "few2_96": Case(96, 2, 4, 16, ragged(21), 2, "f32", holes=True),
    "few2_256": Case(256, 2, 5, 16, ragged(22, 20), 2, "bf16 f32"),
}


def check_reached(c, launches):
    """The case runs what it is there for."""
    a = launches[0]
    assert a.few == c.few
    assert max(a.in_seg.values()) > 1 if c.few == 0 and not c.at_end else True
    if c.several:
        assert a.inside > 0 and a.both > 0 and max(a.in_seg.values()) >= 3
    if c.at_end:
        assert a.at_end > 100
    if c.many:
        heads = len(c.lens) * c.hkv * c.group
        assert heads >= 1024 and 256 % c.d == 0
        assert max(a.pieces) > 32 and any(2 <= n <= 32 for n in a.pieces)
    assert len(launches) == -(-len(c.lens) // 1024)
