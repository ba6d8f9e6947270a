"""Which split of the rows attention_decode_paged_int8 takes for a call, worked
out from its sizes and lengths: the tests that are about one split ask here
whether they reach it. All integers, but for the segment length's float32
quotient."""

import dataclasses

import numpy as np

LEAST = 64          # tokens of a segment, at least
LAUNCH = 1024       # sequences of a launch


@dataclasses.dataclass
class Launch:
    few: int            # segments of `few * 64` tokens of one row; 0: equal ones
    seg: int            # tokens of a segment
    nseg: int
    rows: list          # (sequence, row of it, first segment, segments), rows with a token
    in_seg: dict        # segment -> rows with a token in it
    inside: int         # whole rows in a segment that another row is in too
    at_end: int         # rows that end with a segment, not the last
    both: int           # segments with partials of two rows

    @property
    def pieces(self):
        return [n for *_, n in self.rows]


def tiles_of(group):
    tiles = -(-group // 16)
    tile = -(-group // tiles)
    return -(-group // tile)


def split(lens, hkv, group, page, width, d, cus):
    """One Launch for each 1024 sequences, for D a multiple of 16 up to 256."""
    assert d % 16 == 0 and d <= 256
    span, vrows = page * width, hkv * tiles_of(group)
    lens = np.clip(np.asarray(lens, np.int64), 0, span)
    most = min(len(lens), LAUNCH) * vrows * (-(-span // LEAST))
    nseg = min(4 * cus * (1 if d > 128 else 2), most, 4096)
    short = min(nseg, (8 if d <= 64 else 4) * cus)
    step = 64 if d <= 64 else 32
    out = []
    for b0 in range(0, len(lens), LAUNCH):
        n = lens[b0:b0 + LAUNCH]
        padded = [int((-(-n // to) * to).sum()) * vrows for to in (LEAST, 2 * LEAST)]
        few = 1 if padded[0] <= short * LEAST else 2 if padded[1] <= nseg * 2 * LEAST else 0
        to = max(1, few * LEAST)
        flat = -(-n // to) * to
        total = int(flat.sum()) * vrows
        seg = few * LEAST
        if not few:
            inv = np.float32(np.float32(1 + 2.0 ** -21) / np.float32(nseg))
            seg = max(int(np.float32(total) * inv) + 1, LEAST)
            seg = -(-seg // step) * step
        rows, in_seg, inside, at_end, both = [], {}, 0, 0, {}
        at = 0
        for b, m in enumerate(flat.tolist()):
            for v in range(vrows if m else 0):
                lo, hi = at // seg, (at + m - 1) // seg
                rows.append((b0 + b, v, lo, hi - lo + 1))
                for s in range(lo, hi + 1):
                    in_seg[s] = in_seg.get(s, 0) + 1
                    if lo != hi:
                        both[s] = both.get(s, 0) + 1
                at += m
                at_end += at % seg == 0 and at < total
        inside = sum(n == 1 and in_seg[lo] > 1 for _, _, lo, n in rows)
        assert at == total <= seg * nseg
        out.append(Launch(few, seg, nseg, rows, in_seg, inside, at_end,
                          sum(x == 2 for x in both.values())))
    return out
