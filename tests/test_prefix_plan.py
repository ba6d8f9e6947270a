"""The split of the shared-prefix attention, restated: every token of every
unit is in exactly one piece, the pieces' partials are disjoint and inside the
workspace, and the combine looks for them where they were left."""

import random

import numpy as np
import pytest


def up(a, b):
    return -(-a // b)


def tile_rows(rows, kind):
    return 16 if kind == "general" or rows <= 16 else 64 if kind == "float" or rows <= 64 else 128


class Plan:
    START, MIN_SEGMENT = 768, 256

    @staticmethod
    def cost(rows, kind):
        if kind == "general" or rows <= 16:
            return 4
        return 10 if kind == "float" else 4 if rows <= 64 else 6

    def unit(self, e):
        return self.START + self.n[e] * self.cost(self.rows[e], self.kind) if self.n[e] else 0

    def __init__(self, offsets, plens, lens, gq, hkv, segs, kind):
        b, self.kind = len(lens), kind
        first = np.maximum.accumulate(np.clip(offsets, 0, b))
        self.first = [int(x) for x in first]
        self.groups = len(plens)
        self.rows = [(self.first[g + 1] - self.first[g]) * gq for g in range(self.groups)]
        self.rows += [gq] * b
        self.n = [int(x) for x in plens] + [int(x) for x in lens]
        self.gq, self.hkv = gq, hkv
        self.start, self.gran = [0], [0]
        for e, rows in enumerate(self.rows):
            self.start.append(self.start[-1] +
                              self.unit(e) * hkv * up(rows, tile_rows(rows, kind)))
            self.gran.append(self.gran[-1] + hkv * up(rows, 16))
        self.total = self.start[-1]
        self.seg = max(self.MIN_SEGMENT, up(self.total, segs))
        # as the host sizes the workspace
        self.granules = 8 * segs + hkv * (b * gq // 16 + min(self.groups, b)) + b * hkv * up(gq, 16)

    def pieces(self, s):
        """Segment s: (entry, kv, tile, t0, n, first partial row, rows)."""
        pos, end = s * self.seg, min((s + 1) * self.seg, self.total)
        while pos < end:
            e = int(np.searchsorted(self.start, pos, side="right")) - 1
            off, whole = pos - self.start[e], self.unit(e)
            tr, w = tile_rows(self.rows[e], self.kind), self.cost(self.rows[e], self.kind)
            tiles = up(self.rows[e], tr)
            unit, inside = off // whole, off % whole
            kv, tile = unit // tiles, unit % tiles
            stop = min(whole, end - pos + inside)
            t0, t1 = (up(max(c - self.START, 0), w) for c in (inside, stop))
            m = t1 - t0
            pos += stop - inside
            if m == 0:
                continue
            gran = 8 * s + self.gran[e] + kv * up(self.rows[e], 16) + tile * (tr // 16)
            yield e, kv, tile, t0, m, 16 * gran, min(tr, self.rows[e] - tile * tr)

    def looked_for(self, e, b, kv, j):
        """The partial rows of (b, head kv * gq + j) in entry e."""
        if self.n[e] == 0:
            return []
        first = self.first[e] if e < self.groups else e - self.groups
        r = (b - first) * self.gq + j
        tr = tile_rows(self.rows[e], self.kind)
        tiles, tile = up(self.rows[e], tr), r // tr
        lo = self.start[e] + self.START + (kv * tiles + tile) * self.unit(e)
        s0 = lo // self.seg
        s1 = (lo + self.cost(self.rows[e], self.kind) * (self.n[e] - 1)) // self.seg
        gran = 8 * s0 + self.gran[e] + kv * up(self.rows[e], 16) + tile * (tr // 16)
        return [16 * gran + r - tile * tr + 128 * i for i in range(s1 - s0 + 1)]


@pytest.mark.parametrize("kind", ["half", "float", "general"])
@pytest.mark.parametrize("seed", range(40))
def test_pieces_and_partials(seed, kind):
    r = random.Random(seed)
    b, groups = r.randint(1, 40), r.choice([0, 1, 2, 7])
    gq, hkv, segs = r.choice([1, 3, 4, 8, 16, 33, 64]), r.choice([1, 2, 8]), r.choice([1, 16, 512])
    if seed % 4 == 3:   # any values, falling ones too
        offsets = [r.randint(-5, b + 5) for _ in range(groups + 1)]
    else:
        offsets = sorted(r.randint(0, b) for _ in range(groups + 1))
    plens = [r.choice([0, 1, 63, 64, 1000, 5000]) for _ in range(groups)]
    lens = [r.choice([0, 0, 1, 64, 129, 700]) for _ in range(b)]
    p = Plan(offsets if groups else [0], plens, lens, gq, hkv, segs, kind)
    assert p.seg * segs >= p.total

    seen, left = {}, {}
    taken = np.zeros(16 * p.granules, bool)
    for s in range(segs):
        for e, kv, tile, t0, n, row, rows in p.pieces(s):
            seen.setdefault((e, kv, tile), []).append((t0, n))
            assert 0 < rows and row + rows <= len(taken)   # inside the workspace
            assert not taken[row:row + rows].any()
            taken[row:row + rows] = True
            for i in range(rows):
                left.setdefault((e, kv, tile * tile_rows(p.rows[e], kind) + i), []).append(row + i)
    for e, (rows, n) in enumerate(zip(p.rows, p.n)):
        for kv in range(hkv):
            for tile in range(up(rows, tile_rows(rows, kind))):
                at = 0
                for t0, m in seen.get((e, kv, tile), []):   # in order, without a gap
                    assert t0 == at
                    at += m
                assert at == n
    for x in range(b):
        for e in [g for g in range(p.groups) if p.first[g] <= x < p.first[g + 1]] + [p.groups + x]:
            first = p.first[e] if e < p.groups else x
            for kv in range(hkv):
                for j in range(gq):
                    assert p.looked_for(e, x, kv, j) == left.get((e, kv, (x - first) * gq + j), [])
