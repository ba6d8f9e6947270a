"""GPU tests of attention_decode_paged_prefix against a plain form in 64 bits
(step_refs.attend_prefix).

The bound. Half a step of the output's type, relative to the value. The
weights' error goes into sums of |v| of their mass (A = sum w |v|, both in the
numerator and, at most as much, in the denominator): a score is a sum of D
products in float32 (its sizes are S = sum |q k| / sqrt(D)): the sum of D terms
in any order of the kernels is at most D/16 + 16 sequential adds: (D / 16 + 20)
2^-24 S, the factor log2(e) / sqrt(D) and the exponent's fused product 2 * 2^-24
S more; the exponential 2^-22; sums over tokens and pieces, n / 16 + 200
sequential adds at most, 2^-24 each of what they hold; weights in two parts
2^-17 (bf16) or 2^-22 (fp16), none for float32. All of it twice."""

import numpy as np
import pytest
import torch

import fusedtok_amd as ft
from tests import step_refs as refs

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def dev(x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x)).to(DEV, dtype=dtype)


def i32(x):
    return dev(np.asarray(x, np.int32))


def np64(t):
    return t.double().cpu().numpy()


class Case:
    def __init__(self, seed, hq, hkv, d, page, plens, sizes, lens, dtype, scale=1.0, spare=2):
        rng = np.random.default_rng(seed)
        b = len(lens)
        self.plens, self.lens = list(plens), list(lens)
        self.offsets = [0] + list(np.cumsum(sizes))
        needs = [-(-n // page) for n in self.plens + self.lens]
        nb = sum(needs) + spare
        ids = rng.permutation(nb)
        g = len(plens)
        self.ptable = np.zeros((g, max(needs[:g], default=0) + 1), np.int32)
        self.table = np.zeros((b, max(needs[g:], default=0) + 1), np.int32)
        at = 0
        for i, n in enumerate(needs):
            row = self.ptable[i] if i < g else self.table[i - g]
            row[:n] = ids[at:at + n]
            at += n
        self.q = dev(rng.standard_normal((b, hq, d)) * scale, dtype)
        self.kp, self.vp = (dev(rng.standard_normal((nb, hkv, page, d)), dtype) for _ in range(2))

    def run(self):
        return ft.attention_decode_paged_prefix(
            self.q, self.kp, self.vp, i32(self.ptable), i32(self.plens), i32(self.table),
            i32(self.lens), i32(self.offsets))

    def check(self, got=None):
        got = self.run() if got is None else got
        want, mass, size = refs.attend_prefix(np64(self.q), np64(self.kp), np64(self.vp),
                                              self.ptable, self.plens, self.table, self.lens,
                                              self.offsets)
        near(got, want, mass, size, self.q.dtype, max(self.plens + [0]) + max(self.lens + [0]))
        return got


def near(got, want, mass, size, dtype, tokens):
    d = want.shape[-1]
    split = {torch.bfloat16: 2.0 ** -17, torch.float16: 2.0 ** -22, torch.float32: 0}[dtype]
    part = ((d / 16 + 22) * size + tokens / 16 + 200 + 4) * 2.0 ** -24 + split
    bound = torch.finfo(dtype).eps / 2 * np.abs(want) + 2 * part * mass
    if dtype is torch.float16:
        bound = bound + 2.0 ** -25   # half a step of the least numbers
    over = np.abs(np64(got) - want) - bound
    assert got.dtype == dtype and over.max(initial=-1) <= 0, over.max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [4, 8, 20, 64, 72, 96, 120, 128, 136, 256, 512])
def test_head_sizes(d, dtype):
    Case(d, 8, 2, d, 16, [130], [3], [0, 5, 70], dtype).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 1), (8, 8), (16, 1), (17, 1), (33, 1), (64, 1),
                                    (70, 1), (130, 1), (24, 2)])
def test_groups_of_heads(hq, hkv, dtype):
    Case(hq, hq, hkv, 64, 16, [200, 33], [2, 3], [9, 0, 64, 65, 1], dtype).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 100])
def test_pages(page, dtype):
    Case(page, 8, 2, 128, page, [333], [4], [1, 63, 64, 200], dtype).check()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b", [1, 2, 4, 5, 16, 17, 32, 33, 40, 70])
def test_rows_of_a_prefix(b, d):
    """1 to 280 rows a kv head: every kind of tile, whole and not."""
    for dtype in (torch.bfloat16, torch.float32):
        Case(b, 8, 2, d, 16, [700], [b], [(7 * i) % 30 for i in range(b)], dtype).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("plens,sizes,lens", [
    ([0], [3], [0, 0, 0]),              # nothing at all
    ([0], [3], [5, 0, 70]),             # own tokens alone
    ([77], [3], [0, 0, 0]),             # a prefix alone
    ([5, 0, 64, 1], [1, 0, 2, 1], [3, 0, 0, 9]),   # an empty group, groups of one
    ([100], [2], [1, 2, 3, 4]),         # the last two sequences in no group
    ([1], [1], [0]), ([0], [1], [1])])
def test_empty_parts(plens, sizes, lens, dtype):
    for d in (64, 20):
        c = Case(3, 8, 2, d, 16, plens, sizes, lens, dtype)
        got = c.check()
        none = [x for x in range(len(lens)) if lens[x] == 0 and not any(
            n and c.offsets[g] <= x < c.offsets[g + 1] for g, n in enumerate(plens))]
        assert (got[none] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_long_and_short(dtype):
    Case(1, 8, 2, 64, 16, [20000], [6], [0, 1, 3000, 17, 64, 900], dtype).check()


def test_many_groups():
    rng = np.random.default_rng(8)
    sizes = rng.integers(0, 4, 90)
    b = int(sizes.sum())
    Case(8, 4, 1, 64, 16, rng.integers(0, 90, 90), sizes, rng.integers(0, 40, b),
         torch.float16).check()


def test_most_sequences():
    rng = np.random.default_rng(9)
    b, g = 3000, 1096
    sizes = np.bincount(rng.integers(0, g, b), minlength=g)
    Case(9, 2, 1, 8, 4, rng.integers(0, 9, g), sizes, rng.integers(0, 6, b),
         torch.bfloat16).check()
    Case(9, 2, 1, 4, 4, rng.integers(0, 9, g), sizes, rng.integers(0, 6, b),
         torch.float32).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, 30.0])
def test_flat_and_sharp(scale, dtype):
    """Equal scores, and scores of hundreds of nats."""
    Case(2, 8, 2, 64, 16, [500], [4], [3, 90, 0, 10], dtype, scale=scale).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 20])
@pytest.mark.parametrize("b", [3, 12, 40])
def test_what_lies_behind_the_tokens_does_not_matter(b, d, dtype):
    c = Case(5, 8, 2, d, 16, [150], [b], [(11 * i) % 50 for i in range(b)], dtype)
    want = c.run()
    counted = torch.zeros(c.kp.shape[0], 16, dtype=torch.bool, device=DEV)
    for row, n in list(zip(c.ptable, c.plens)) + list(zip(c.table, c.lens)):
        for t in range(n):
            counted[row[t // 16], t % 16] = True
    for bad in (float("nan"), float("inf"), -float("inf")):
        for pool in (c.kp, c.vp):
            pool.masked_fill_(~counted[:, None, :, None], bad)
        assert torch.equal(c.run(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 20])
@pytest.mark.parametrize("b", [3, 12, 40])
def test_entries_without_a_block(b, d, dtype):
    """Tokens of entries outside the pools weigh nothing, whatever block 0 or
    the last one hold."""
    c = Case(6, 8, 2, d, 16, [150], [b], [(13 * i) % 60 for i in range(b)], dtype)
    c.ptable[0, 2], c.ptable[0, 5] = -1, c.kp.shape[0]
    c.table[1, 0], c.table[2, :] = 2 ** 31 - 1, -2 ** 31
    c.check()


@pytest.mark.parametrize("d", [64, 20])
def test_any_lengths_and_offsets_are_safe(d):
    c = Case(7, 8, 2, d, 16, [100, 40, 30], [2, 2, 2], [9, 0, 30, 5, 1, 20], torch.bfloat16)
    width, own = c.ptable.shape[1] * 16, c.table.shape[1] * 16
    c.plens, c.lens = [2 ** 31 - 1, -5, 31], [-1, 2 ** 31 - 1, 7, 0, -2 ** 31, 20]
    got = c.run()
    c.plens, c.lens = [width, 0, 31], [0, own, 7, 0, 0, 20]
    assert torch.equal(got, c.run())
    c.check(got)
    c.offsets = [-7, 3, 1, 2 ** 31 - 1]   # as [0, 3, 3, 6]
    got = c.run()
    c.offsets = [0, 3, 3, 6]
    c.check(got)


def test_no_lengths_and_no_offsets():
    c = Case(4, 8, 2, 128, 16, [96], [3], [32, 32, 32], torch.float16)
    c.ptable, c.table = c.ptable[:, :6].copy(), c.table[:, :2].copy()
    got = ft.attention_decode_paged_prefix(c.q, c.kp, c.vp, i32(c.ptable), None, i32(c.table))
    c.check(got)
    # tables and lengths from the host
    got2 = ft.attention_decode_paged_prefix(c.q, c.kp, c.vp, c.ptable, [96], c.table, [32] * 3,
                                            [0, 3])
    assert torch.equal(got, got2)
    none = torch.zeros((0, 4), device=DEV, dtype=torch.int32)
    alone = ft.attention_decode_paged_prefix(c.q, c.kp, c.vp, none, None, i32(c.table),
                                             i32(c.lens), i32([0]))
    c.plens, c.ptable, c.offsets = [], c.ptable[:0], [0]
    c.check(alone)
    empty = ft.attention_decode_paged_prefix(c.q[:0], c.kp, c.vp, none, None, none, i32([]))
    assert empty.shape == (0, 8, 128)


@pytest.mark.parametrize("dtype", TYPES)
def test_equals_one_table_of_both_parts(dtype):
    """A prefix of whole blocks: the paged decode over the joined tables, to
    the two bounds."""
    c = Case(11, 8, 2, 128, 16, [160], [5], [1, 40, 16, 0, 100], dtype)
    joined = np.concatenate([np.repeat(c.ptable[:, :10], 5, 0), c.table], 1)
    other = ft.attention_decode_paged(c.q, c.kp, c.vp, i32(joined), i32(np.add(c.lens, 160)))
    got, want, mass = np64(c.check()), *refs.attend_prefix(
        np64(c.q), np64(c.kp), np64(c.vp), c.ptable, c.plens, c.table, c.lens, c.offsets)[:2]
    # that op rounds fp16 weights to fp16 once: 2^-11 of a weight, in the
    # numerator alone (its bf16 weights and float32 ones have more bits than
    # this op's bound counts)
    room = 2.0 ** -11 * mass if dtype is torch.float16 else 0
    eps = torch.finfo(dtype).eps
    assert (np.abs(np64(other) - got) <= eps * np.abs(want) + 2.0 ** -14 * mass + room).all()


def test_rows_not_aligned_to_16_bytes():
    """Operands at 8-byte places take the general kernel."""
    c = Case(12, 8, 2, 64, 16, [90], [4], [5, 0, 33, 60], torch.bfloat16)
    flat = torch.empty(c.q.numel() + 4, device=DEV, dtype=c.q.dtype)
    q = flat[4:].view_as(c.q)
    q.copy_(c.q)
    c.q = q
    c.check()


def test_block_offsets_past_31_bits():
    """Blocks whose elements lie past 2^32 of the pool."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    hkv, page, d, nb = 8, 64, 128, (1 << 32) // (8 * 64 * 128) + 8
    kp, vp = (torch.zeros((nb, hkv, page, d), device=DEV, dtype=torch.bfloat16) for _ in range(2))
    rng = np.random.default_rng(1)
    used = [nb - 1, 3, nb - 4, nb - 2]
    for p in (kp, vp):
        p[used] = dev(rng.standard_normal((4, hkv, page, d)), torch.bfloat16)
    q = dev(rng.standard_normal((3, 16, d)), torch.bfloat16)
    got = ft.attention_decode_paged_prefix(q, kp, vp, i32([used[:2]]), i32([100]),
                                           i32([[used[2]], [used[3]], [0]]), i32([64, 30, 0]))
    small = [x[used].contiguous() for x in (kp, vp)]
    want = ft.attention_decode_paged_prefix(q, *small, i32([[0, 1]]), i32([100]),
                                            i32([[2], [3], [0]]), i32([64, 30, 0]))
    assert torch.equal(got, want)


def test_streams_and_graphs_at_once():
    cases = [Case(s, 8, 2, 128, 16, [900], [20], [(s * i) % 90 for i in range(20)],
                  torch.bfloat16) for s in (3, 5)]
    want = [c.run() for c in cases]
    args = [(c.q, c.kp, c.vp, i32(c.ptable), i32(c.plens), i32(c.table), i32(c.lens),
             i32(c.offsets)) for c in cases]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for a in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ft.attention_decode_paged_prefix(*a))
        graphs.append(graph)
    torch.cuda.synchronize()
    for turn in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = ft.attention_decode_paged_prefix(*args[turn % 2])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[turn % 2])
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_refusals():
    c = Case(0, 8, 2, 64, 16, [40], [2], [3, 4], torch.bfloat16)
    f, pt, pl, t, n = (ft.attention_decode_paged_prefix, i32(c.ptable), i32(c.plens),
                       i32(c.table), i32(c.lens))
    for bad, exc, word in [
            (lambda: f(c.q.cpu(), c.kp, c.vp, pt, pl, t, n), TypeError, "GPU"),
            (lambda: f(c.q.half(), c.kp, c.vp, pt, pl, t, n), TypeError, "dtype"),
            (lambda: f(c.q, c.kp, c.vp[:1], pt, pl, t, n), ValueError, "pools"),
            (lambda: f(c.q[..., :32].contiguous(), c.kp, c.vp, pt, pl, t, n), ValueError, "pools"),
            (lambda: f(c.q.transpose(0, 1), c.kp, c.vp, pt, pl, t, n), ValueError, "contiguous"),
            (lambda: f(c.q[:, :7].contiguous(), c.kp, c.vp, pt, pl, t, n), ValueError, "multiple"),
            (lambda: f(c.q, c.kp, c.vp, pt[0], pl, t, n), ValueError, "prefix_table"),
            (lambda: f(c.q, c.kp, c.vp, pt, i32([1, 2]), t, n), ValueError, "prefix_lens"),
            (lambda: f(c.q, c.kp, c.vp, pt, pl, t[:1], n), ValueError, "block_table"),
            (lambda: f(c.q, c.kp, c.vp, pt, pl, t, n[:1]), ValueError, "lens"),
            (lambda: f(c.q, c.kp, c.vp, pt, pl, t, n, i32([0, 1, 2])), ValueError, "entry more"),
            (lambda: f(c.q, c.kp, c.vp, pt.repeat(2, 1), pl.repeat(2), t, n), ValueError,
             "group_offsets"),
            (lambda: f(c.q, c.kp, c.vp, pt, [99999], t, n), ValueError, "prefix_lens"),
            (lambda: f(c.q, c.kp, c.vp, pt, pl, [[-1], [0]], n), ValueError, "block_table"),
            (lambda: f(c.q, c.kp, c.vp, pt, pl, t, n, [0, 3]), ValueError, "group_offsets"),
            (lambda: f(c.q, c.kp, c.vp, pt, pl.float(), t, [1.5, 2]), TypeError, "integer")]:
        with pytest.raises(exc, match=word):
            bad()
