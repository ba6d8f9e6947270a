"""GPU tests of the paged KV cache in 8 bits: block_table_extend,
kv_append_paged_int8 and attention_decode_paged_int8 against plain numpy forms
(cache8_refs). Tables, slots and codes are whole numbers and equal; scales are
equal bit for bit (float32 divisions); attention is held to a bound derived
from the arithmetic plus half a rounding step of the output's type."""

import numpy as np
import pytest
import torch

import fusedtok_amd as ft
from tests import cache8_refs as refs

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def dev(x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x)).to(DEV, dtype=dtype)


def i32(x):
    return dev(np.asarray(x, np.int32))


def rounded(x, dtype):
    """x rounded to a torch type, as float32."""
    return torch.as_tensor(np.asarray(x, np.float32)).to(dtype).float().numpy()


# ---------------------------------------------------------------------------
# tables
# ---------------------------------------------------------------------------


def run_extend(table, lens, counts, free, n_free, page, tokens):
    tb = i32(table)
    got = ft.block_table_extend(tb, i32(lens), i32(counts), i32(free), i32([n_free]), page,
                                tokens)
    return (tb.cpu().numpy(),) + tuple(x.cpu().numpy() for x in got)


def check_extend(table, lens, counts, free, n_free, page, tokens):
    table = np.asarray(table, np.int32).reshape(len(lens), -1)
    got = run_extend(table, lens, counts, free, n_free, page, tokens)
    want = refs.extend(table, lens, counts, free, n_free, page, tokens)
    for name, g, w in zip(("table", "slots", "positions", "offsets", "lens", "n_free"), got, want):
        np.testing.assert_array_equal(g, w, err_msg=name)


@pytest.mark.parametrize("page", [1, 5, 16, 64, 1024])
@pytest.mark.parametrize("b", [1, 3, 64, 257])
def test_extend_mixed(b, page):
    rng = np.random.default_rng(100 * b + page)
    width = 6
    lens = rng.integers(0, 3 * page + 1, b)
    counts = rng.integers(0, 2 * page + 2, b)   # idle, single tokens, chunks
    counts[rng.random(b) < 0.2] = 0
    free = rng.permutation(4 * b + 40).astype(np.int32)
    table = rng.integers(0, 1000, (b, width)).astype(np.int32)
    total = int(counts.sum())
    for tokens in (total, total + 7, max(0, total - 3)):
        check_extend(table, lens, counts, free, len(free) - 1, page, tokens)


def test_extend_edges():
    full = np.arange(8, dtype=np.int32).reshape(2, 4)
    free = np.arange(100, 140, dtype=np.int32)
    # a sequence exactly at a block's end, and one at the table's
    check_extend(full, [8, 16], [1, 2], free, 40, 4, 3)
    # behind the table's end: no block, no slot
    check_extend(full, [14, 15], [9, 1], free, 40, 4, 10)
    # lens past the capacity and negative values
    check_extend(full, [99, -3], [2, 2], free, 40, 4, 4)
    check_extend(full, [3, 4], [-5, 2], free, 40, 4, 4)
    # the list spent in the middle, empty, and already short
    check_extend(np.full((3, 8), 7), [0, 3, 5], [9, 9, 9], free, 3, 4, 27)
    check_extend(full, [4, 8], [1, 1], free[:0], 0, 4, 2)
    check_extend(full, [4, 8], [1, 1], free, -2, 4, 2)
    # a count that claims more than the list holds reads nothing behind it
    check_extend(full, [4, 8], [1, 1], free[:2], 4, 4, 2)
    # tokens in a block that could not be had get no slot either
    holed = np.array([[3, -1, 0, 0]])
    check_extend(holed, [5], [2], free, 40, 4, 2)
    # nothing at all
    got = run_extend(np.zeros((0, 4), np.int32), [], [], free, 40, 4, 3)
    assert got[1].tolist() == [-1] * 3 and got[2].tolist() == [0] * 3
    assert got[3].tolist() == [0] and got[5].tolist() == [40]
    check_extend(full, [4, 8], [0, 0], free, 40, 4, 0)


def test_extend_most_sequences():
    rng = np.random.default_rng(5)
    b, page = 4096, 16
    lens, counts = rng.integers(0, 60, b), rng.integers(0, 3, b)
    free = rng.permutation(3 * b).astype(np.int32)
    check_extend(rng.integers(0, 99, (b, 5)), lens, counts, free, len(free), page,
                 int(counts.sum()))


def test_extend_many_tokens():
    rng = np.random.default_rng(6)
    lens, counts = np.array([3, 0, 100]), np.array([30000, 0, 12345])
    free = rng.permutation(5000).astype(np.int32)
    check_extend(np.zeros((3, 2000)), lens, counts, free, 5000, 16, 42345)


def test_extend_steps_add_up():
    """Prompts, then steps fed with each other's outputs: every token of a
    sequence ends at the slot its table gives."""
    page, b = 4, 3
    table = torch.full((b, 16), -1, dtype=torch.int32, device=DEV)
    free = i32(np.random.default_rng(7).permutation(64))
    n_free = i32([64])
    lens = i32([0] * b)
    seen = [[] for _ in range(b)]
    for step in range(12):
        counts = [5, 1, 7] if step == 0 else [step % 2, 1, 2]
        slots, pos, off, lens, n_free = ft.block_table_extend(table, lens, i32(counts), free,
                                                              n_free, page, sum(counts) + 1)
        s, o = slots.tolist(), off.tolist()
        for i in range(b):
            seen[i] += s[o[i]:o[i + 1]]
    tb = table.cpu().numpy()
    for i in range(b):
        n = int(lens[i])
        assert n == len(seen[i])
        assert seen[i] == [int(tb[i, p // page]) * page + p % page for p in range(n)]
    used = tb[tb >= 0]
    assert len(set(used.tolist())) == len(used) == 64 - int(n_free)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------


def pools(rng, nb, hkv, page, d):
    kp, vp = (rng.integers(-127, 128, (nb, hkv, page, d)).astype(np.int8) for _ in range(2))
    ks, vs = ((0.01 + 0.05 * rng.random((nb, hkv))).astype(np.float32) for _ in range(2))
    return kp, vp, ks, vs


def check_append(cache, k, v, slots, dtype):
    got = [dev(x) for x in cache]
    kd, vd = (torch.as_tensor(np.asarray(x, np.float32)).to(dtype) for x in (k, v))
    ft.kv_append_paged_int8(*got, kd.to(DEV), vd.to(DEV), i32(slots))
    kp, vp, ks, vs = (x.cpu().numpy() for x in got)
    for name, codes, scales, c0, s0, new in (("k", kp, ks, cache[0], cache[2], kd),
                                             ("v", vp, vs, cache[1], cache[3], vd)):
        want_c, want_s = refs.append(c0, s0, new.float().numpy(), np.asarray(slots))
        np.testing.assert_array_equal(scales, want_s, err_msg=name + " scales")
        np.testing.assert_array_equal(codes, want_c, err_msg=name + " codes")
    return kp, vp, ks, vs


def seq_slots(rng, nb, page, lens, fresh):
    """Slots of `fresh` tokens behind `lens` cached ones, blocks permuted."""
    ids, at, slots = rng.permutation(nb), 0, []
    for n, add in zip(lens, fresh):
        need = -(-(n + add) // page)
        blocks = ids[at:at + need]
        at += need
        slots += [int(blocks[p // page]) * page + p % page for p in range(n, n + add)]
    assert at <= nb
    return slots


SHAPES = [(2, 16, 128), (3, 16, 64), (1, 64, 128), (8, 24, 128), (2, 5, 100), (1, 1, 4),
          (2, 1024, 8), (1, 16, 512), (2, 32, 256), (1, 128, 128), (4, 7, 36)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("hkv,page,d", SHAPES)
def test_append(hkv, page, d, dtype):
    rng = np.random.default_rng(hkv + 10 * page + d)
    lens = [0, 1, page - 1, page, 2 * page + page // 2, 0]
    fresh = [page + 1, 1, 1, 1, page + 3, 0]
    nb = sum(-(-(n + a) // page) for n, a in zip(lens, fresh)) + 3
    cache = pools(rng, nb, hkv, page, d)
    slots = seq_slots(rng, nb, page, lens, fresh) + [-1, -1]
    k, v = (rng.standard_normal((len(slots), hkv, d)) * 3 for _ in range(2))
    k[::3] *= 0.05   # rows that grow no scale, among rows that do
    check_append(cache, k, v, slots, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("t,hkv,page,d", [(700, 8, 16, 128), (3000, 4, 64, 64), (2111, 2, 24, 128),
                                          (5000, 1, 16, 64)])
def test_append_prompts(t, hkv, page, d, dtype):
    rng = np.random.default_rng(t)
    fresh = [t // 2, t // 3, t - t // 2 - t // 3]
    lens = [0, 3, page]
    nb = sum(-(-(n + a) // page) for n, a in zip(lens, fresh)) + 1
    cache = pools(rng, nb, hkv, page, d)
    slots = seq_slots(rng, nb, page, lens, fresh)
    k, v = (rng.standard_normal((t, hkv, d)) for _ in range(2))
    check_append(cache, k, v, slots, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,hkv,page,d", [(9, 2, 16, 128), (70, 8, 16, 128), (200, 16, 64, 64),
                                             (300, 8, 24, 96)])
def test_append_padded_batch(rows, hkv, page, d, dtype):
    """[sequences, rows] padded to one length: -1 behind each sequence's own,
    some sequences with none; few rows and enough for windows of a block."""
    rng = np.random.default_rng(rows)
    b = 14
    lens = rng.integers(0, 3 * page, b)
    fresh = rng.integers(0, rows + 1, b)
    fresh[[0, 5, b - 1]] = 0, rows, 0
    nb = int(sum(-(-(n + a) // page) for n, a in zip(lens, fresh))) + 2
    cache = pools(rng, nb, hkv, page, d)
    flat, at = seq_slots(rng, nb, page, lens, fresh), 0
    slots = np.full((b, rows), -1)
    for i, a in enumerate(fresh):
        slots[i, :a] = flat[at:at + a]
        at += a
    k, v = (rng.standard_normal((b * rows, hkv, d)) * 2 for _ in range(2))
    check_append(cache, k, v, slots.reshape(-1), dtype)


@pytest.mark.parametrize("b", [1, 100, 1024, 1025, 3000])
@pytest.mark.parametrize("page,d", [(16, 64), (5, 32), (64, 128)])
def test_append_step(b, page, d):
    """One token for each of b sequences, in the middle of a block, at its
    start and at its end."""
    rng = np.random.default_rng(b)
    nb = b + 2
    cache = pools(rng, nb, 2, page, d)
    rows = rng.integers(0, page, b)
    rows[::5], rows[1::5] = 0, page - 1
    slots = rng.permutation(nb)[:b] * page + rows
    slots[3::11] = -1
    k, v = (rng.standard_normal((b, 2, d)) * rng.choice([0.1, 5], (b, 1, 1)) for _ in range(2))
    check_append(cache, k, v, slots, torch.bfloat16)


@pytest.mark.parametrize("page,d", [(16, 128), (5, 64), (64, 128)])
def test_append_odd_slots(page, d):
    """Slots outside the pools, gaps between a block's rows, rows out of
    order, the same slot twice and three times, rows of no sequence first."""
    rng = np.random.default_rng(page)
    nb = 9
    cache = pools(rng, nb, 2, page, d)
    last = nb * page
    slots = [-1, last, -2 ** 31, 2 ** 31 - 1,
             2 * page + 3, 2 * page + 1, 2 * page + 4,       # out of order
             5 * page + 2, 5 * page + 2, 5 * page + 2,       # one slot three times
             -7, 0, 4, 2, 0,                                 # row 0: starts over; gaps
             last - 1, last]
    k, v = (rng.standard_normal((len(slots), 2, d)) * 4 for _ in range(2))
    check_append(cache, k, v, slots, torch.float32)


@pytest.mark.parametrize("rows,hkv,page,d", [(150, 1, 16, 64), (700, 64, 16, 64),
                                             (900, 40, 64, 128), (2000, 8, 16, 64)])
def test_append_longer_run_than_a_block(rows, hkv, page, d):
    """The same rows again and again: a run of more rows than the block has,
    and one that reaches over several windows."""
    rng = np.random.default_rng(3)
    cache = pools(rng, 4, hkv, page, d)
    slots = [page + (7 * i) % 11 + 2 for i in range(rows)]
    k, v = (rng.standard_normal((rows, hkv, d)) for _ in range(2))
    check_append(cache, k, v, slots, torch.bfloat16)


def test_append_off_alignment():
    """Rows at 8 elements' alignment and at 4: the same codes."""
    rng = np.random.default_rng(14)
    cache = pools(rng, 3, 2, 16, 64)
    k, v = (rng.standard_normal((20, 2, 64)).astype(np.float32) for _ in range(2))
    slots = i32(np.arange(20))
    got = []
    for off in (0, 4, 12):
        at = [dev(x) for x in cache]
        kv = []
        for x in (k, v):
            buf = torch.zeros(x.size + 16, dtype=torch.float16, device=DEV)
            kv.append(buf[off:off + x.size].view(x.shape))
            kv[-1].copy_(dev(x))
        ft.kv_append_paged_int8(*at, *kv, slots)
        got.append(at)
    for other in got[1:]:
        assert all(torch.equal(x, y) for x, y in zip(got[0], other))
    with pytest.raises(ValueError):
        bad = torch.zeros(20 * 2 * 64 + 2, dtype=torch.float16, device=DEV)[2:].view(20, 2, 64)
        ft.kv_append_paged_int8(*got[0], bad, kv[1], slots)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_append_values(dtype):
    """Infinities and NaN beside ordinary values, zeros, values below the
    least scale, the type's largest, halves of a step."""
    rng = np.random.default_rng(4)
    page, d, nb = 16, 64, 8
    cache = pools(rng, nb, 1, page, d)
    top = float(torch.finfo(dtype).max)
    rows = [np.full(d, x) for x in (0.0, 1e-40, -top, np.inf, np.nan)]
    mixed = rng.standard_normal(d)
    mixed[::7], mixed[1::7], mixed[2::7] = np.inf, -np.inf, np.nan
    halves = np.arange(d) - 31.5
    halves[0] = 127.0
    rows += [mixed, halves, np.zeros(d)]
    slots = [i * page + (0 if i % 2 else 3) for i in range(8)]
    k = np.stack(rows)[:, None]
    kp, _, ks, _ = check_append(cache, k, k[::-1], slots, dtype)
    assert np.isfinite(ks).all()
    # a block that starts over with zeros alone: zero codes
    assert not kp[7, 0, 0].any()


def test_append_keeps_the_rest():
    """Only the touched blocks change; without growth only the fresh rows."""
    rng = np.random.default_rng(8)
    cache = pools(rng, 6, 2, 16, 128)
    k = rng.standard_normal((1, 2, 128)) * 1e-3
    kp, vp, ks, vs = check_append(cache, k, k, [2 * 16 + 5], torch.bfloat16)
    keep = np.ones(kp.shape, bool)
    keep[2, :, 5] = False
    assert (kp[keep] == cache[0][keep]).all() and (vp[keep] == cache[1][keep]).all()
    assert (ks == cache[2]).all() and (vs == cache[3]).all()


def test_append_nothing():
    rng = np.random.default_rng(9)
    cache = pools(rng, 3, 1, 16, 64)
    check_append(cache, np.zeros((0, 1, 64)), np.zeros((0, 1, 64)), [], torch.float32)
    empty = pools(rng, 0, 1, 16, 64)
    got = [dev(x) for x in empty]
    new = torch.zeros(2, 1, 64, device=DEV)
    ft.kv_append_paged_int8(*got, new, new, i32([0, 1]))


def test_append_off_by_half_a_step():
    """What the cache holds after one append: within half a step of x."""
    rng = np.random.default_rng(10)
    x = rng.standard_normal((16, 1, 128)).astype(np.float32)
    cache = pools(rng, 2, 1, 16, 128)
    kp, _, ks, _ = check_append(cache, x, x, np.arange(16), torch.float32)
    held = kp[0, 0].astype(np.float64) * ks[0, 0]
    # half a step, and the roundings of x * (1 / scale) (2 of 2^-24 of 127)
    assert np.abs(held - x[:, 0]).max() <= ks[0, 0] * (0.5 + 127 * 2.0 ** -22)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def paged(rng, b, hkv, page, d, lens, spare=2):
    lens = np.asarray(lens)
    need = -(-lens // page)
    width = max(1, int(need.max(initial=0)))
    nb = int(need.sum()) + spare
    ids = rng.permutation(nb)
    table = rng.integers(0, nb, (b, width)).astype(np.int32)
    at = 0
    for i in range(b):
        table[i, :need[i]] = ids[at:at + need[i]]
        at += need[i]
    return pools(rng, nb, hkv, page, d), table


def check_attend(q, cache, table, lens, dtype, given=None):
    qd = torch.as_tensor(np.asarray(q, np.float32)).to(dtype)
    out = ft.attention_decode_paged_int8(qd.to(DEV), *[dev(x) for x in cache], i32(table),
                                         i32(lens) if given is None else given[0])
    want, room = refs.attend(qd.float().numpy(), *cache, table, lens)
    got = out.cpu().double().numpy()
    assert out.dtype is dtype and np.isfinite(got).all()
    tol = refs.half_step(dtype) * np.abs(want) + room
    tol = tol + refs.PARTS[str(dtype)] * abs_out(qd.float().numpy(), cache, table, lens)
    if dtype is torch.float16:
        tol = tol + 2.0 ** -25   # half a step of its smallest numbers
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.abs(got - want)[bad].max(), tol[bad].min(), np.argwhere(bad)[:5])
    return out


def abs_out(q, cache, table, lens):
    kp, vp, ks, vs = cache
    return refs.attend(q, kp, np.abs(vp.astype(np.int16)), ks, np.abs(vs), table, lens)[0]


LENS = {"short": [1, 0, 2, 17], "mixed": [33, 1, 0, 300, 64, 129], "long": [2500, 7]}


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("hkv,group,page,d", [
    (2, 4, 16, 128), (2, 4, 16, 64), (1, 16, 64, 128), (3, 1, 24, 64), (2, 5, 5, 128),
    (1, 20, 16, 128), (1, 33, 16, 64), (2, 3, 1, 64), (2, 4, 16, 256), (1, 8, 128, 128),
    (2, 2, 7, 36), (1, 4, 16, 512), (1, 1, 1024, 4), (2, 4, 16, 96), (2, 3, 16, 16),
    (1, 4, 5, 48), (2, 8, 16, 80), (1, 17, 24, 112), (2, 4, 16, 144), (1, 2, 32, 192),
    (1, 9, 16, 240), (2, 4, 16, 260), (1, 6, 3, 100)])
def test_attend(hkv, group, page, d, lens, dtype):
    lens = LENS[lens]
    rng = np.random.default_rng(hkv + 7 * group + 11 * page + d + len(lens))
    cache, table = paged(rng, len(lens), hkv, page, d, lens)
    q = rng.standard_normal((len(lens), hkv * group, d)) * 2
    check_attend(q, cache, table, lens, dtype)


@pytest.mark.parametrize("d", [64, 128, 32, 20])
def test_attend_whole_table(d):
    """lens None: every row; lens beyond the capacity and negative ones are
    clamped."""
    rng = np.random.default_rng(d)
    cache, table = paged(rng, 3, 2, 16, d, [80, 80, 80])
    q = rng.standard_normal((3, 8, d))
    qd, args = dev(q, torch.bfloat16), [dev(x) for x in cache]
    check_attend(q, cache, table, [80] * 3, torch.bfloat16, given=(None,))
    # (how a row is cut, so its last bits, may depend on the others' lengths)
    got, same, none = (ft.attention_decode_paged_int8(qd, *args, i32(table), i32(lens))
                       for lens in ([999, -4, 80], [80, 0, 80], [0, 0, 0]))
    assert torch.equal(got, same)
    assert not got[1].any() and not none.any()


@pytest.mark.parametrize("page", [16, 5, 64])
@pytest.mark.parametrize("d", [64, 128, 96, 36])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attend_holes(d, page, dtype):
    """Table entries outside the pools: their tokens weigh nothing; a row of
    nothing else is zero."""
    rng = np.random.default_rng(d + page)
    lens = [200, 64, 5, 130]
    cache, table = paged(rng, 4, 2, page, d, lens)
    nb = cache[0].shape[0]
    table[0, 1], table[0, 3], table[3, 0] = -1, nb, -2 ** 31
    table[1, :], table[2, 0] = -1, 2 ** 31 - 1
    q = rng.standard_normal((4, 8, d)) * 2
    out = check_attend(q, cache, table, lens, dtype)
    assert not out[1].any() and not out[2].any()


@pytest.mark.parametrize("d", [64, 128, 96, 36])
def test_attend_unused_values(d):
    """Blocks and scales behind a row's last token - NaN, infinity, anything -
    reach no output."""
    rng = np.random.default_rng(d)
    lens = [33, 47]
    (kp, vp, ks, vs), table = paged(rng, 2, 2, 16, d, lens, spare=8)
    used = set(table[0, :3].tolist() + table[1, :3].tolist())
    table = np.concatenate([table, np.full((2, 4), -1, np.int32)], 1)
    rest = [i for i in range(kp.shape[0]) if i not in used]
    table[:, 3], table[:, 4] = rest[0], rest[1]
    ks[rest], vs[rest] = np.nan, np.inf
    q = rng.standard_normal((2, 4, d))
    for dtype in TYPES:
        check_attend(q, (kp, vp, ks, vs), table, lens, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128, 96, 36])
def test_attend_small_weights(d, dtype):
    """Thousands of keys 25 nats below four dominant ones whose values are 0:
    what they add is small, and has to come out right."""
    rng = np.random.default_rng(1)
    n, page = 4096, 16
    (kp, vp, ks, vs), table = paged(rng, 1, 1, page, d, [n])
    kp[:] = 0
    kp[..., 0] = rng.integers(-3, 4, kp.shape[:-1])
    ks[:] = vs[:] = 0.5
    first = table[0, 0]
    kp[first, 0, :4, 0] = 100
    vp[first, 0, :4] = 0
    q = np.zeros((1, 4, d))
    q[..., 0] = 25.0 / 48.5 * d ** 0.5
    check_attend(q, (kp, vp, ks, vs), table, [n], dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128, 96, 36])
def test_attend_scales_of_all_sizes(d, dtype):
    """Blocks' scales from 1e-30 to 1e4, zero scales, large and small q."""
    rng = np.random.default_rng(2)
    lens = [500, 100]
    (kp, vp, ks, vs), table = paged(rng, 2, 2, 16, d, lens)
    ks[:] = 10.0 ** rng.uniform(-30, -1.5, ks.shape)
    vs[:] = 10.0 ** rng.uniform(-30, 2, vs.shape)
    ks[::5], vs[::7] = 0.0, 0.0
    q = rng.standard_normal((2, 8, d)) * 10.0 ** rng.uniform(-4, 0.5, (2, 8, 1))
    check_attend(q, (kp, vp, ks, vs), table, lens, dtype)


@pytest.mark.parametrize("b,hkv,lens", [(300, 1, 9), (70, 8, 3), (2100, 1, 2), (5, 2, 1500)])
def test_attend_many_rows(b, hkv, lens):
    rng = np.random.default_rng(b)
    lens = rng.integers(0, lens + 1, b)
    cache, table = paged(rng, b, hkv, 16, 64, lens)
    q = rng.standard_normal((b, 2 * hkv, 64))
    check_attend(q, cache, table, lens, torch.float32)


@pytest.mark.parametrize("d", [128, 96, 100])
def test_cache_beyond_32_bits(d):
    """A pool of more than 2^32 bytes: append to its last blocks, attend
    them."""
    page, hkv = 64, 8
    nb = 2 ** 32 // (page * hkv * d) + 40
    kp, vp = (torch.zeros(nb, hkv, page, d, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(nb, hkv, device=DEV) for _ in range(2))
    rng = np.random.default_rng(11)
    lens = [130, 70]
    table = np.array([[nb - 1, 3, nb - 17], [nb - 30, nb - 2, 0]], np.int32)
    slots = [int(table[i, p // page]) * page + p % page for i in range(2) for p in range(lens[i])]
    k, v = (rng.standard_normal((200, hkv, d)).astype(np.float32) for _ in range(2))
    ft.kv_append_paged_int8(kp, vp, ks, vs, dev(k), dev(v), i32(slots))
    used = np.unique(table)
    at = {int(n): i for i, n in enumerate(used)}
    pick = torch.as_tensor(used, dtype=torch.int64, device=DEV)
    cache = [x[pick].cpu().numpy() for x in (kp, vp, ks, vs)]
    zero = np.zeros_like(cache[0]), np.zeros_like(cache[2])
    small = [at[s // page] * page + s % page for s in slots]
    for codes, scales, new in ((cache[0], cache[2], k), (cache[1], cache[3], v)):
        want_c, want_s = refs.append(*zero, new, small)
        np.testing.assert_array_equal(codes, want_c)
        np.testing.assert_array_equal(scales, want_s)
    q = rng.standard_normal((2, 16, d)).astype(np.float32)
    out = ft.attention_decode_paged_int8(dev(q), kp, vp, ks, vs, i32(table), i32(lens))
    local = np.vectorize(at.get)(table)
    want, room = refs.attend(q, *cache, local, lens)
    tol = room + 2.0 ** -24 * np.abs(want) + 2.0 ** -22 * abs_out(q, cache, local, lens)
    assert (np.abs(out.cpu().double().numpy() - want) <= tol).all()


# ---------------------------------------------------------------------------
# together: streams, captures, a decode loop
# ---------------------------------------------------------------------------


def decode_state(rng, b=4, hkv=2, group=4, page=16, d=128, width=12, dtype=torch.bfloat16):
    nb = b * width
    cache = [dev(x) for x in pools(rng, nb, hkv, page, d)]
    return dict(cache=cache, table=torch.full((b, width), -1, dtype=torch.int32, device=DEV),
                free=i32(rng.permutation(nb)), n_free=i32([nb]), lens=i32([0] * b),
                hkv=hkv, group=group, page=page, d=d, b=b, dtype=dtype)


def step(st, counts, tokens, q, k, v):
    slots, pos, off, lens, n_free = ft.block_table_extend(
        st["table"], st["lens"], counts, st["free"], st["n_free"], st["page"], tokens)
    ft.kv_append_paged_int8(*st["cache"], k, v, slots)
    out = ft.attention_decode_paged_int8(q, *st["cache"], st["table"], lens)
    st["lens"].copy_(lens)
    st["n_free"].copy_(n_free)
    return out


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_then_decode_steps(d):
    """Prompts of different lengths, then steps: after each the attention over
    the cache is that of the cache's own values, and near the attention over
    the values that were appended."""
    rng = np.random.default_rng(d)
    st = decode_state(rng, d=d)
    b, hkv = st["b"], st["hkv"]
    lens = np.zeros(b, int)
    kept = [[[] for _ in range(b)] for _ in range(2)]
    for turn in range(20):
        counts = np.array([40, 3, 0, 16]) if turn == 0 else np.array([1, 1, turn % 2, 1])
        tokens = int(counts.sum()) + 2
        k, v = (rounded(rng.standard_normal((tokens, hkv, d)), st["dtype"]) for _ in range(2))
        q = rounded(rng.standard_normal((b, hkv * st["group"], d)), st["dtype"])
        out = step(st, i32(counts), tokens, dev(q, st["dtype"]), dev(k, st["dtype"]),
                   dev(v, st["dtype"]))
        at = 0
        for i in range(b):
            for kind, x in ((0, k), (1, v)):
                kept[kind][i].extend(x[at:at + counts[i]])
            at += counts[i]
        lens += counts
        assert st["lens"].tolist() == lens.tolist()
        cache = [x.cpu().numpy() for x in st["cache"]]
        table = st["table"].cpu().numpy()
        want, room = refs.attend(q, *cache, table, lens)
        tol = room + (2.0 ** -8) * np.abs(want) + 2.0 ** -15 * abs_out(q, cache, table, lens)
        assert (np.abs(out.cpu().double().numpy() - want) <= tol).all()
        # the cached values: within (1 + growths) / 2 steps of what went in; a
        # block's scale grows at most once a row
        for i in range(b):
            for codes, scales, rows in ((cache[0], cache[2], kept[0][i]),
                                        (cache[1], cache[3], kept[1][i])):
                for p in range(lens[i]):
                    n = table[i, p // st["page"]]
                    got = codes[n, :, p % st["page"]] * scales[n][:, None]
                    assert (np.abs(got - rows[p]) <= scales[n][:, None] * 9).all()


def test_captured_step_replays():
    """The whole step in one graph, replayed with eager work between, against
    the same steps run eagerly from the same start."""
    def make(seed):
        rng = np.random.default_rng(seed)
        st = decode_state(rng)
        prompt = [20, 5, 1, 37]
        n = sum(prompt)
        k, v = (dev(rng.standard_normal((n, 2, 128)), torch.bfloat16) for _ in range(2))
        q = dev(rng.standard_normal((4, 8, 128)), torch.bfloat16)
        step(st, i32(prompt), n, q, k, v)
        return rng, st
    rng, eager = make(1)
    _, graphed = make(1)
    ones = i32([1, 1, 0, 1])
    q, k, v = (torch.zeros(s, dtype=torch.bfloat16, device=DEV)
               for s in ((4, 8, 128), (4, 2, 128), (4, 2, 128)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out = step(graphed, ones, 4, q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(12):
        new = [dev(rng.standard_normal(x.shape), torch.bfloat16) for x in (q, k, v)]
        for x, y in zip((q, k, v), new):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = step(eager, ones, 4, *new)   # eager work between the replays
        assert torch.equal(got, want)
        for x, y in zip(graphed["cache"] + [graphed["table"], graphed["lens"], graphed["n_free"]],
                        eager["cache"] + [eager["table"], eager["lens"], eager["n_free"]]):
            assert torch.equal(x, y)


@pytest.mark.parametrize("d", [128, 36])
def test_values_that_are_not_finite(d):
    """A query or a scale that is not finite reaches the rows that attend it
    and no other."""
    rng = np.random.default_rng(13)
    lens = [40, 70, 100]
    (kp, vp, ks, vs), table = paged(rng, 3, 2, 16, d, lens)
    q = rng.standard_normal((3, 8, d)).astype(np.float32)
    args = [dev(x) for x in (q, kp, vp, ks, vs)]
    clean = ft.attention_decode_paged_int8(*args, i32(table), i32(lens))
    bad_q, bad_v = args[0].clone(), args[4].clone()
    bad_q[0, 3, 1] = float("nan")
    bad_q[1, 0, 2] = float("inf")
    bad_v[int(table[2, 1]), 1] = float("nan")
    out = ft.attention_decode_paged_int8(bad_q, *args[1:4], bad_v, i32(table), i32(lens))
    hit = torch.zeros(3, 8, dtype=torch.bool, device=DEV)
    hit[0, 3] = hit[1, 0] = True
    hit[2, 4:] = True
    assert torch.equal(out[~hit], clean[~hit])
    assert out[hit].isnan().any(-1).all()


def test_calls_on_two_streams():
    """Calls in flight on two streams at once, and two captured graphs
    replayed at once, share nothing."""
    rng = np.random.default_rng(12)
    calls = []
    for lens in ([3000, 20, 700], [1500, 1500, 9]):
        cache, table = paged(rng, 3, 4, 16, 128, lens)
        q = dev(rng.standard_normal((3, 16, 128)), torch.bfloat16)
        calls.append((q, *[dev(x) for x in cache], i32(table), i32(lens)))
    want = [ft.attention_decode_paged_int8(*c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(s):
                got[i].append(ft.attention_decode_paged_int8(*c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    graphs, outs = [], []
    for c, s in zip(calls, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(ft.attention_decode_paged_int8(*c))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(10):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------


def good():
    rng = np.random.default_rng(0)
    kp, vp, ks, vs = (dev(x) for x in pools(rng, 4, 2, 16, 64))
    return dict(q=torch.zeros(1, 4, 64, device=DEV), k_pool=kp, v_pool=vp, k_scales=ks,
                v_scales=vs, block_table=i32([[0, 1]]), lens=i32([5]))


@pytest.mark.parametrize("change,error", [
    (dict(q=lambda x: x.double()), TypeError), (dict(q=lambda x: x.cpu()), TypeError),
    (dict(k_pool=lambda x: x.float()), TypeError), (dict(k_scales=lambda x: x.half()), TypeError),
    (dict(v_pool=lambda x: x[:3]), ValueError), (dict(v_scales=lambda x: x[:, :1]), ValueError),
    (dict(k_pool=lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)), ValueError),
    (dict(q=lambda x: x[:, :3].contiguous()), ValueError), (dict(q=lambda x: x[0]), ValueError),
    (dict(q=lambda x: x[..., :32].contiguous()), ValueError),
    (dict(block_table=lambda x: x[0]), ValueError), (dict(lens=lambda x: i32([1, 2])), ValueError),
    (dict(block_table=lambda x: [[0, 4]]), ValueError), (dict(lens=lambda x: [33]), ValueError),
    (dict(q=lambda x: torch.zeros(257, device=DEV)[1:].view(1, 4, 64)), ValueError),
])
def test_attend_refuses(change, error):
    args = good()
    for name, f in change.items():
        args[name] = f(args[name])
    with pytest.raises(error):
        ft.attention_decode_paged_int8(**args)


@pytest.mark.parametrize("d,page", [(6, 16), (516, 16), (64, 1025)])
def test_sizes_refused(d, page):
    kp, vp = (torch.zeros(2, 1, page, d, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(2, 1, device=DEV) for _ in range(2))
    x = torch.zeros(1, 1, d, device=DEV)
    with pytest.raises(ValueError):
        ft.attention_decode_paged_int8(x, kp, vp, ks, vs, i32([[0]]))
    with pytest.raises(ValueError):
        ft.kv_append_paged_int8(kp, vp, ks, vs, x, x, i32([0]))


def test_append_refuses():
    a = good()
    new = torch.zeros(2, 2, 64, device=DEV)
    slots = i32([0, 1])
    pools_ = (a["k_pool"], a["v_pool"], a["k_scales"], a["v_scales"])
    for args, error in [
            ((*pools_, new, new, slots.long()), TypeError),
            ((*pools_, new, new.half(), slots), TypeError),
            ((*pools_, new, new[:1], slots), ValueError),
            ((*pools_, new[:, :1].contiguous(), new[:, :1].contiguous(), slots), ValueError),
            ((*pools_, new, new, slots[:1]), ValueError),
            ((*pools_, new, new, [0, 1]), TypeError),
            ((a["k_pool"], a["k_pool"], *pools_[2:], new, new, slots), ValueError),
            ((*pools_[:3], a["k_scales"], new, new, slots), ValueError),
            ((*pools_[:2], a["k_scales"].double(), pools_[3], new, new, slots), TypeError),
            ((*pools_, new.cpu(), new, slots), TypeError)]:
        with pytest.raises(error):
            ft.kv_append_paged_int8(*args)


def test_extend_refuses():
    table, one = i32([[0, 1]]), i32([1])
    free = i32([5, 6])
    ok = dict(block_table=table, lens=one, counts=one, free_blocks=free, n_free=one, page=16,
              tokens=1)
    ft.block_table_extend(**ok)
    for change, error in [
            (dict(block_table=table.long()), TypeError), (dict(lens=one.long()), TypeError),
            (dict(lens=[1]), TypeError), (dict(counts=i32([1, 2])), ValueError),
            (dict(n_free=i32([1, 2])), ValueError), (dict(free_blocks=table), ValueError),
            (dict(block_table=i32(np.zeros((4, 2)))[:, :1]), ValueError),
            (dict(page=0), ValueError), (dict(page=1025), ValueError),
            (dict(tokens=-1), ValueError), (dict(block_table=table.cpu()), TypeError)]:
        with pytest.raises(error):
            ft.block_table_extend(**{**ok, **change})
    many = torch.zeros(4097, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        ft.block_table_extend(torch.zeros(4097, 1, dtype=torch.int32, device=DEV), many, many,
                              free, one, 16, 1)
