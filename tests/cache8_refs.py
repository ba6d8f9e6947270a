"""Plain numpy forms of the 8-bit paged cache's operators: tables and slots by
a loop over tokens, the append's codes by its float32 definition, attention in
64 bits with a bound on what float32 arithmetic may add."""

import math

import numpy as np

LEAST = np.float32(2.0 ** -120)


def extend(table, lens, counts, free, n_free, page, tokens):
    """(table, slots, positions, offsets, new_lens, new_free) of
    block_table_extend, token by token."""
    table = table.copy()
    width = table.shape[1]
    span, left = width * page, int(n_free)
    slots, pos, offsets, after = [], [], [0], []
    for b in range(len(lens)):
        n, add = min(max(int(lens[b]), 0), span), max(int(counts[b]), 0)
        for p in range(n, n + add):
            slot = -1
            if p < span:
                if p % page == 0:
                    left -= 1
                    table[b, p // page] = free[left] if 0 <= left < len(free) else -1
                if table[b, p // page] >= 0:
                    slot = int(table[b, p // page]) * page + p % page
            slots.append(slot)
            pos.append(p)
        offsets.append(offsets[-1] + add)
        after.append(min(n + add, span))
    slots = (slots + [-1] * tokens)[:tokens]
    pos = (pos + [0] * tokens)[:tokens]
    as32 = [np.array(x, np.int32) for x in (slots, pos, offsets, after, [left])]
    return (table, *as32)


def append(pool, scales, new, slots):
    """(codes, scales) of one of K and V after kv_append_paged_int8: new
    [T, Hkv, D] float32 (exact values of the stored type)."""
    pool, scales = pool.copy(), scales.copy()
    nb, hkv, page, _ = pool.shape
    f32 = np.float32
    runs = []   # (block, {row: source})
    for i, s in enumerate(slots):
        if not 0 <= s < nb * page:
            runs.append((None, {}))
            continue
        block, row = divmod(int(s), page)
        if not runs or runs[-1][0] != block:
            runs.append((block, {}))
        runs[-1][1][row] = i
    for block, rows in runs:
        if block is None:
            continue
        src = np.array(list(rows.values()))
        at = np.array(list(rows.keys()))
        others = np.setdiff1d(np.arange(page), at)
        for h in range(hkv):
            x = new[src, h].astype(f32)
            mag = np.abs(x)
            a = mag[np.isfinite(mag)].max(initial=f32(0))
            held = f32(0) if 0 in rows else f32(scales[block, h])
            now = max(held, f32(a) / f32(127), LEAST)
            inv, ratio = f32(1) / now, held / now
            with np.errstate(invalid="ignore", over="ignore"):
                c = np.rint(x * inv)
            c = np.clip(np.where(np.isnan(c), 0, c), -127, 127)
            if 0 not in rows and now > held:
                old = pool[block, h, others].astype(f32)
                pool[block, h, others] = np.rint(old * ratio).astype(np.int8)
            pool[block, h, at] = c.astype(np.int8)
            scales[block, h] = now
    return pool, scales


def attend(q, k_pool, v_pool, k_scales, v_scales, table, lens):
    """(out, room): decode attention in 64 bits, and for each output how far a
    float32 evaluation may be off before its last rounding.

    With u = 2^-24: a score is a sum of D products of float32 (the code's
    product with q is exact or rounded once), scaled twice: off by at most
    (D + 4) u sum|q k| sd, and its exponential's argument by another 2 u |s| in
    log2 units and back - (D + 8) u sum|q k| sd together, e. Each weight is
    then off by a factor of 1 +- (e + 4 u) (the exponential itself). T terms are
    summed in chains of at most T. Numerator and denominator both: twice. The
    result is relative to the weighted sum of |v|. What the weights' parts may
    leave out (PARTS below) is not in it: the caller adds that."""
    b, hq, d = q.shape
    nb, hkv, page, _ = k_pool.shape
    out = np.zeros((b, hq, d))
    room = np.zeros((b, hq, d))
    u = 2.0 ** -24
    for bi in range(b):
        n = int(lens[bi])
        t = np.arange(n)
        ids = table[bi, t // page]
        ok = (ids >= 0) & (ids < nb)
        t, ids = t[ok], ids[ok]
        if not len(t):
            continue
        for h in range(hq):
            kv = h // (hq // hkv)
            k = k_pool[ids, kv, t % page].astype(np.float64) * k_scales[ids, kv][:, None]
            v = v_pool[ids, kv, t % page].astype(np.float64) * v_scales[ids, kv][:, None]
            x = q[bi, h].astype(np.float64)
            s = k @ x / math.sqrt(d)
            e = (d + 8) * u * (np.abs(k) @ np.abs(x)).max() / math.sqrt(d)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[bi, h] = p @ v
            room[bi, h] = (2 * (e + 4 * u) + 2 * (len(t) + 16) * u) * (p @ np.abs(v))
    return out, room


def half_step(dtype):
    """Half a rounding step of a torch type, relative to the value."""
    import torch
    return torch.finfo(dtype).eps / 2


#: what the weights' parts may leave out, relative to the weighted sum of |v|
#: (three parts of 8 bits, truncated, leave out 2^-23 at most: the half types'
#: 2^-15, of two parts, is wider than they need)
PARTS = {"torch.bfloat16": 2.0 ** -15, "torch.float16": 2.0 ** -15, "torch.float32": 2.0 ** -22}
