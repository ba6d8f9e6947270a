"""Plain forms in 64 bits of the head norms with rotation, the shared-prefix
attention and the filtered sampling, written from their definitions."""

import numpy as np


def turn(x, pos, rot, theta, neox, sections=None):
    """x [T, heads, D] with its first rot values turned; pos [axes, T]."""
    half = rot // 2
    sections = sections or [half]
    axis = np.repeat(np.arange(len(sections)), sections)
    freq = np.power(np.longdouble(theta), np.arange(half, dtype=np.longdouble) * -2 / rot)
    angle = pos[axis].T.astype(np.longdouble) * freq
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    out = x.astype(np.longdouble).copy()
    lo = np.arange(half) if neox else 2 * np.arange(half)
    hi = lo + (half if neox else 1)
    a, b = x[..., lo], x[..., hi]
    out[..., lo], out[..., hi] = a * c - b * s, b * c + a * s
    return out.astype(np.float64)


def qk_norm_rope(qkv, hq, hkv, qw, kw, pos, rot, theta, eps, neox, sections=None):
    """q, k, v and, for each, the largest magnitude that a head's value may
    take (the norm's output), which roundings are relative to."""
    t = qkv.shape[0]
    x = qkv.astype(np.float64).reshape(t, hq + 2 * hkv, -1)
    parts = []
    for part, w in ((x[:, :hq], qw), (x[:, hq:hq + hkv], kw)):
        if w is not None:
            part = part / np.sqrt((part ** 2).mean(-1, keepdims=True) + eps) * w
        parts.append(turn(part, pos, rot, theta, neox, sections))
    return parts[0], parts[1], x[:, hq + hkv:]


def attend_prefix(q, k_pool, v_pool, ptable, plens, table, lens, offsets):
    """The attention's rows, and for each row the sums that its bound needs:
    the weighted magnitudes of V, and the largest magnitude of a score (in
    nats, before the sum over dims cancels)."""
    b, hq, d = q.shape
    nb, hkv, page, _ = k_pool.shape
    q, k_pool, v_pool = (x.astype(np.float64) for x in (q, k_pool, v_pool))
    out, mass, size = np.zeros_like(q), np.zeros_like(q), np.zeros((b, hq, 1))

    def rows(row, n):
        t = np.arange(min(max(int(n), 0), len(row) * page))
        e = np.asarray(row)[t // page]
        ok = (e >= 0) & (e < nb)
        return e[ok], t[ok] % page

    for x in range(b):
        e, o = rows(table[x], lens[x])
        for g in range(len(plens)):
            if offsets[g] <= x < offsets[g + 1]:
                pe, po = rows(ptable[g], plens[g])
                e, o = np.concatenate([pe, e]), np.concatenate([po, o])
        if not len(e):
            continue
        for h in range(hq):
            k, v = (p[e, h // (hq // hkv), o] for p in (k_pool, v_pool))
            s = k @ q[x, h] / np.sqrt(d)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[x, h], mass[x, h] = w @ v, w @ np.abs(v)
            size[x, h] = (np.abs(k) @ np.abs(q[x, h])).max() / np.sqrt(d)
    return out, mass, size


def sample(x, u, temp, k, p, minp):
    """One row's token (a Python int), from the definition: float64 weights as
    whole numbers, a full sort, exact sums."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return -1
    if not temp > 0:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore"):
        far = np.where(x == top, 0.0, (x - top) / np.float64(temp))
    w = np.rint(np.exp(far) * 2.0 ** 40)
    w = np.where(np.isnan(w), 0, w).astype(np.int64)
    order = np.lexsort((np.arange(len(x)), -x))
    if k > 0:
        order = order[:k]
    if p < 1:
        sums = np.cumsum(w[order])
        before = (sums - w[order]).astype(np.float64)
        keep = before < np.float64(p) * np.float64(sums[-1])
        keep[0] = True
        order = order[keep]
    kept = np.sort(order[w[order] >= min(float(minp), 1.0) * 2.0 ** 40])
    sums = np.cumsum(w[kept])
    aim = int(np.float64(u) * np.float64(sums[-1])) if u > 0 else 0
    aim = min(aim, int(sums[-1]) - 1)
    return int(kept[np.searchsorted(sums, aim, side="right")])
