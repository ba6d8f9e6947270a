"""Attention over the 8-bit cache at the sizes of serving batches: its splits
into equal segments over all rows, which hold the ends and starts of several,
and into 128 tokens of one row; the combine of four heads a workgroup. Each
case is checked to reach the split it is there for. Every output is compared
with the formula in 64 bits.

Two kinds of values. `random` ones have scores of a spread of about 1.5.
`counted` ones are a number in the dim that the token's position gives (t mod
D), 0 elsewhere, and nearly equal weights: an output counts a row's tokens of
one position class, so a token lost, taken twice or of another row shows.

How far float32 arithmetic may be off, with u = 2^-24 and relative to the
weighted sum of |v|: a score (D products, exact or rounded once, two scalings,
the exponential's argument) is off by e = (D + 8) u sum|q k| / sqrt(D), its
weight by e + 4 u; each term of the sums is rounded with at most 4 times a
piece's tokens (three parts of a weight, a rescale) and the pieces and 32 of
the folds; numerator and denominator both, so twice. The weights go in as
three parts, with 2^-22 left out at most. Then half a step of the output."""

import math

import numpy as np
import pytest
import torch

import fusedtok_amd as ft
from tests import cache8_refs as refs
from tests import cache8_split as sp
from tests.cache8_split_cases import CASES, check_reached
from tests.test_gpu_cache8 import dev, i32, paged

pytestmark = pytest.mark.gpu

TYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = 2.0 ** -24


def attend64(q, cache, table, lens, chain):
    """(out, room) [B, Hq, D] float64 on the GPU; chain: the roundings of a
    term of the sums."""
    kp, vp, ks, vs = cache
    (b, hq, d), (nb, hkv, page, _) = q.shape, kp.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    room = torch.zeros_like(out)
    for i, n in enumerate(lens):
        t = torch.arange(n, device=q.device)
        ids = table[i].long()[t // page]
        ok = (ids >= 0) & (ids < nb)
        t, ids = t[ok], ids[ok]
        if not t.numel():
            continue

        def rows(pool, scales):   # [hkv, tokens, d]
            x = pool[ids, :, t % page].double() * scales[ids].double()[..., None]
            return x.transpose(0, 1).contiguous()

        k, v = rows(kp, ks), rows(vp, vs)
        x = q[i].double().view(hkv, hq // hkv, d).transpose(1, 2).contiguous()
        s = torch.bmm(k, x) / math.sqrt(d)
        e = (d + 8) * U * torch.bmm(k.abs(), x.abs()).amax(1) / math.sqrt(d)   # [hkv, group]
        p = torch.softmax(s, dim=1).transpose(1, 2).contiguous()
        out[i] = torch.bmm(p, v).view(hq, d)
        off = 2 * (e + 4 * U) + 2 * chain * U + 2.0 ** -22
        room[i] = (off[..., None] * torch.bmm(p, v.abs())).view(hq, d)
    return out, room


def counted(cache, table, lens):
    """The cache with its V values by position."""
    kp, vp, ks, vs = cache
    page, d = vp.shape[2:]
    vp = np.zeros_like(vp)
    for row, n in zip(table, lens):
        t = np.arange(n)
        vp[row[t // page], :, t % page, t % d] = 50 + t[:, None] % 71
    return kp, vp, ks, vs


@pytest.mark.parametrize("kind", ["random", "counted"])
@pytest.mark.parametrize("name,dtype", [(n, t) for n, c in CASES.items() for t in c.dtypes.split()])
def test_split(name, dtype, kind):
    c, dtype = CASES[name], TYPE[dtype]
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    launches = sp.split(c.lens, c.hkv, c.group, c.page, c.width, c.d, cus)
    check_reached(c, launches)
    rng = np.random.default_rng(len(name) + c.d)
    b, hq = len(c.lens), c.hkv * c.group
    cache, table = paged(rng, b, c.hkv, c.page, c.d, c.lens)
    if kind == "counted":
        cache = counted(cache, table, c.lens)
    assert table.shape[1] == c.width
    if c.holes:
        out_of = rng.choice([-1, cache[0].shape[0], -2 ** 31, 2 ** 31 - 1], table.shape)
        table = np.where(rng.random(table.shape) < 0.05, out_of, table).astype(np.int32)
        table[5] = -1
    q = rng.standard_normal((b, hq, c.d)) * (0.6 if kind == "random" else 0.05)
    q = dev(q, dtype)
    cache = [dev(x) for x in cache]
    table = i32(table)
    got = ft.attention_decode_paged_int8(q, *cache, table, None if c.whole else i32(c.lens))
    again = ft.attention_decode_paged_int8(q, *cache, table, None if c.whole else i32(c.lens))
    assert torch.equal(got, again)
    chain = max(4 * a.seg + max(a.pieces) for a in launches) + 32
    want, room = attend64(q, cache, table, c.lens, chain)
    room += refs.half_step(dtype) * want.abs()
    if dtype is torch.float16:
        room += 2.0 ** -25   # half a step of its smallest numbers
    off = (got.double() - want).abs()
    bad = off > room
    assert got.isfinite().all()
    assert not bad.any(), (float(off[bad].max()), float(room[bad].min()),
                           bad.nonzero()[:5].tolist(), int(bad.sum()))
    for i, n in enumerate(c.lens):
        assert n or not got[i].any()


def test_a_lost_token_shows():
    """The bound of the counted values notices one token less in the longest
    row (in the oracle, on the same inputs)."""
    c = CASES["ragged_128"]
    rng = np.random.default_rng(5)
    cache, table = paged(rng, len(c.lens), c.hkv, c.page, c.d, c.lens)
    cache = [dev(x) for x in counted(cache, table, c.lens)]
    q = dev(rng.standard_normal((len(c.lens), c.hkv * c.group, c.d)) * 0.05)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    (a,) = sp.split(c.lens, c.hkv, c.group, c.page, c.width, c.d, cus)
    chain = 4 * a.seg + max(a.pieces) + 32
    row = int(np.argmax(c.lens))
    lens = [n if i == row else 0 for i, n in enumerate(c.lens)]
    want, room = attend64(q, cache, i32(table), lens, chain)
    lens[row] -= 1
    less, _ = attend64(q, cache, i32(table), lens, chain)
    d = (c.lens[row] - 1) % c.d
    assert ((less - want).abs() > 2 * room)[row, :, d].all()
