"""GPU tests of qk_norm_rope and qk_norm_rope_kv_append_paged against a plain
form in 64 bits (step_refs).

The bound. Half a step of the output's type, relative to the value, once; and
the float32 arithmetic, relative to the pair's length L (a pair (a, b) of
normed values, |a'| <= L): the sum of D squares in up to D/16 + 6 sequential
adds, at most 2^-24 each, halved by the root: (D/32 + 3) 2^-24; mean, eps,
root, reciprocal, its product with the weight and with x: 6 * 2^-24; the
cosine and sine 1.5 * 2^-24 each and what the two fused operations round,
2 * 2^-24 - in all under (D/32 + 14) 2^-24 L. The angle's own error is below
2^-52 * (position * 2) and counts from positions of 2^27 on."""

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


def near(got, want, dtype, d, far=0):
    got, want = got.double().cpu().numpy(), np.asarray(want)
    # a pair's length is at most the head's largest value times sqrt(2)
    length = np.abs(want).max(-1, keepdims=True) * np.sqrt(2) * np.sqrt(2)
    bound = (torch.finfo(dtype).eps / 2 * np.abs(want) +
             ((d / 32 + 14) * 2.0 ** -24 + far * 2.0 ** -51) * length)
    if dtype is torch.float16:
        bound = bound + 2.0 ** -25   # half a step of the least numbers
    over = np.abs(got - want) - bound
    assert got.shape == want.shape and over.max(initial=-1) <= 0, over.max()


def inputs(seed, t, hq, hkv, d, dtype, axes=1, far=5000, pad=0):
    rng = np.random.default_rng(seed)
    width = (hq + 2 * hkv) * d
    wide = dev(rng.standard_normal((t, width + pad)) * 3, dtype)
    w = [(rng.standard_normal(d) * 0.3 + 1).astype(np.float32) for _ in range(2)]
    pos = rng.integers(0, far, (axes, t)).astype(np.int32)
    return wide[:, :width], w, pos


def check(t, hq, hkv, d, dtype, *, rot=None, theta=1e4, neox=True, norm=True, sections=None,
          far=5000, pad=0, seed=0):
    axes = len(sections) if sections else 1
    qkv, w, pos = inputs(seed, t, hq, hkv, d, dtype, axes, far, pad)
    got = ft.qk_norm_rope(qkv, hq, hkv, dev(w[0]) if norm else None, dev(w[1]) if norm else None,
                          dev(pos if sections else pos[0]), sections=sections, theta=theta,
                          rotary_dim=rot, eps=1e-5, neox=neox)
    want = refs.qk_norm_rope(qkv.double().cpu().numpy(), hq, hkv, w[0] if norm else None,
                             w[1] if norm else None, pos, rot or d, theta, 1e-5, neox, sections)
    for g, e in zip(got, want):
        assert g.is_contiguous()
        near(g, e, dtype, d, far)
    assert torch.equal(got[2].reshape(t, -1), qkv[:, -hkv * d:])   # v is copied


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [2, 6, 16, 64, 80, 96, 128, 256, 510, 512])
def test_head_sizes(d, dtype, neox):
    check(9, 4, 2, d, dtype, neox=neox)


@pytest.mark.parametrize("t,hq,hkv", [(1, 1, 1), (1, 32, 8), (7, 40, 1), (64, 32, 8), (2500, 3, 1),
                                      (9001, 2, 1), (5, 70, 70)])
def test_tokens_and_heads(t, hq, hkv):
    check(t, hq, hkv, 128, torch.bfloat16)
    check(t, hq, hkv, 64, torch.float32, neox=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rot", [(128, 64), (96, 48), (64, 2), (80, 24), (128, 126), (10, 6)])
@pytest.mark.parametrize("neox", [True, False])
def test_part_of_a_head(d, rot, dtype, neox):
    check(11, 3, 1, d, dtype, rot=rot, neox=neox)


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("sections", [[64], [16, 24, 24], [0, 64], [1, 62, 1], [10, 20, 30, 4]])
def test_axes(sections, neox):
    check(33, 4, 2, 128, torch.float32, sections=sections, neox=neox)
    check(33, 4, 2, 128, torch.float16, sections=sections, neox=neox)


@pytest.mark.parametrize("far", [10, 1000000, 2 ** 31 - 1])
def test_far_positions(far):
    check(50, 2, 1, 128, torch.float32, far=far, theta=1e6)


def test_negative_positions_turn_back():
    """A turn by -p undoes one by p."""
    qkv, _, pos = inputs(3, 40, 2, 1, 64, torch.float32)
    q, k, v = ft.qk_norm_rope(qkv, 2, 1, None, None, dev(pos[0]))
    again = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    q, k, _ = ft.qk_norm_rope(again, 2, 1, None, None, dev(-pos[0]))
    back = torch.cat([q.flatten(1), k.flatten(1)], 1)
    # two turns' roundings, and the length of a pair
    assert (back - qkv[:, :192]).abs().max() <= 2 * 8 * 2.0 ** -24 * 2 * qkv.abs().max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [1, 8, 63])
def test_rows_inside_wider_ones(pad, dtype):
    check(17, 4, 2, 96, dtype, pad=pad)
    check(17, 4, 2, 96, dtype, pad=pad, norm=False, neox=False)


def test_weights_of_other_types_and_no_tokens():
    qkv, w, pos = inputs(1, 6, 2, 1, 64, torch.bfloat16)
    w16 = [dev(x, torch.bfloat16) for x in w]
    a = ft.qk_norm_rope(qkv, 2, 1, *w16, dev(pos[0]))
    b = ft.qk_norm_rope(qkv, 2, 1, *(x.float() for x in w16), dev(pos[0]))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    q, k, v = ft.qk_norm_rope(qkv[:0], 2, 1, *w16, dev(pos[0, :0]))
    assert q.shape == (0, 2, 64) and k.shape == v.shape == (0, 1, 64)


def test_a_row_of_nan_stays_alone():
    qkv, w, pos = inputs(2, 5, 2, 1, 64, torch.float32)
    clean = ft.qk_norm_rope(qkv, 2, 1, dev(w[0]), dev(w[1]), dev(pos[0]))
    qkv[2, 70] = float("nan")   # q head 1 of token 2
    got = ft.qk_norm_rope(qkv, 2, 1, dev(w[0]), dev(w[1]), dev(pos[0]))
    assert got[0][2, 1].isnan().all()
    got[0][2, 1] = clean[0][2, 1]
    assert all(torch.equal(x, y) for x, y in zip(got, clean))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page", [(64, 16), (128, 24), (96, 1), (6, 5)])
@pytest.mark.parametrize("t", [1, 70, 5000])
def test_into_a_paged_cache(t, d, page, dtype):
    hq, hkv, nb = 4, 2, -(-t // page) + 3
    qkv, w, pos = inputs(t + d, t, hq, hkv, d, dtype)
    w = [dev(x) for x in w]
    rng = np.random.default_rng(t)
    slots = rng.permutation(nb * page)[:t].astype(np.int32)
    slots[t // 2 + 1::7] = rng.choice([-1, -2 ** 31, nb * page, 2 ** 31 - 1])
    pools = [dev(rng.standard_normal((nb, hkv, page, d)), dtype) for _ in range(2)]
    want = [p.clone() for p in pools]
    q, k, v = ft.qk_norm_rope(qkv, hq, hkv, *w, dev(pos[0]), neox=True)
    held = (slots >= 0) & (slots < nb * page)
    at = dev(slots[held]).long()
    for p, x in zip(want, (k, v)):
        p[at // page, :, at % page] = x[dev(held)]
    got = ft.qk_norm_rope_kv_append_paged(qkv, hq, hkv, *w, dev(pos[0]), *pools, dev(slots),
                                          neox=True)
    assert torch.equal(got, q)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_equals_the_framework_own_steps():
    """Without weights: rope_kv_append_paged's q and pools, within the bound
    of one rounding step (that op turns in float64)."""
    b, hq, hkv, d, page = 5, 8, 2, 128, 16
    qkv, _, _ = inputs(9, b, hq, hkv, d, torch.float32)
    table = torch.arange(b * 4, device=DEV, dtype=torch.int32).view(b, 4)
    lens = torch.tensor([0, 15, 16, 40, 63], device=DEV, dtype=torch.int32)
    pools = [torch.zeros(b * 4, hkv, page, d, device=DEV) for _ in range(4)]
    q0 = ft.rope_kv_append_paged(qkv, hq, hkv, *pools[:2], table, lens, neox=True)
    slots = table.gather(1, (lens // page).long()[:, None])[:, 0] * page + lens % page
    q1 = ft.qk_norm_rope_kv_append_paged(qkv, hq, hkv, None, None, lens, *pools[2:],
                                         slots.int(), neox=True)
    for a, c in ((q0, q1), (pools[0], pools[2])):
        assert (a - c).abs().max() <= 8 * 2.0 ** -24 * 2 * qkv.abs().max()
    assert torch.equal(pools[1], pools[3])


def test_on_another_stream_and_in_a_graph():
    qkv, w, pos = inputs(4, 64, 8, 2, 128, torch.bfloat16)
    w, pos = [dev(x) for x in w], dev(pos[0])
    pools = [torch.zeros(8, 2, 16, 128, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    slots = torch.randperm(128, device=DEV)[:64].int()
    want = ft.qk_norm_rope_kv_append_paged(qkv, 8, 2, *w, pos, *pools, slots)
    kept = [p.clone() for p in pools]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ft.qk_norm_rope_kv_append_paged(qkv, 8, 2, *w, pos, *pools, slots)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ft.qk_norm_rope_kv_append_paged(qkv, 8, 2, *w, pos, *pools, slots)
    for turn in range(3):
        for p in pools:
            p.zero_()
        got.zero_()
        pos.add_(turn)   # other positions for the second and third replay
        graph.replay()
        torch.cuda.synchronize()
        fresh = [torch.zeros_like(p) for p in pools]
        want = ft.qk_norm_rope_kv_append_paged(qkv, 8, 2, *w, pos, *fresh, slots)
        assert torch.equal(got, want)
        assert all(torch.equal(a, b) for a, b in zip(pools, fresh))
        assert turn or all(torch.equal(a, b) for a, b in zip(pools, kept))


def test_refusals():
    qkv, w, pos = inputs(0, 4, 2, 1, 64, torch.float32)
    w, pos = [dev(x) for x in w], dev(pos[0])
    f = ft.qk_norm_rope
    for bad, exc, word in [
            (lambda: f(qkv, 3, 1, *w, pos), ValueError, "qkv must be"),
            (lambda: f(qkv, 0, 1, *w, pos), ValueError, "heads"),
            (lambda: f(qkv.double(), 2, 1, *w, pos), TypeError, "float32"),
            (lambda: f(qkv.cpu(), 2, 1, *w, pos), TypeError, "GPU"),
            (lambda: f(qkv.t(), 2, 1, *w, pos), ValueError, "contiguous"),
            (lambda: f(qkv, 2, 1, w[0], None, pos), ValueError, "together"),
            (lambda: f(qkv, 2, 1, w[0][:3], w[1], pos), ValueError, "D entries"),
            (lambda: f(qkv, 2, 1, *w, pos.long()), TypeError, "int32"),
            (lambda: f(qkv, 2, 1, *w, pos[:3]), ValueError, "positions"),
            (lambda: f(qkv, 2, 1, *w, pos.cpu()), TypeError, "positions"),
            (lambda: f(qkv, 2, 1, *w, pos, sections=[16, 16]), ValueError, "sections"),
            (lambda: f(qkv, 2, 1, *w, pos, sections=[31]), ValueError, "sum"),
            (lambda: f(qkv, 2, 1, *w, pos.repeat(2, 1)), ValueError, "sections"),
            (lambda: f(qkv, 2, 1, *w, pos.repeat(2, 1), sections=[16, 17]), ValueError, "sum"),
            (lambda: f(qkv, 2, 1, *w, pos.repeat(2, 1), sections=[33, -1]), ValueError,
             "sections must"),
            (lambda: f(qkv, 2, 1, *w, pos.repeat(5, 1), sections=[8, 8, 8, 4, 4]), ValueError,
             "axes"),
            (lambda: f(qkv, 2, 1, *w, pos, rotary_dim=66), ValueError, "rotary_dim"),
            (lambda: f(qkv, 2, 1, *w, pos, rotary_dim=7), ValueError, "rotary_dim"),
            (lambda: f(qkv, 2, 1, *w, pos, theta=0.0), ValueError, "theta"),
            (lambda: f(qkv, 2, 1, *w, pos, eps=-1.0), ValueError, "eps")]:
        with pytest.raises(exc, match=word):
            bad()
    g = ft.qk_norm_rope_kv_append_paged
    pool = torch.zeros(2, 1, 16, 64, device=DEV)
    other, slots = torch.zeros_like(pool), torch.zeros(4, device=DEV, dtype=torch.int32)
    for bad, exc, word in [
            (lambda: g(qkv, 2, 1, *w, pos, pool, pool, slots), ValueError, "own"),
            (lambda: g(qkv, 2, 1, *w, pos, pool, other.half(), slots), TypeError, "dtype"),
            (lambda: g(qkv, 2, 1, *w, pos, pool, other[:1], slots), ValueError, "pools"),
            (lambda: g(qkv, 2, 1, *w, pos, pool[..., :32], other[..., :32], slots), ValueError,
             "pools"),
            (lambda: g(qkv, 2, 1, *w, pos, pool, other, slots[:2]), ValueError, "slots"),
            (lambda: g(qkv, 2, 1, *w, pos, pool, other, slots.long()), TypeError, "slots")]:
        with pytest.raises(exc, match=word):
            bad()
