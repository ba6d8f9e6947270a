"""The head norms with rotation, the shared-prefix attention and the filtered
sampling on the host: the C entry points refuse bad arguments before any HIP
call, host tensors are refused, and the plain forms that the GPU is tested
against hold what the definitions say."""

import ctypes
import os

import numpy as np
import pytest
import torch  # noqa: F401  (HIP runtime first: the library binds to it)

import fusedtok_amd as ft
from tests import step_refs as refs

LIB = os.path.join(os.path.dirname(ft.__file__), "libfusedtok_amd.so")
FT_OK, FT_EINVAL = 0, 1
P, I, L, U, F, D = (ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t,
                    ctypes.c_float, ctypes.c_double)


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    lib.ft_last_error.restype = ctypes.c_char_p
    lib.ft_qk_norm_rope_launch.argtypes = ([P, I, L, P, P, P, I, P, I, D, F, I, P, P, P] + [I] * 4 +
                                           [U])
    lib.ft_qk_norm_rope_kv_append_paged_launch.argtypes = (
        [P, I, L, P, P, P, I, P, I, D, F, I, P, P, P, P] + [I] * 6 + [U])
    lib.ft_attention_decode_paged_prefix_workspace.argtypes = [I] * 9 + [P]
    lib.ft_attention_decode_paged_prefix_launch.argtypes = ([P, I] + [P] * 9 + [L] + [I] * 9 + [U])
    lib.ft_sample_filtered_batched_workspace.argtypes = [I, I, P]
    lib.ft_sample_filtered_batched_launch.argtypes = [P, I, L, I, I, P, P, F, P, I, P, F, P, F, P, P,
                                                      L, U]
    return lib


X = 64  # a pointer that is never followed: every call here is refused


@pytest.mark.parametrize("change,word", [
    (dict(dtype=3), b"type"), (dict(tokens=-1), b"tokens"), (dict(hq=0), b"heads"),
    (dict(dim=63), b"even"), (dict(dim=514, ld=10 ** 6), b"512"), (dict(rot=0), b"rotary_dim"),
    (dict(rot=66), b"rotary_dim"), (dict(rot=31), b"rotary_dim"), (dict(theta=0.0), b"theta"),
    (dict(theta=float("inf")), b"theta"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"),
    (dict(axes=0), b"axes"), (dict(axes=5), b"axes"), (dict(axes=2, sections=0), b"sections"),
    (dict(axes=2, sections=(16, 17)), b"sum"), (dict(axes=2, sections=(40, -8)), b"sum"),
    (dict(axes=2, sections=(-8, 40)), b">= 0"), (dict(axes=2, sections=(2 ** 31 - 1, 1)), b"sum"),
    (dict(ld=383), b"stride"), (dict(hq=2 ** 30), b"heads"), (dict(qw=0), b"together"),
    (dict(qkv=0), b"null"), (dict(pos=0), b"null"), (dict(q=0), b"null"), (dict(k=0), b"null")])
def test_qk_refusals(lib, change, word):
    a = dict(qkv=X, dtype=1, ld=384, qw=X, kw=X, pos=X, axes=1, sections=0, rot=64, theta=1e4,
             eps=1e-6, q=X, k=X, tokens=3, hq=4, hkv=1, dim=64)
    a.update(change)
    sec = (ctypes.c_int * len(a["sections"]))(*a["sections"]) if a["sections"] else 0
    st = lib.ft_qk_norm_rope_launch(a["qkv"], a["dtype"], a["ld"], a["qw"], a["kw"], a["pos"],
                                    a["axes"], sec, a["rot"], a["theta"], a["eps"], 1, a["q"],
                                    a["k"], X, a["tokens"], a["hq"], a["hkv"], a["dim"], 0)
    assert st == FT_EINVAL and word in lib.ft_last_error()


@pytest.mark.parametrize("change,word", [(dict(blocks=-1), b"blocks"), (dict(page=0), b"page"),
                                         (dict(slots=0), b"null"), (dict(pool=0), b"null")])
def test_qk_append_refusals(lib, change, word):
    a = dict(blocks=4, page=16, slots=X, pool=X)
    a.update(change)
    st = lib.ft_qk_norm_rope_kv_append_paged_launch(X, 1, 384, X, X, X, 1, 0, 64, 1e4, 1e-6, 1, X,
                                                    a["pool"], X, a["slots"], 3, 4, 1, 64,
                                                    a["blocks"], a["page"], 0)
    assert st == FT_EINVAL and word in lib.ft_last_error()


def test_qk_of_nothing(lib):
    assert lib.ft_qk_norm_rope_launch(0, 1, 384, 0, 0, 0, 1, 0, 64, 1e4, 1e-6, 1, 0, 0, 0, 0, 4, 1,
                                      64, 0) == FT_OK


@pytest.mark.parametrize("change,word", [
    (dict(dtype=9), b"type"), (dict(batch=-1), b"batch"), (dict(hq=0), b"heads"),
    (dict(hq=5), b"multiple"), (dict(groups=-1), b"groups"), (dict(dim=30), b"multiple of 4"),
    (dict(dim=516), b"512"), (dict(page=0), b"page"), (dict(pwidth=-1), b"widths"),
    (dict(page=1024, width=2 ** 20), b"capacity"), (dict(page=1024, pwidth=2 ** 20), b"capacity"),
    (dict(batch=4000, groups=97), b"4096"), (dict(batch=4000, hq=8192), b"too large")])
def test_prefix_refusals(lib, change, word):
    a = dict(dtype=1, batch=2, hq=8, hkv=2, groups=1, page=16, pwidth=4, width=4, dim=64)
    a.update(change)
    sizes = [a["batch"], a["hq"], a["hkv"], a["groups"]]
    got = ctypes.c_longlong(-1)
    st = lib.ft_attention_decode_paged_prefix_workspace(a["dtype"], *sizes, a["page"], a["pwidth"],
                                                        a["width"], a["dim"], ctypes.byref(got))
    assert st == FT_EINVAL and word in lib.ft_last_error() and got.value == -1
    st = lib.ft_attention_decode_paged_prefix_launch(X, a["dtype"], *[X] * 9, 1 << 40, *sizes, 4,
                                                     a["page"], a["pwidth"], a["width"], a["dim"],
                                                     0)
    assert st == FT_EINVAL and word in lib.ft_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(q=0), b"null"), (dict(k=0), b"null"), (dict(ptable=0), b"null"), (dict(table=0), b"null"),
    (dict(out=0), b"null"), (dict(groups=2, offsets=0), b"group_offsets"),
    (dict(blocks=-1), b"blocks"), (dict(q=X + 4), b"aligned"), (dict(k=X + 2), b"aligned"),
    (dict(out=X + 4), b"aligned"), (dict(ws=X + 8), b"aligned")])
def test_prefix_operand_refusals(lib, change, word):
    a = dict(q=X, k=X, ptable=X, offsets=X, table=X, out=X, ws=X, groups=1, blocks=4)
    a.update(change)
    st = lib.ft_attention_decode_paged_prefix_launch(
        a["q"], 1, a["k"], X, a["ptable"], X, a["offsets"], a["table"], X, a["out"], a["ws"],
        1 << 40, 2, 8, 2, a["groups"], a["blocks"], 16, 4, 4, 64, 0)
    assert st == FT_EINVAL and word in lib.ft_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(dtype=5), b"type"), (dict(rows=-1), b"rows"), (dict(n=0), b"empty"),
    (dict(n=2 ** 22 + 1), b"2^22"), (dict(rows=2 ** 26, n=2 ** 20), b"too many"),
    (dict(temp=-1.0), b"temperature"), (dict(temp=float("nan")), b"temperature"),
    (dict(k=-1), b"top_k"), (dict(p=0.0), b"top_p"), (dict(p=1.5), b"top_p"),
    (dict(p=float("nan")), b"top_p"), (dict(minp=-0.1), b"min_p"), (dict(minp=1.1), b"min_p"),
    (dict(ld=99), b"stride"), (dict(x=0), b"null"), (dict(u=0), b"null"), (dict(out=0), b"null"),
    (dict(n=40000, ld=40000, ws=0), b"workspace"), (dict(n=40000, ld=40000, room=100), b"workspace"),
    (dict(n=40000, ld=40000, ws=X + 8), b"aligned")])
def test_sample_refusals(lib, change, word):
    a = dict(x=X, dtype=0, ld=100, rows=3, n=100, u=X, temp=1.0, k=0, p=1.0, minp=0.0, out=X, ws=X,
             room=1 << 40)
    a.update(change)
    st = lib.ft_sample_filtered_batched_launch(a["x"], a["dtype"], a["ld"], a["rows"], a["n"],
                                               a["u"], 0, a["temp"], 0, a["k"], 0, a["p"], 0,
                                               a["minp"], a["out"], a["ws"], a["room"], 0)
    assert st == FT_EINVAL and word in lib.ft_last_error()


def test_sample_workspace(lib):
    got = ctypes.c_longlong(-1)
    for rows, n, none in ((5, 32768, True), (0, 70000, True), (5, 32769, False)):
        assert lib.ft_sample_filtered_batched_workspace(rows, n, ctypes.byref(got)) == FT_OK
        assert (got.value == 0) == none
    assert got.value >= 5 * 32769 * 4


def test_host_tensors_are_refused():
    x, i = torch.zeros(2, 8, 64), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(1, 2, 16, 64)
    with pytest.raises(TypeError, match="GPU"):
        ft.qk_norm_rope(x.view(2, -1), 4, 2, None, None, i)
    with pytest.raises(TypeError, match="GPU"):
        ft.qk_norm_rope_kv_append_paged(x.view(2, -1), 4, 2, None, None, i, pool, pool, i)
    with pytest.raises(TypeError, match="GPU"):
        ft.attention_decode_paged_prefix(x, pool, pool, [[0]], [1], [[0], [0]], [1, 1])
    with pytest.raises(TypeError, match="GPU"):
        ft.sample_filtered_batched(x[0], torch.zeros(8))


# ---- the plain forms --------------------------------------------------------


def test_plain_rotation_by_hand():
    x = np.array([[[1.0, 0.0, 2.0, 0.0]]])
    quarter = np.pi / 2
    # neox pairs (0, 2), (1, 3) by position * (1, theta^-0.5); theta huge: the second stays
    got = refs.turn(x, np.array([[quarter]]), 4, 1e300, True)
    np.testing.assert_allclose(got[0, 0], [-2, 0, 1, 0], atol=1e-15)
    got = refs.turn(x, np.array([[quarter]]), 2, 1e4, False)   # pair (0, 1) alone
    np.testing.assert_allclose(got[0, 0], [0, 1, 2, 0], atol=1e-15)
    got = refs.turn(x, np.array([[0.0], [quarter]]), 4, 1.0, False, [1, 1])
    np.testing.assert_allclose(got[0, 0], [1, 0, 0, 2], atol=1e-15)


def test_plain_norm_by_hand():
    qkv = np.array([[3.0, 4.0, 0.0, 2.0, 7.0, 9.0]])
    q, k, v = refs.qk_norm_rope(qkv, 1, 1, np.ones(2), np.full(2, 2.0), np.array([[0]]), 2, 1e4,
                                0.0, True)
    np.testing.assert_allclose(q[0, 0], np.array([3, 4]) / np.sqrt(12.5))
    np.testing.assert_allclose(k[0, 0], [0, 2 * np.sqrt(2)])
    assert v[0, 0].tolist() == [7, 9]


def test_plain_prefix_attention_is_a_mean_for_equal_scores():
    rng = np.random.default_rng(0)
    vp = rng.standard_normal((4, 1, 4, 8))
    out, _, _ = refs.attend_prefix(np.zeros((2, 2, 8)), vp, vp, np.array([[2, -1]]), [6],
                                   np.array([[0], [3]]), [1, 0], [0, 2])
    np.testing.assert_allclose(out[0, 0], np.concatenate([vp[2, 0], vp[0, 0, :1]]).mean(0))
    np.testing.assert_allclose(out[1, 1], vp[2, 0].mean(0))


def test_plain_sampling_by_hand():
    x = np.log(np.array([1.0, 4.0, 2.0, 4.0, 1.0]))
    draw = lambda u, **kw: refs.sample(x, u, **dict(dict(temp=1.0, k=0, p=1.0, minp=0.0), **kw))
    # shares 1, 4, 2, 4, 1 of 12 in the order of the indices
    assert [draw((i + 0.5) / 12) for i in range(12)] == [0] + [1] * 4 + [2] * 2 + [3] * 4 + [4]
    assert {draw((i + 0.5) / 8, k=2) for i in range(8)} == {1, 3}
    assert {draw((i + 0.5) / 8, k=1) for i in range(8)} == {1}          # the first of equals
    assert {draw((i + 0.5) / 8, p=0.3) for i in range(8)} == {1}        # 4 of 12 come to 0.3
    assert {draw((i + 0.5) / 8, p=0.4) for i in range(8)} == {1, 3}
    assert {draw((i + 0.5) / 30, minp=0.5) for i in range(30)} == {1, 2, 3}
    assert draw(0.99, temp=0.0) == 1
    assert refs.sample(np.full(3, -np.inf), 0.5, 1.0, 0, 1.0, 0.0) == -1
