"""The 8-bit paged cache on the host: the C entry points refuse bad arguments
before any HIP call, and the plain forms that the GPU is tested against hold
what the definitions say."""

import ctypes
import os

import numpy as np
import pytest
import torch  # noqa: F401  (HIP runtime first: the library binds to it)

import fusedtok_amd as ft
from tests import cache8_refs as refs

LIB = os.path.join(os.path.dirname(ft.__file__), "libfusedtok_amd.so")
FT_OK, FT_EINVAL = 0, 1
P, I, L, U = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    lib.ft_last_error.restype = ctypes.c_char_p
    lib.ft_block_table_extend_launch.argtypes = [P, P, P, P, I] + [P] * 6 + [I] * 4 + [U]
    lib.ft_kv_append_paged_int8_launch.argtypes = [P, P, I] + [P] * 5 + [I] * 5 + [U]
    lib.ft_attention_decode_paged_int8_workspace.argtypes = [I] * 7 + [P]
    lib.ft_attention_decode_paged_int8_launch.argtypes = [P, I] + [P] * 8 + [L] + [I] * 7 + [U]
    return lib


X = 64  # a pointer that is never followed: every call here is refused


@pytest.mark.parametrize("change,word", [
    (dict(batch=-1), b"batch"), (dict(batch=4097), b"batch"), (dict(page=0), b"page"),
    (dict(width=-1), b"width"), (dict(tokens=-1), b"tokens"), (dict(free_len=-1), b"page"),
    (dict(page=1024, width=2 ** 21), b"capacity"), (dict(n_free=0), b"null"),
    (dict(table=0), b"null"), (dict(free=0), b"null"), (dict(slots=0), b"null")])
def test_extend_refusals(lib, change, word):
    a = dict(table=X, free=X, free_len=3, n_free=X, slots=X, batch=2, page=16, width=4, tokens=5)
    a.update(change)
    st = lib.ft_block_table_extend_launch(a["table"], X, X, a["free"], a["free_len"], a["n_free"],
                                          a["slots"], X, X, X, X, a["batch"], a["page"],
                                          a["width"], a["tokens"], 0)
    assert st == FT_EINVAL and word in lib.ft_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(dim=6), b"multiple of 4"), (dict(dim=516), b"512"), (dict(page=0), b"page"),
    (dict(page=1025), b"page"), (dict(hkv=0), b"heads"), (dict(tokens=-1), b"tokens"),
    (dict(dtype=7), b"type"), (dict(blocks=2 ** 28), b"31 bits"),
    (dict(blocks=2 ** 26, hkv=64), b"32 bits"), (dict(k=0), b"null"), (dict(k=X + 2), b"aligned"),
    (dict(pool=X + 1), b"aligned")])
def test_append_refusals(lib, change, word):
    a = dict(k=X, dtype=1, pool=X, tokens=3, hkv=2, dim=64, blocks=4, page=16)
    a.update(change)
    st = lib.ft_kv_append_paged_int8_launch(a["k"], X, a["dtype"], X, a["pool"], X, X, X,
                                            a["tokens"], a["hkv"], a["dim"], a["blocks"],
                                            a["page"], 0)
    assert st == FT_EINVAL and word in lib.ft_last_error()


def test_append_of_more_rows_than_are_counted(lib):
    """Rows and heads whose (run, head, pool) triples pass 31 bits."""
    f = lib.ft_kv_append_paged_int8_launch
    assert f(X, X, 1, X, X, X, X, X, 1024, 2 ** 20, 4, 1024, 1, 0) == FT_EINVAL
    assert b"too many rows" in lib.ft_last_error()


def test_append_of_nothing(lib):
    f = lib.ft_kv_append_paged_int8_launch
    assert f(None, None, 1, None, None, None, None, None, 0, 2, 64, 4, 16, 0) == FT_OK
    assert f(None, None, 1, None, None, None, None, None, 3, 2, 64, 0, 16, 0) == FT_OK


@pytest.mark.parametrize("change,word", [
    (dict(hq=5), b"multiple"), (dict(dim=30), b"multiple of 4"), (dict(page=2000), b"page"),
    (dict(batch=-1), b"batch"), (dict(page=1024, width=2 ** 21), b"capacity")])
def test_attention_refusals(lib, change, word):
    a = dict(batch=2, hq=8, hkv=2, page=16, width=4, dim=64)
    a.update(change)
    got = ctypes.c_longlong(-1)
    st = lib.ft_attention_decode_paged_int8_workspace(1, a["batch"], a["hq"], a["hkv"], a["page"],
                                                      a["width"], a["dim"], ctypes.byref(got))
    assert st == FT_EINVAL and word in lib.ft_last_error() and got.value == -1
    st = lib.ft_attention_decode_paged_int8_launch(X, 1, X, X, X, X, X, X, X, X, 1 << 40,
                                                   a["batch"], a["hq"], a["hkv"], 4, a["page"],
                                                   a["width"], a["dim"], 0)
    assert st == FT_EINVAL and word in lib.ft_last_error()


def test_attention_of_too_many_heads_without_a_block(lib):
    st = lib.ft_attention_decode_paged_int8_launch(X, 1, 0, 0, 0, 0, X, X, X, X, 1 << 40, 2 ** 21,
                                                   1024, 8, 0, 16, 4, 64, 0)
    assert st == FT_EINVAL and b"too large" in lib.ft_last_error()


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 64)
    pool, scale = torch.zeros(1, 2, 16, 64, dtype=torch.int8), torch.zeros(1, 2)
    with pytest.raises(TypeError, match="GPU"):
        ft.attention_decode_paged_int8(x, pool, pool, scale, scale, [[0]], [1])
    with pytest.raises(TypeError, match="GPU"):
        ft.kv_append_paged_int8(pool, pool, scale, scale, x, x, torch.zeros(1, dtype=torch.int32))
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TypeError, match="GPU"):
        ft.block_table_extend(i.view(1, 1), i, i, i, i, 16, 1)


class On:
    """A stand-in for a tensor on a device."""

    def __init__(self, device):
        self.device = device

    def get_device(self):
        return self.device


def test_operands_of_two_devices(monkeypatch):
    monkeypatch.setattr(ft, "_current_device", lambda: 1)
    assert ft._one_device("ab", (On(1), On(1)))
    assert not ft._one_device("ab", (On(0), On(0)))   # another than the current one
    with pytest.raises(ValueError, match="a on 0, b on 1"):
        ft._one_device("ab", (On(0), On(1)))


# ---- the plain forms --------------------------------------------------------


def test_plain_extend_by_hand():
    table, slots, pos, off, lens, left = refs.extend(
        np.zeros((2, 3), np.int32), [3, 0], [2, 1], [7, 8, 9], 3, 4, 4)
    assert table.tolist() == [[0, 9, 0], [8, 0, 0]]
    assert slots.tolist() == [3, 36, 32, -1] and pos.tolist() == [3, 4, 0, 0]
    assert off.tolist() == [0, 2, 3] and lens.tolist() == [5, 1] and left.tolist() == [1]


def test_plain_append_by_hand():
    pool, scales = np.full((2, 1, 2, 4), 100, np.int8), np.ones((2, 1), np.float32)
    new = np.array([[[0, 127, -254, 63.5]]], np.float32)
    codes, s = refs.append(pool, scales, new, [3])   # block 1, row 1: the scale doubles
    assert s[:, 0].tolist() == [1, 2]
    assert codes[1, 0].tolist() == [[50, 50, 50, 50], [0, 64, -127, 32]]
    codes, s = refs.append(pool, scales, new / 256, [2])   # row 0: starts over
    assert codes[1, 0].tolist() == [[0, 64, -127, 32], [100] * 4] and s[1, 0] == 2.0 ** -7
    assert (codes[0] == pool[0]).all()


def test_plain_attend_is_a_mean_for_equal_scores():
    rng = np.random.default_rng(0)
    vp = rng.integers(-127, 128, (3, 1, 4, 8)).astype(np.int8)
    ones = np.ones((3, 1), np.float32)
    out, room = refs.attend(np.zeros((1, 2, 8), np.float32), vp, vp, ones, ones * 0.5,
                            np.array([[2, -1, 0]]), [10])
    want = np.concatenate([vp[2, 0], vp[0, 0, :2]]).astype(float).mean(0) / 2
    np.testing.assert_allclose(out[0, 0], want, rtol=1e-12)
    assert (room > 0).all() and room.max() < 1e-2
