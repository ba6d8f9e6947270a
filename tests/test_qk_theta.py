"""The bases that qk_norm_rope takes: theta from 2^-10 on, so that no angle is
beyond what its reduction to a quarter turn holds; refused below, on the host
before any HIP call."""

import ctypes
import os

import numpy as np
import pytest
import torch

import fusedtok_amd as ft

LIB = os.path.join(os.path.dirname(ft.__file__), "libfusedtok_amd.so")
P, I, L, U, F, D = (ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t,
                    ctypes.c_float, ctypes.c_double)
X = 64  # a pointer that is never followed: every call is refused


@pytest.mark.parametrize("theta", [1e-300, 1e-12, 0.9 * 2.0 ** -10, 0.0, -1.0, float("nan")])
@pytest.mark.parametrize("paged", [False, True])
def test_small_bases_are_refused(paged, theta):
    lib = ctypes.CDLL(LIB)
    lib.ft_last_error.restype = ctypes.c_char_p
    head = [P, I, L, P, P, P, I, P, I, D, F, I, P, P, P]
    args = [X, 1, 384, X, X, X, 1, 0, 64, theta, 1e-6, 1, X, X, X]
    if paged:
        lib.ft_qk_norm_rope_kv_append_paged_launch.argtypes = head + [P] + [I] * 6 + [U]
        st = lib.ft_qk_norm_rope_kv_append_paged_launch(*args, X, 3, 4, 1, 64, 4, 16, 0)
    else:
        lib.ft_qk_norm_rope_launch.argtypes = head + [I] * 4 + [U]
        st = lib.ft_qk_norm_rope_launch(*args, 3, 4, 1, 64, 0)
    assert st == 1 and b"theta" in lib.ft_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("theta", [2.0 ** -10, 0.03, 1.0, 1e300])
@pytest.mark.parametrize("rot", [2, 48, 64])
def test_bases_of_any_size(rot, theta):
    """Positions of up to 2^20, angles of up to 2^20 / theta; the bound is that of
    the norms' and rotation's own test, an angle's error 2^-51 of it."""
    from tests import step_refs as refs
    from tests.test_gpu_qknorm import dev, inputs, near
    far = 2 ** 20
    qkv, w, pos = inputs(rot, 40, 3, 1, 64, torch.float32, far=far)
    got = ft.qk_norm_rope(qkv, 3, 1, dev(w[0]), dev(w[1]), dev(pos[0]), theta=theta,
                          rotary_dim=rot, eps=1e-5)
    want = refs.qk_norm_rope(qkv.double().cpu().numpy(), 3, 1, *w, pos, rot, theta, 1e-5, False)
    for g, e in zip(got, want):
        near(g, e, torch.float32, 64, far / min(theta, 1.0))
    qkv = torch.randn(40, 5 * 64, device="cuda")
    pos = torch.as_tensor(np.arange(40, dtype=np.int32) * 26000, device="cuda")
    q, k, _ = ft.qk_norm_rope(qkv, 3, 1, None, None, pos, theta=theta)
    # a turn keeps a head's length: 64 squares, a rounding of each value and of the turn's parts
    for new, old in ((q, qkv[:, :192].view(40, 3, 64)), (k, qkv[:, 192:256].view(40, 1, 64))):
        a, b = new.double().norm(dim=-1), old.double().norm(dim=-1)
        assert ((a - b).abs() <= 8 * 2.0 ** -24 * b).all()
