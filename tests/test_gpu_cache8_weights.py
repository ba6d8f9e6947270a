"""The softmax weights of attention over the 8-bit cache keep all their bits: a
row of one token is code * scale, rounded once to the output's type."""

import numpy as np
import pytest
import torch

import fusedtok_amd as ft
from tests.test_gpu_cache8 import TYPES, dev, i32, paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("group,d", [(4, 64), (4, 128), (2, 256), (5, 96), (20, 128), (3, 16),
                                     (4, 36)])
def test_one_token_is_its_value(group, d, dtype):
    """One token has weight 1, so its V scale alone is what enters the PV
    product. code * scale has 31 bits: a float32 sum of it is off by 2^-24
    (2^-23 where the adder cuts bits off), the division by the weights' sum, 1,
    by nothing; the half types then round that once more. So float32 is within
    2^-22, and a half result is the rounding of code * scale, except where that
    lies within 2^-22 of the middle between two results, where either may come
    out. (2^-15 of the value, as two truncated parts of 8 bits leave out,
    changes one result in a hundred in fp16.)"""
    rng = np.random.default_rng(group + d)
    b, hkv, page = 60, 4, 16
    (kp, vp, ks, _), table = paged(rng, b, hkv, page, d, [1] * b)
    # from 2^-12 to 2^6 (fp16 holds them times 127), all 24 bits drawn
    vs = (2.0 ** rng.uniform(-12, 6, ks.shape)).astype(np.float32)
    q = rng.standard_normal((b, hkv * group, d))
    out = ft.attention_decode_paged_int8(dev(q, dtype), dev(kp), dev(vp), dev(ks), dev(vs),
                                         i32(table), i32([1] * b))
    first = table[:, 0]
    exact = vp[first, :, 0].astype(np.float64) * vs[first].astype(np.float64)[..., None]
    exact = np.repeat(exact, group, axis=1)   # [b, hq, d]
    got = out.cpu().double().numpy()
    slack = 2.0 ** -22 * np.abs(exact)
    if dtype is torch.float32:
        assert (np.abs(got - exact) <= slack).all()
        return
    # half a step of the result's binade (of fp16's smallest numbers below 2^-14)
    _, e = np.frexp(np.abs(exact))
    if dtype is torch.float16:
        e = np.maximum(e, -13)
    half = np.ldexp(torch.finfo(dtype).eps / 2, e - 1)
    bad = np.abs(got - exact) > half + slack
    assert not bad.any(), (int(bad.sum()), bad.size)
