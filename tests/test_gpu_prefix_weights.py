"""GPU test of how many bits of a softmax weight attention_decode_paged_prefix
takes into the product with V, where the values cancel.

Three tokens: two with a score of exactly 0 and one with -a / sqrt(D), so the
weights are 1, 1 and w = exp(-a / sqrt(D)); their values are -hi, -lo and 1 with
hi + lo next to w in two numbers of the type. The output (w - hi - lo) / (2 + w) is
what the type's parts of w leave, and no rounding of the output hides it.

The bound. The scores are exact (one product of two numbers of the type). The
exponent t, |t| <= 2, is off by a rounding of its factor and one of its own, so
w by ln(2) |t| 2 * 2^-24 <= 2.8 * 2^-24 of it, and by 2 * 2^-24 for the exponential.
The numerator is a sum of at most 6 additions, a unit in the last place (2^-23)
each of what they hold, at most W = w + |hi + lo|: 12 * 2^-24 W. In all under 20 *
2^-24 W / (2 + w), and 2^-22 of w more for fp16's two parts. The sum of the weights
and the quotient: 6 * 2^-24 of the output; half a step of the type for it."""

import numpy as np
import pytest
import torch

import fusedtok_amd as ft

pytestmark = pytest.mark.gpu

DEV = "cuda"
HKV, GQ, PAGE = 2, 4, 16


def rounded(x, dtype):
    return torch.as_tensor(np.ascontiguousarray(x)).to(dtype).double().numpy()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 72, 128])
@pytest.mark.parametrize("size", [1, 4, 5, 16, 17, 32, 40])
@pytest.mark.parametrize("own", [False, True])
def test_weights_keep_their_bits(own, size, d, dtype):
    """Groups of `size` sequences, 4 * size rows a kv head; the tokens are the
    groups' prefixes or (own) the sequences' own."""
    groups = 12
    b = groups * size
    rng = np.random.default_rng(size * d)
    a = rounded(rng.uniform(0.1, 1.38, (b, HKV * GQ)) * np.sqrt(d), dtype)
    w = np.exp(-a / np.sqrt(d))
    entries, per = (b, 1) if own else (groups, size)
    # entry e, head kv, dim i: the weight of one of the rows that read them
    rows = w.reshape(entries, per, HKV, GQ).transpose(0, 2, 1, 3).reshape(entries, HKV, -1)
    r = rows[:, :, np.arange(d) % rows.shape[2]]
    hi = rounded(r, dtype)
    lo = rounded(r - hi, dtype)
    k, v = np.zeros((entries, HKV, PAGE, d)), np.zeros((entries, HKV, PAGE, d))
    k[:, :, 2, 0] = -1.0
    v[:, :, 0], v[:, :, 1], v[:, :, 2] = -hi, -lo, 1.0
    q = np.zeros((b, HKV * GQ, d))
    q[:, :, 0] = a

    def dev(x, t=dtype):
        return torch.as_tensor(np.ascontiguousarray(x)).to(DEV, dtype=t)

    table = np.arange(entries).reshape(-1, 1)
    none = np.full((groups if own else b, 1), -1)
    lens = [np.full(entries, 3), np.zeros(len(none))]
    if own:
        table, none, lens = none, table, lens[::-1]
    got = ft.attention_decode_paged_prefix(
        dev(q), dev(k), dev(v), dev(table, torch.int32), dev(lens[0], torch.int32),
        dev(none, torch.int32), dev(lens[1], torch.int32),
        dev(np.arange(groups + 1) * size, torch.int32)).double().cpu().numpy()

    left = (hi + lo)[np.arange(b) // per].repeat(GQ, axis=1)     # [b, heads, d]
    w = w[:, :, None]
    want = (w - left) / (2 + w)
    assert np.abs(want).reshape(groups, -1).min(-1).max() < 2.0 ** -16   # they do cancel
    part = 20 * 2.0 ** -24 * (w + left) + (2.0 ** -22 * w if dtype is torch.float16 else 0)
    bound = part / (2 + w) + (torch.finfo(dtype).eps / 2 + 6 * 2.0 ** -24) * np.abs(want)
    if dtype is torch.float16:
        bound = bound + 2.0 ** -25    # half a step of the least numbers
    over = np.abs(got - want) - bound
    assert over.max() <= 0, over.max()
