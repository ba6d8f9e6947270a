"""GPU tests of sample_filtered_batched by the way its cuts are found: limits
in a bin of few logits or of many, before or behind the bins with weight, min-p's
bins inside or outside the cut. Tokens are equal to the plain form's
(step_refs.sample), as in test_gpu_sample_filtered. A row is one workgroup's up
to 32768 logits (of up to 4096, 16384 and 32768 at a time) and slices of 8192
above."""

import numpy as np
import pytest
import torch

from tests.test_gpu_sample_filtered import check, dev

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [4000, 20000, 32768, 32769, 50257])
def test_both_limits_in_full_bins(n, dtype):
    """Hundreds of logits in each bin (a bin is 0.043 wide): k's limit and p's
    each go from a bin into narrower histograms, in many rows at once."""
    rng = np.random.default_rng(n)
    x, u = dev(rng.uniform(-2.5, 0.0, (96, n)), dtype), rng.random(96).astype(np.float32)
    for k, p in ((n // 2, 0.6), (n // 3, 0.97), (n - 2, 0.2), (0, 0.8), (n // 5, 1.0)):
        check(x, u, 1.0, k, p)
    check(x, u, 1.0, rng.integers(1, n, 96).astype(np.int32), rng.uniform(0.05, 0.99, 96), 0.2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 65, 2000, 32768, 40000])
@pytest.mark.parametrize("values", [1, 3, 1000])
def test_a_top_p_of_nothing_keeps_the_first_token(values, n, dtype):
    """p of 0 and less, in rows of which many logits share the first bin:
    equal ones (zeros too), a few values, a dense line."""
    rng = np.random.default_rng(n + values)
    x = rng.integers(0, values, (12, n)) * (0.3 / values)
    x = np.concatenate([x, x + 3.0, -3.0 - x, np.zeros((4, n))])
    x[-1, n // 2 + 1:] = -np.inf
    x, u = dev(x, dtype), rng.random(len(x)).astype(np.float32)
    first = np.argmax(x.float().cpu().numpy(), 1).tolist()
    rows = np.arange(len(x))
    p = np.array([0.0, -2.0, -0.0, -np.inf, 2.0 ** -149])[rows % 5]
    for temp, k, minp in ((1.0, 0, 0.0), (1.0, 40, 0.0), (0.3, 0, 0.7), (5.0, 700, 1.0)):
        got = check(x, u, temp, k, p, minp)
        assert got.tolist() == first
    # among rows with limits of their own
    p = np.where(rows % 3, p, 0.6)
    check(x, u, 1.0, np.where(rows % 2, 0, 100), p)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("minp", [0.02, 0.05, 0.5, 1.0])
@pytest.mark.parametrize("n", [20000, 33000, 50257])
def test_a_mask_that_leaves_fewer_than_k(n, minp, dtype):
    """k beyond the tokens that have weight cuts nothing and min-p does: masked
    rows (-inf, the type's lowest value, far logits), weights all over and next
    to min-p's border, in one slice and in all of them."""
    rng = np.random.default_rng(n)
    rows, left = 24, 30
    low = [-np.inf, torch.finfo(dtype).min, -200.0]
    x = np.empty((rows, n))
    for r in range(rows):
        x[r] = low[r % 3]
        at = rng.choice(n if r % 4 else 5000, left, False)
        x[r, at] = rng.standard_normal(left) if r % 2 else np.log(minp) + rng.normal(0, 0.06, left)
        x[r, at[0]] = x[r, at].max() if r % 2 else 0.0
        x[r, at[1]] = x[r, at[0]]
    x, u = dev(x, dtype), rng.random(rows).astype(np.float32)
    for v in (u, u / 8, 1 - u / 16):
        check(x, v, 1.0, 50, 1.0, minp)
        check(x, v, 1.0, 50, 0.9, minp)
    # left and left + 1: the last k that cuts nothing and the first that may
    for k in (left - 1, left, left + 1, 10000):
        check(x, u, 0.8, k, 1.0, minp)


def test_a_token_behind_k_that_min_p_keeps():
    """Two tokens with weight, far apart: the second has its share."""
    x = torch.full((1000, 40000), -100.0, device="cuda")
    x[:, 0], x[:, 20000] = 0.0, float(np.log(0.052))
    u = (np.arange(1000) + 0.5).astype(np.float32) / 1000
    got = check(x, u, 1.0, 10, 1.0, 0.05)
    assert abs(got.eq(20000).sum().item() - 1000 * 0.052 / 1.052) <= 1
