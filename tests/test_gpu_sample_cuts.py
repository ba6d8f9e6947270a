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
