"""Dropout, the scaled lookup and group norm at the ends of what they take: the largest values and sizes, the longest sums, sums that are exact."""
import pytest
import torch

import test_gpu_norm as norm_checks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,S,C,G,start", [(6, 4001, 256, 32, (0, 3015, 3797)), (1, 40000, 16, 2, (0, 39999)), (2, 30001, 48, 3, None)])
def test_norm_of_values_whose_squares_are_too_large(B, S, C, G, start, dtype):
    """Values of some 3e19, whose squares leave the type that sums are formed in, all close together: their mean's error counts, e = 80 u 3e19 = 1.5e14 for a
    deviation of 2e17, and nothing is infinite.  Levels that have fewer keys in a tile than the threads side by side: some of those have none."""
    torch.manual_seed(S)
    step = 2.0 ** 57                                             # of bfloat16 from 2^64 to 2^65
    x = (2.0 ** 64 * 1.5 + step * torch.randint(-2, 3, (B, S, C), device="cuda")).to(dtype)
    assert bool(x.isfinite().all()) and bool((x.double() >= 2.0 ** 64).all())
    norm_checks.check(x, G, *norm_checks.params(C, dtype), start=start, act="silu")
