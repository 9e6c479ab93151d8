"""qk_norm_rotate at the edges of its range."""

import pytest
import torch

from test_qk_norm_rotate_gpu import BF16, FP32, compare, make, run, want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,HQ,HK,D,R", [
    (1, 7, 5, 1, 128, 128), (2, 3, 3, 7, 64, 32), (1, 1, 1, 1, 16, 16), (3, 11, 5, 3, 96, 96), (1, 5, 3, 1, 256, 256), (2, 5, 5, 3, 90, 42)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_without_eps(B, T, HQ, HK, D, R, dtype, interleaved):
    """Heads and tokens that do not fill a warp's rows: what is not there has no norm, and no part in a weight's gradient."""
    d = make(B, T, HQ, HK, D, R, dtype, 11)
    compare(run(d, interleaved, eps=0.0), want(d, interleaved, eps=0.0), B * T * max(HQ, HK))
