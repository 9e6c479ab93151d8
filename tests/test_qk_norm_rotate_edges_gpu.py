"""qk_norm_rotate at the edges of its range."""

import math
from fractions import Fraction

import pytest
import torch

from conftest import assert_close
from test_qk_norm_rotate_gpu import BF16, FP32, FP32_RTOL, compare, make, run, want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,HQ,HK,D,R", [
    (1, 7, 5, 1, 128, 128), (2, 3, 3, 7, 64, 32), (1, 1, 1, 1, 16, 16), (3, 11, 5, 3, 96, 96), (1, 5, 3, 1, 256, 256), (2, 5, 5, 3, 90, 42)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_without_eps(B, T, HQ, HK, D, R, dtype, interleaved):
    """Heads and tokens that do not fill a warp's rows: what is not there has no norm, and no part in a weight's gradient."""
    d = make(B, T, HQ, HK, D, R, dtype, 11)
    compare(run(d, interleaved, eps=0.0), want(d, interleaved, eps=0.0), B * T * max(HQ, HK))


@pytest.mark.parametrize("power", [-55, -44, -30, 30, 43, 55])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("D", [128, 90])
def test_rows_of_any_size_whose_squares_are_numbers(power, dtype, D):
    """A power of two changes no rounding: results are those of ordinary rows, gradients by as much smaller or larger."""
    d = make(2, 9, 3, 2, D, D // 2 // 8 * 8, dtype, 13)
    for n in "qk":
        d[n] *= 2.0 ** power
    got, ref = run(d, eps=0.0), want(d, eps=0.0)
    for n in "qk":
        got["d" + n], ref["d" + n] = got["d" + n].double() * 2.0 ** power, ref["d" + n] * 2.0 ** power
    compare({n: t.to(dtype) if n in ("dq", "dk") else t for n, t in got.items()}, ref, 54)


PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


@pytest.mark.parametrize("first", [2 ** 33 + 5, 2 ** 36 + 12345, -(2 ** 36) - 7, 2 ** 40 + 3, 2 ** 45 + 1])
def test_positions_as_far_out_as_64_bits_hold_the_turn(first):
    """Against angles in whole numbers.  Half a unit of 2^-64 of a turn for inv_freq's two parts each, and one for what is
    below: an angle is off by |position| * 2^-63 of a turn beside fp32's rounding (compare's tolerance)."""
    T, D = 3, 16
    d = make(1, T, 2, 1, D, D, FP32, 12, first=first, rows=False)
    d["freq"] = torch.tensor([1.0, 0.7310585786, 3.25, 0.01, 1e-4, 0.3678794, 17.0, 2.0 ** -20], device="cuda")
    got = run(d)
    turns = [[float(t * Fraction(f) / (2 * PI) % 1) for f in d["freq"].tolist()] for t in range(first, first + T)]
    angle = 2 * math.pi * torch.tensor(turns, dtype=torch.float64)[:, None]
    for n in "qk":
        x = d[n].double().cpu()
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * d[n + "w"].double().cpu()
        a, b = x[..., :D // 2], x[..., D // 2:]
        y = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)
        # a turned pair moves by its length, at most sqrt(D) times the row's root mean square, times the angle's error
        assert_close(got["y" + n], y, FP32_RTOL + D ** 0.5 * 2 * math.pi * abs(first) * 2.0 ** -63, n, outlier_frac=0.0)
