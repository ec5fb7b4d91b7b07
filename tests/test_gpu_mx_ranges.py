"""The microscaled operators at the ends of their ranges: values, scales, sizes and places in memory."""
import numpy as np
import pytest

import mx_plain as plain
from gpu_util import say
from test_gpu_mx import TYPES, check_mx, f64, to_dev

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import vcsr_mc_amd as vm  # noqa: E402


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [96, 5000, 40000])
@pytest.mark.parametrize("sign", [1, -1])
def test_norm_past_the_largest_number(fmt, type_, cols, sign):
    """A normalised value past the largest 32-bit number is an infinity: its block is NaN, and no
    other.  The largest finite ones keep theirs."""
    say("norm overflow", fmt, type_, cols, sign)
    x = np.ones((2, cols))
    x[0, 5] = 8 * sign             # y near 8 * 3e38 in one block of the first row alone
    w = np.ones(cols)
    w[5] = w[cols - 1] = 3e38      # y near 3e38 elsewhere
    xd, wd = to_dev(x, type_), to_dev(w, "f32")
    q, _ = vm.rms_norm_mx(xd, wd, eps=0.0, fmt=fmt)
    y, _ = plain.norm(f64(xd), None, f64(wd), 0.0)
    y = np.where(np.abs(y) >= 2.0 ** 128 - 2.0 ** 103, np.inf, y)
    assert np.isinf(y).sum() == 1
    check_mx(q, y, fmt)
