"""The microscaled operators at the ends of their ranges: values, scales, sizes and places in memory."""
import numpy as np
import pytest

import mx_plain as plain
from gpu_util import say
from test_gpu_mx import check_mx, check_product, f64, mx_random, to_dev

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


def check_many_rows(rng, act, M, N, seams):
    """A product with N weight rows of 128 ones, but for 64 random ones at each of `seams`."""
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0]
    need = N * (64 + 16 + 2 * M) + (8 << 30)
    if free < need:
        pytest.skip(f"needs {need >> 30} GiB of device memory")
    say("many rows", act, M, N)
    w = vm.MXTensor.empty((N, 128), "fp4")
    w.codes.fill_(0x22)   # ones
    w.scales.fill_(127)
    part, pv = mx_random(rng, (64,), 128, "fp4")
    for at in seams:
        w.codes[at:at + 64] = part.codes
        w.scales[at:at + 64] = part.scales
    x, xv = mx_random(rng, (M,), 128, act, narrow=True)
    y = vm.mx_matmul(x, w)
    check_product(y[:, :1], xv, np.ones((1, 128)), "bf16")
    for at in seams:
        check_product(y[:, at:at + 64], xv, pv, "bf16")
        y[:, at:at + 64] = y[:, :1]
    for row in y:
        assert bool((row == row[0]).all())


@pytest.mark.parametrize("M,N", [(1, 1 << 30), (17, (1 << 29) + 70)])
def test_product_many_weight_rows(rng, M, N):
    """Work-groups of few tokens whose work-items would pass 2^32 in one dimension of a grid."""
    check_many_rows(rng, "fp8", M, N, [(1 << 27) - 32, (1 << 28) - 32, N - 64])


@pytest.mark.parametrize("act", ["fp4", "fp8"])
@pytest.mark.parametrize("N", [1 << 30, (1 << 29) + 70])
def test_product_many_tiles(rng, act, N):
    """2^21 tiles and more, whose work-groups continue in the grid's second dimension."""
    check_many_rows(rng, act, 33, N, [(1 << 28) - 32, N - 64])
