"""The microscaled operators at the ends of their ranges: values, scales, sizes and places in memory."""
import numpy as np
import pytest

import mx_plain as plain
from gpu_util import say
from test_gpu_mx import (ACTS, TAU, act_of, check_moe, check_mx, check_product, f64, moe_case, mx_random,
                         to_dev)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import vcsr_mc_amd as vm  # noqa: E402


# ---- values ----------------------------------------------------------------------------------
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


# ---- scales ----------------------------------------------------------------------------------
@pytest.mark.parametrize("act,narrow", [("fp8", True), ("fp4", False)])
@pytest.mark.parametrize("mid_x,mid_w", [(2, 250), (5, 248), (250, 4), (252, 2)])
@pytest.mark.parametrize("M", [1, 20, 100])
def test_product_scales(rng, act, narrow, mid_x, mid_w, M):
    """Scales of X at one end of their range, of W at the other: products are of normal size."""
    say("product scales", act, mid_x, mid_w, M)
    x, xv = mx_random(rng, (M,), 300, act, mid=mid_x, narrow=narrow)
    w, wv = mx_random(rng, (200,), 300, "fp4", mid=mid_w)
    check_product(vm.mx_matmul(x, w, dtype=torch.float32), xv, wv, "f32")


@pytest.mark.parametrize("mid_x,mid_w", [(5, 235), (9, 231), (60, 180), (244, 8)])
@pytest.mark.parametrize("T,D,F,E", [(1, 256, 64, 2), (3, 200, 100, 2), (20, 300, 64, 3)])
def test_moe_scales(rng, mid_x, mid_w, T, D, F, E):
    """Scales of x and of the gate and up rows far apart, bytes 3 to 246: h is of normal size."""
    say("moe scales", mid_x, mid_w, T, D, F, E)
    x, xv = mx_random(rng, (T,), D, "fp8", mid=mid_x)
    w13, a = mx_random(rng, (E, 2 * F), D, "fp4", mid=mid_w)
    w2, b = mx_random(rng, (E, D), F, "fp4", mid=119)
    y = vm.mx_moe(x, torch.zeros((E, D), device="cuda"), w13, w2, E, dtype=torch.float32)
    with np.errstate(over="ignore"):  # sigmoid of large gates
        check_moe(y, (xv, np.zeros((E, D)), a, b), E, True, "f32", router_gap=False)


@pytest.mark.parametrize("T", [1, 3, 20])
def test_moe_router_of_tiny_activations(rng, T):
    """Activations below 2^-126 under a large router: logits of normal size choose as they should."""
    D, F, E, k = 256, 64, 8, 2
    x, xv = mx_random(rng, (T,), D, "fp8", mid=5, narrow=True)
    router = to_dev(rng.standard_normal((E, D)) * 2.0 ** 118)
    w13, a = mx_random(rng, (E, 2 * F), D, "fp4", mid=233)
    w2, b = mx_random(rng, (E, D), F, "fp4", mid=119)
    y = vm.mx_moe(x, router, w13, w2, k, dtype=torch.float32)
    check_moe(y, (xv, f64(router), a, b), k, True, "f32")


# ---- sizes -----------------------------------------------------------------------------------
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


# ---- streams and gradients -------------------------------------------------------------------
def _calls(g):
    """For every entry point, a call with a stream and the operands that it alone holds."""
    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    w = vm.mx_quantise(normal(512, 1024), "fp4")
    w13 = vm.mx_quantise(normal(4 * 256, 1024), "fp4")
    w13 = vm.MXTensor(w13.codes.view(4, 256, -1), w13.scales.view(4, 256, -1), 1024, "fp4")
    w2 = vm.mx_quantise(normal(4 * 1024, 128), "fp4")
    w2 = vm.MXTensor(w2.codes.view(4, 1024, -1), w2.scales.view(4, 1024, -1), 128, "fp4")
    x, r, gain, router = normal(96, 1024), normal(96, 1024), normal(1024), normal(4, 1024)
    q = vm.mx_quantise(x)
    return {"quantise": (lambda x, s: vm.mx_quantise(x, stream=s).codes, [x]),
            "dequantise": (lambda c, e, s: vm.mx_dequantise(vm.MXTensor(c, e, 1024, "fp8"), stream=s),
                           [q.codes, q.scales]),
            "norm": (lambda x, r, w, s: vm.rms_norm_mx(x, w, residual=r, stream=s)[1], [x, r, gain]),
            "matmul": (lambda c, e, s: vm.mx_matmul(vm.MXTensor(c, e, 1024, "fp8"), w, stream=s),
                       [q.codes, q.scales]),
            "moe": (lambda c, e, r, s: vm.mx_moe(vm.MXTensor(c, e, 1024, "fp8"), r, w13, w2, 2, stream=s),
                    [q.codes, q.scales, router])}


@pytest.mark.parametrize("name", ["quantise", "dequantise", "norm", "matmul", "moe"])
def test_operands_dropped_before_their_stream_is_done(name):
    """What the caller drops behind a call on another stream keeps its memory until that stream has
    passed the call, and the result is right."""
    say("dropped operands", name)
    call, held = _calls(torch.Generator(device="cuda").manual_seed(3))[name]
    want = call(*held, None)
    side, busy = torch.cuda.Stream(), torch.randn((8192, 8192), device="cuda")
    out = torch.empty_like(busy)
    torch.matmul(busy, busy, out=out)
    operands = [t.clone() for t in held]
    where = {t.data_ptr() for t in operands}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(30):
            torch.matmul(busy, busy, out=out)
    got = call(*operands, side)
    sizes = [t.numel() * t.element_size() for t in operands]
    del operands
    new = [torch.empty((n,), dtype=torch.uint8, device="cuda") for n in sizes for _ in range(4)]
    late = not side.query()
    taken = where & {t.data_ptr() for t in new}
    for t in new:
        t.fill_(0xff)
    side.synchronize()
    assert late and not taken
    assert torch.equal(got, want)


def test_gradients_are_refused_not_lost():
    """The sum that a norm returns and a layer's output carry no gradient: who asks for one is told."""
    say("gradients")
    calls = _calls(torch.Generator(device="cuda").manual_seed(3))
    norm, (x, r, gain) = calls["norm"]
    moe, (codes, scales, router) = calls["moe"]
    want_h, want_y = norm(x, r, gain, None), moe(codes, scales, router, None)
    asks = [t.clone().requires_grad_() for t in (x, r, router)]
    for call in (lambda: norm(asks[0], r, gain, None), lambda: norm(x, asks[1], gain, None),
                 lambda: moe(codes, scales, asks[2], None)):
        with pytest.raises(vm.VCSRMCError, match="no_grad") as e:
            call()
        assert e.value.status == vm.ERR_ARG
    # in codes nothing is lost that torch could follow; a weight does not reach the sum
    assert torch.equal(vm.rms_norm_mx(asks[0], gain)[0].codes, vm.rms_norm_mx(x, gain)[0].codes)
    assert torch.equal(norm(x, r, torch.nn.Parameter(gain), None), want_h)
    assert torch.equal(vm.mx_quantise(asks[0]).codes, vm.mx_quantise(x).codes)
    with torch.no_grad():
        assert torch.equal(norm(asks[0], asks[1], gain, None), want_h)
        assert torch.equal(moe(codes, scales, asks[2], None), want_y)
