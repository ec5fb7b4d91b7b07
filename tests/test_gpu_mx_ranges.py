"""The microscaled operators at the ends of their ranges: values, scales, sizes and places in memory."""
import numpy as np
import pytest

import mx_plain as plain
from gpu_util import say
from test_gpu_mx import (ACTS, act_of, check_moe, check_mx, check_product, f64, moe_case, mx_random,
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


def check_norm_exact(q, x, r, w, eps):
    """Scales and codes are those of the normalised values in 64 bits, rounded once.  Those values
    carry a few roundings of 2^-53 on either side, so where a change by 1e-12 of them changes a code
    or a scale, either is right; such places are a few in a million at most."""
    h = x.float() if r is None else x.float() + r.float()   # the norm's h has 32 bits
    y, _ = plain.norm(f64(h), None, f64(w), np.float32(eps))
    cols = y.shape[1]
    nb = plain.pad(cols, 32) // 32
    got_c, got_s = q.codes.cpu().numpy(), q.scales.cpu().numpy()
    right_v, right_s, values, scales = 0, 0, [], []
    got = plain.unpack(got_c, got_s, cols, q.fmt)
    for f in (1, 1 - 1e-12, 1 + 1e-12):
        c, s = plain.quantise(y * f, q.fmt)
        values.append(plain.values(c, s, q.fmt)[:, :cols])
        scales.append(s)
        right_v |= got == values[-1]
        right_s |= got_s[:, :nb] == s
    assert np.all(right_s) and np.all(right_v)
    assert np.mean(values[1] != values[2]) <= 1e-5 + 1 / y.size
    assert np.mean(scales[1] != scales[2]) <= 1e-5 + 1 / scales[0].size
    assert not np.any(got_s[:, nb:])


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("type_,wtype", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"),
                                         ("bf16", "f32")])
@pytest.mark.parametrize("rows,cols,residual", [(1, 1, True), (3, 100, False), (2, 511, True), (40, 4096, True),
                                                (33, 5000, False), (20, 8200, True), (9, 33000, True)])
def test_norm_rounds_once(rng, fmt, type_, wtype, rows, cols, residual):
    say("norm exact", fmt, type_, wtype, rows, cols, residual)
    x = to_dev(rng.standard_normal((rows, cols)) * 3, type_)
    r = to_dev(rng.standard_normal((rows, cols)), type_) if residual else None
    w = to_dev(1 + 0.2 * rng.standard_normal(cols), wtype)
    q, _ = vm.rms_norm_mx(x, w, residual=r, eps=1e-5, fmt=fmt)
    check_norm_exact(q, x, r, w, 1e-5)


def test_norm_rounds_once_over_many(rng):
    """17 million values: what a norm in 32 bits gets wrong a few times in a million."""
    x, r = (to_dev(rng.standard_normal((2100, 8192), np.float32)) for _ in range(2))
    w = to_dev(1 + 0.2 * rng.standard_normal(8192))
    q, _ = vm.rms_norm_mx(x, w, residual=r, eps=1e-5)
    check_norm_exact(q, x, r, w, 1e-5)


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


# ---- experts -----------------------------------------------------------------------------------
@pytest.mark.parametrize("T", [1, 5, 40])
@pytest.mark.parametrize("D,router_type", [(1024, "f32"), (1025, "f32"), (2049, "bf16"), (2500, "f32"), (3100, "f16"),
                                           (4000, "bf16"), (4224, "f32"), (9000, "f32")])
def test_moe_logits_in_parts(rng, T, D, router_type):
    """Routers' rows in one to four parts."""
    say("moe parts", T, D, router_type)
    ops, v = moe_case(rng, T, D, 64, 20, router_type)
    check_moe(vm.mx_moe(*ops, 3, renormalise=False, dtype=torch.float32), v, 3, False, "f32")


@pytest.mark.parametrize("T", [1, 6, 40])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
@pytest.mark.parametrize("E,k", [(6, 2), (100, 3)])
def test_moe_infinite_logits(rng, T, value, E, k):
    """An infinite logit of one or of all experts.  A softmax over +inf is NaN; -inf comes after all
    finite ones and has weight zero where it is chosen."""
    say("moe infinite", T, value, E, k)
    (x, router, w13, w2), v = moe_case(rng, T, 96, 32, E)
    x.codes[:, 7] = 0x38     # the value whose weight in the router is infinite is positive
    xv = plain.unpack(x.codes.cpu().numpy(), x.scales.cpu().numpy(), 96, "fp8")
    one = router.clone()
    one[E - 1, 7] = value
    y = vm.mx_moe(x, one, w13, w2, k, dtype=torch.float32)
    if value > 0:
        assert torch.all(torch.isnan(y))
    else:  # as if that expert were the least of all
        r = f64(router)
        ids = plain.choose(np.where(np.arange(E) == E - 1, -np.inf, xv @ r.T), k)
        assert not np.any(ids == E - 1)
        check_moe(y, (xv, r[:E - 1], v[2][:E - 1], v[3][:E - 1]), k, True, "f32")
    router[:, 7] = value
    assert torch.all(torch.isnan(vm.mx_moe(x, router, w13, w2, k, dtype=torch.float32)))


def test_moe_chosen_at_minus_infinity(rng):
    """All experts are chosen, one of them at -inf: it has weight zero."""
    (x, router, w13, w2), (xv, r, a, b) = moe_case(rng, 5, 96, 32, 4)
    x.codes[:, 7] = 0x38
    xv = plain.unpack(x.codes.cpu().numpy(), x.scales.cpu().numpy(), 96, "fp8")
    router[2, 7] = -np.inf
    rest = [0, 1, 3]
    for renormalise in (True, False):
        y = vm.mx_moe(x, router, w13, w2, 4, renormalise=renormalise, dtype=torch.float32)
        check_moe(y, (xv, r[rest], a[rest], b[rest]), 3, renormalise, "f32")


class Experts:
    """float64 values of an MX tensor's matrices, made when they are asked for."""

    def __init__(self, q):
        self.q, self.shape, self.made = q, q.shape, {}
        byte = np.arange(256)
        pairs = np.stack((byte & 15, byte >> 4), -1)
        self.pairs = np.where(pairs >= 8, -1, 1) * plain.GRID["fp4"][pairs % 8]

    def __getitem__(self, e):
        if e not in self.made:
            v = self.pairs[self.q.codes[int(e)].cpu().numpy()].reshape(self.shape[1], -1, 32)
            s = np.ldexp(1.0, self.q.scales[int(e)].cpu().numpy().astype(int) - 127)
            self.made[e] = (v * s[:, :v.shape[1], None]).reshape(self.shape[1], -1)[:, :self.shape[2]]
        return self.made[e]


@pytest.mark.parametrize("T,k,rows", [(1, 4, [0]), (1, 8, [0]), (7, 6, [0, 6]), (64, 8, [0, 31, 63])])
def test_moe_full_layer(rng, T, k, rows):
    """64 experts of 4096 x 2048: some tokens' results against the definition."""
    D, F, E = 4096, 2048, 64
    say("moe full", T, k)
    g = torch.Generator(device="cuda").manual_seed(T)

    def weights(n, cols):
        codes = torch.randint(0, 256, (E, n, cols // 2), dtype=torch.uint8, device="cuda", generator=g)
        return vm.MXTensor(codes, torch.randint(117, 121, (E, n, cols // 32), dtype=torch.uint8, device="cuda",
                                                generator=g), cols, "fp4")

    w13, w2 = weights(2 * F, D), weights(D, F)
    x, xv = mx_random(rng, (T,), D, "fp8", mid=121, narrow=True)
    router = to_dev(rng.standard_normal((E, D)) / np.sqrt(D) / 4, "bf16")
    y = vm.mx_moe(x, router, w13, w2, k, dtype=torch.float32)
    check_moe(y[rows], (xv[rows], f64(router), Experts(w13), Experts(w2)), k, True, "f32")


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
    del w, y, row
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M,N", [(1, 1 << 30), (17, (1 << 29) + 70)])
def test_product_many_weight_rows(rng, M, N):
    """Work-groups of few tokens whose work-items would pass 2^32 in one dimension of a grid."""
    check_many_rows(rng, "fp8", M, N, [(1 << 27) - 32, (1 << 28) - 32, N - 64])


@pytest.mark.parametrize("act", ["fp4", "fp8"])
@pytest.mark.parametrize("N", [1 << 30, (1 << 29) + 70])
def test_product_many_tiles(rng, act, N):
    """2^21 tiles and more, whose work-groups continue in the grid's second dimension."""
    check_many_rows(rng, act, 33, N, [(1 << 28) - 32, N - 64])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", [(33, 50000, 200), (64, 50000, 130), (65, 50000, 400), (33, 25000, 1030)])
def test_product_few_tokens_many_rows(rng, act, M, N, K):
    """The largest tiles, mostly empty along the tokens."""
    say("product wide", act, M, N, K)
    x, xv, tau = act_of(rng, M, K, act)
    w, wv = mx_random(rng, (N,), K, "fp4")
    check_product(vm.mx_matmul(x, w, dtype=torch.float32), xv, wv, "f32", tau)


@pytest.mark.parametrize("act", ["fp8", "fp4"])
def test_product_tiles_far_offsets(rng, act):
    """Tiles of weights and of results past 4 GB: rows of ones, and random ones at the end."""
    M, N, K = 2100, 1_100_000, 8192
    say("product tiles far", act)
    w = vm.MXTensor.empty((N, K), "fp4")
    w.codes.fill_(0x22)   # ones
    w.scales.fill_(127)
    part, pv = mx_random(rng, (64,), K, "fp4")
    w.codes[-64:] = part.codes
    w.scales[-64:] = part.scales
    x, xv = mx_random(rng, (M,), K, act, narrow=True)
    y = vm.mx_matmul(x, w)
    assert w.codes.numel() > 1 << 32 and y.numel() * 2 > 1 << 32
    check_product(y[:, -64:], xv, pv, "bf16")
    check_product(y[:, :1], xv, np.ones((1, K)), "bf16")
    for t in range(0, M, 100):
        assert bool((y[t:t + 100, :-64] == y[t:t + 100, :1]).all())


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
