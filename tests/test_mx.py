"""What the microscaled operators refuse, before any device work, and their layouts; no GPU."""
import ctypes
import importlib.util
import pathlib
import re
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mx_plain as plain
import vcsr_mc_amd as vm
from vcsr_mc_amd import mx


def refused(fn, *words):
    with pytest.raises(vm.VCSRMCError) as e:
        fn()
    assert e.value.status == vm.ERR_ARG
    for w in words:
        assert w in str(e.value)


def call(name, *args):
    """Status and message of a C entry point."""
    L = vm.lib()
    rc = getattr(L, name)(*args)
    return rc, L.vcsrmc_last_error().decode()


@pytest.mark.parametrize("cols", [1, 31, 32, 127, 128, 129, 511, 512, 513, 1000, 8192])
@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
def test_layout(cols, fmt):
    code, scale = ctypes.c_longlong(), ctypes.c_longlong()
    rc, _ = call("vcsrmc_mx_row_bytes", cols, mx.FORMATS[fmt], ctypes.byref(code),
                 ctypes.byref(scale))
    assert rc == vm.OK
    want = plain.pad(cols, 128) * mx.FORMATS[fmt] // 8, plain.pad(cols, 512) // 32
    assert (code.value, scale.value) == want == vm.mx_layout(cols, fmt)


def test_layout_refusals():
    refused(lambda: vm.mx_layout(0, "fp8"), "2^30")
    refused(lambda: vm.mx_layout((1 << 30) + 1, "fp8"))
    refused(lambda: vm.mx_layout(64, "fp6"), "fp4")
    out = ctypes.c_longlong()
    for cols, fmt in ((0, 8), (64, 6), (-1, 4)):
        rc, msg = call("vcsrmc_mx_row_bytes", cols, fmt, ctypes.byref(out), ctypes.byref(out))
        assert rc == vm.ERR_ARG and msg
    assert call("vcsrmc_mx_row_bytes", 64, 8, None, None)[0] == vm.ERR_ARG


def test_tensors_must_be_on_the_device():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    refused(lambda: vm.MXTensor(u8(2, 128), u8(2, 16), 128, "fp8"), "codes", "device")
    x = torch.zeros((2, 64))
    refused(lambda: vm.mx_quantise(x), "device")
    refused(lambda: vm.mx_quantise(x, "int8"), "fp4")
    refused(lambda: vm.rms_norm_mx(x, torch.ones(64)), "device")
    refused(lambda: vm.mx_matmul(x, x), "MXTensor")
    refused(lambda: vm.mx_moe(x, x, x, x, 1), "MXTensor")
    refused(lambda: vm.mx_dequantise(x), "MXTensor")


def test_torch_without_its_private_names(monkeypatch):
    """The module loads, and finds devices and streams by torch's public functions."""
    for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
        monkeypatch.delattr(torch._C, name, raising=False)
    spec = importlib.util.spec_from_file_location("vcsr_mc_amd.mx_again", mx.__file__)
    again = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(again)
    assert again._current_device is torch.cuda.current_device
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda device: types.SimpleNamespace(cuda_stream=70 + device))
    assert again._current_stream(2) == 72


def test_streams_of_another_device():
    """Refused, not passed over for that device's current stream."""
    other = types.SimpleNamespace(device=torch.device("cuda:1"))

    def enter():
        with mx._on(torch.device("cuda:0"), other):
            pass

    refused(enter, "stream", "cuda:1", "cuda:0")


A = 4096  # an address that is never read: every call below is refused first


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "null"), (dict(type=3), "type"), (dict(type=-1), "type"), (dict(rows=-1), "rows"),
    (dict(cols=0), "columns"), (dict(ldx=63), "stride"), (dict(fmt=5), "format"),
    (dict(codes=None), "codes"), (dict(scales=None), "codes"), (dict(codes=A + 8), "aligned"),
    (dict(x=A + 1), "aligned"), (dict(cols=(1 << 30) + 1, ldx=1 << 31), "columns")])
def test_quantise_refusals(change, word):
    a = dict(x=A, type=1, rows=2, cols=64, ldx=64, fmt=8, codes=A, scales=A) | change
    rc, msg = call("vcsrmc_mx_quantise", *a.values(), None)
    assert rc == vm.ERR_ARG and word in msg, msg
    a = dict(codes=A, scales=A, rows=2, cols=64, fmt=8, x=A, type=1, ldx=64) | change
    rc, msg = call("vcsrmc_mx_dequantise", *a.values(), None)
    assert rc == vm.ERR_ARG and word in msg, msg


@pytest.mark.parametrize("change,word", [
    (dict(weight=None), "weight"), (dict(wtype=2), "weight"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(ldr=10), "stride"), (dict(out=A, ldo=72), "stride"),
    (dict(out=2 * A, ldo=72), "stride"), (dict(x=None), "null"), (dict(fmt=0), "format"),
    (dict(weight=A + 1), "weight")])
def test_norm_refusals(change, word):
    a = dict(x=A, residual=2 * A, weight=A, type=1, wtype=1, rows=2, cols=64, ldx=64, ldr=64,
             eps=1e-6, out=None, ldo=64, fmt=8, codes=A, scales=A) | change
    rc, msg = call("vcsrmc_rms_norm_mx", *a.values(), None)
    assert rc == vm.ERR_ARG and word in msg, msg


@pytest.mark.parametrize("change,word", [
    (dict(xfmt=16), "format"), (dict(M=-1), "rows"), (dict(N=-3), "rows"), (dict(K=0), "columns"),
    (dict(xc=None), "codes"), (dict(ws=None), "codes"), (dict(wc=A + 4), "aligned"),
    (dict(out=None), "null"), (dict(type=9), "type"), (dict(ldo=31), "stride"),
    (dict(out=A + 1), "aligned"), (dict(K=(1 << 22) + 1), "columns")])
def test_matmul_refusals(change, word):
    a = dict(xc=A, xs=A, xfmt=8, M=2, wc=A, ws=A, N=32, K=64, out=A, type=1,
             ldo=32) | change
    rc, msg = call("vcsrmc_mx_matmul", *a.values(), None)
    assert rc == vm.ERR_ARG and word in msg, msg


@pytest.mark.parametrize("change,word", [
    (dict(T=-1), "rows"), (dict(D=0), "columns"), (dict(F=0), "size"), (dict(E=0), "experts"),
    (dict(E=1025), "experts"), (dict(k=0), "top_k"), (dict(k=9), "top_k"), (dict(renorm=2), "renorm"),
    (dict(router=None), "null"), (dict(rtype=4), "type"), (dict(w13c=None), "codes"),
    (dict(w2s=A + 1), "aligned"), (dict(out=None), "null"), (dict(type=7), "type"),
    (dict(ldo=8), "stride"), (dict(work=None), "workspace"), (dict(work=A + 16), "workspace"),
    (dict(bytes=10), "workspace"), (dict(E=65, k=65), "top_k"), (dict(F=(1 << 22) + 1), "size"),
    (dict(D=1301, F=3300000, ldo=1301), "codes")])
def test_moe_refusals(change, word):
    a = dict(xc=A, xs=A, T=2, D=64, router=A, rtype=0, E=8, w13c=A, w13s=A, F=32, w2c=A, w2s=A, k=2,
             renorm=1, out=A, type=2, ldo=64, work=A, bytes=1 << 40) | change
    rc, msg = call("vcsrmc_mx_moe", *a.values(), None)
    assert rc == vm.ERR_ARG and word in msg, msg


def test_plain_forms_agree_with_torch(rng):
    """The float64 definitions against torch's own E4M3 rounding, and the nearest-value rule of
    E2M1 by trial of all its values."""
    x = rng.standard_normal((6, 128)) * np.exp2(rng.integers(-6, 6, (6, 1)))
    c, s = plain.quantise(x, "fp8")
    v = x / np.repeat(np.ldexp(1.0, s.astype(int) - 127), 32, 1)
    t = torch.from_numpy(v).clamp(-448, 448).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(plain.values(c, np.full_like(s, 127), "fp8"), t)
    q = plain.grid(x, "fp4")
    _, s = plain.quantise(x, "fp4")
    step = np.repeat(np.ldexp(1.0, s.astype(int) - 127), 32, 1)
    grid = np.concatenate((plain.GRID["fp4"], -plain.GRID["fp4"]))
    best = np.abs(x[..., None] - grid * step[..., None]).min(-1)
    assert np.allclose(np.abs(x - q), best, rtol=0, atol=0)


@pytest.mark.parametrize("args", [["--top-k", "0"], ["--experts", "4", "--top-k", "5"], ["--tokens", "0"]])
def test_block_command_refuses(args, capsys):
    from vcsr_mc_amd import mx_block
    with pytest.raises(SystemExit) as e:
        mx_block.main(args)
    assert e.value.code == 2 and "top-k" in capsys.readouterr().err


def test_assembly_names_what_it_writes():
    """Every piece of inline assembly that sets m0 tells the compiler so."""
    csrc = pathlib.Path(vm.__file__).parent / "csrc"
    found = 0
    for path in sorted(csrc.glob("*.h*")):
        for piece in re.findall(r"\basm\b[^;]*?\((.*?)\);", path.read_text(), re.S):
            if re.search(r"\bs_mov_b32 m0\b", piece):
                found += 1
                assert '"m0"' in piece.rsplit(":", 1)[1], path.name
    assert found
