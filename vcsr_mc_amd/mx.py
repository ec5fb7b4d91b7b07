"""Microscaled (MX) operators: norms, products and mixtures of experts on operands in 4 and 8 bits.

What a layer of a language model needs when its weights are held in MXFP4: activations brought to
8 or 4 bits (``mx_quantise``, or ``rms_norm_mx`` with the residual's addition in the same pass),
their product with the weights (``mx_matmul``) and a whole mixture-of-experts layer for a few
tokens (``mx_moe``).  Thin wrappers of the C ABI (include/vcsrmc.h, "microscaled operators"): they
check their operands on the host, allocate what the caller does not give, and launch on ``stream``
(default: torch's current stream of the operands' device) without waiting.

``stream`` is a torch stream or the handle of any other.  Operands are to be ready on it (the caller
lets it wait for the streams that make them).  A caller may drop them at once where it is a torch
stream: their memory is kept for it.  Under the handle of another stream, or an ExternalStream of
it, the caller keeps them until the call has run.

For serving: nothing here has a gradient.  Where a result in 16 or 32 bits would lose one silently,
the operand that requires it is refused, as long as torch records gradients.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import functools

import torch

from . import ERR_ARG, VCSRMCError, _check, lib

FORMATS = {"fp4": 4, "fp8": 8}
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_EXPERTS, MAX_TOP_K = 1024, 64
# Without the checks and the objects of torch's public functions, which cost more than a small
# launch does; those serve where a torch lacks these.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                          lambda device: torch.cuda.current_stream(device).cuda_stream)
_U8 = torch.uint8


def _refuse(msg: str):
    raise VCSRMCError(ERR_ARG, msg)


def _no_gradient(what: str, *operands):
    """Refuses operands whose gradient a result would have to carry: none of these has one."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands):
        _refuse(f"{what} has no gradient: call under torch.no_grad(), or detach what requires one")


def _format(fmt) -> int:
    code = FORMATS.get(fmt)
    if code is None:
        _refuse(f"MX format must be 'fp4' or 'fp8', not {fmt!r}")
    return code


@functools.lru_cache(maxsize=4096)
def mx_layout(cols: int, fmt: str) -> tuple[int, int]:
    """(bytes of codes, bytes of scales) of one row of `cols` values."""
    bits, cols = _format(fmt), int(cols)
    if not 1 <= cols <= 1 << 30:
        _refuse(f"MX rows hold 1 to 2^30 values, not {cols}")
    return (cols + 127) // 128 * 128 * bits // 8, (cols + 511) // 512 * 16


class MXTensor:
    """Rows of `cols` values in an MX format: `codes` (..., rows, code bytes) and `scales`
    (..., rows, scale bytes), contiguous uint8 device tensors as ``mx_layout`` sizes them.  Leading
    dimensions are free; ``rows`` is the product of all but the last."""

    __slots__ = ("codes", "scales", "cols", "fmt", "rows", "bits")

    def __init__(self, codes, scales, cols: int, fmt: str):
        cb, sb = mx_layout(cols, fmt)
        cs, ss = codes.shape, scales.shape
        if codes.dtype is not _U8 or not codes.is_cuda or not codes.is_contiguous() \
                or len(cs) < 2 or cs[-1] != cb:
            _refuse(f"codes must be a contiguous uint8 device tensor with rows of {cb} bytes")
        if scales.dtype is not _U8 or not scales.is_contiguous() or ss[-1:] != (sb,):
            _refuse(f"scales must be a contiguous uint8 device tensor with rows of {sb} bytes")
        if cs[:-1] != ss[:-1] or codes.get_device() != scales.get_device():
            _refuse("codes and scales must have the same rows, on the same GPU")
        self.codes, self.scales, self.cols, self.fmt = codes, scales, int(cols), fmt
        self.rows = codes.numel() // cb
        self.bits = FORMATS[fmt]

    @classmethod
    def empty(cls, shape, fmt: str, device="cuda") -> "MXTensor":
        """An uninitialised MX tensor of `shape` (..., rows, cols)."""
        *lead, cols = shape
        cb, sb = mx_layout(cols, fmt)
        codes = torch.empty((*lead, cb), dtype=_U8, device=device)
        return cls(codes, torch.empty((*lead, sb), dtype=_U8, device=device), cols, fmt)

    @classmethod
    def _new(cls, x, rows: int, cols: int, fmt: str) -> "MXTensor":
        """An uninitialised rows x cols tensor beside x, with nothing to check."""
        cb, sb = mx_layout(cols, fmt)
        q = object.__new__(cls)
        q.codes = x.new_empty((rows, cb), dtype=_U8)
        q.scales = x.new_empty((rows, sb), dtype=_U8)
        q.cols, q.fmt, q.rows, q.bits = cols, fmt, rows, FORMATS[fmt]
        return q

    @classmethod
    def from_blocks(cls, codes, scales, cols: int, fmt: str) -> "MXTensor":
        """From unpadded rows (a checkpoint's): codes (..., rows, ceil(cols * bits / 8)) and one
        scale byte a block, (..., rows, ceil(cols / 32)).  Copies only where rows need padding."""
        cb, sb = mx_layout(cols, fmt)
        bits = FORMATS[fmt]
        want = ((cols * bits + 7) // 8, (cols + 31) // 32)
        if codes.shape[-1] != want[0] or scales.shape[-1] != want[1]:
            _refuse(f"unpadded rows of {cols} values hold {want[0]} code and {want[1]} scale bytes")
        pad = torch.nn.functional.pad
        codes, scales = codes.contiguous(), scales.contiguous()
        if bits == 4 and cols % 2:  # the last byte's upper nibble lies past the row
            codes = codes.clone()
            codes[..., -1] &= 15
        if codes.shape[-1] != cb:
            codes = pad(codes, (0, cb - codes.shape[-1]))
        if scales.shape[-1] != sb:
            scales = pad(scales, (0, sb - scales.shape[-1]))
        return cls(codes, scales, cols, fmt)

    @property
    def shape(self):
        return (*self.codes.shape[:-1], self.cols)

    @property
    def device(self):
        return self.codes.device

    def __repr__(self):
        return f"MXTensor(shape={tuple(self.shape)}, fmt={self.fmt!r}, device={self.device})"


@contextlib.contextmanager
def _on(device, stream, *operands):
    """`device` and `stream` current: what is allocated inside belongs to that stream, and what the
    caller frees of the operands is not used again before that stream has passed the call.  The
    entry points enter it only where they are not current already: it costs more than a small
    launch."""
    if getattr(stream, "device", device) != device:
        _refuse(f"the stream is of {stream.device}, the operands are on {device}")
    with torch.cuda.device(device):
        given = stream
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=device)
        with torch.cuda.stream(stream):
            yield
        # a stream that is not torch's may be gone when the operand is freed: its owner keeps them
        if isinstance(given, torch.cuda.Stream) and not isinstance(given, torch.cuda.ExternalStream):
            for t in operands:
                for part in (t.codes, t.scales) if isinstance(t, MXTensor) else (t,):
                    if part is not None:
                        part.record_stream(given)


def _matrix(t, name: str, rows: int | None = None, cols: int | None = None, like=None):
    """Checks a plain 2-D device matrix with unit column stride; returns its row stride.  like: a
    tensor whose GPU it has to share."""
    shape = t.shape
    if len(shape) != 2 or not t.is_cuda or t.dtype not in TYPES:
        _refuse(f"{name} must be a 2-D float32, float16 or bfloat16 device tensor")
    r, c = shape
    if rows is not None and (r != rows or c != cols):
        _refuse(f"{name} must be {rows} x {cols}, not {r} x {c}")
    if like is not None and t.get_device() != like.get_device():
        _refuse(f"{name} must be on {like.device}")
    if c and t.is_contiguous():
        return c
    ld, step = t.stride()
    if c == 0 or (c > 1 and step != 1):
        _refuse(f"{name} must have contiguous, non-empty rows")
    if r <= 1:
        return c
    if ld < c:
        _refuse(f"{name}'s rows overlap")
    return ld


def _mx(q, name: str, fmt: str | None = None):
    if not isinstance(q, MXTensor):
        _refuse(f"{name} must be an MXTensor")
    if fmt is not None and q.fmt != fmt:
        _refuse(f"{name} must be in {fmt}, not {q.fmt}")


def _mx_out(out, rows: int, cols: int, fmt: str, like):
    if out is None:
        return MXTensor._new(like, rows, cols, fmt)
    _mx(out, "out", fmt)
    if out.rows != rows or out.cols != cols or out.codes.get_device() != like.get_device():
        _refuse(f"out must hold {rows} x {cols} values on {like.device}")
    return out


def _plain_out(out, rows: int, cols: int, dtype, like):
    if out is None:
        if dtype not in TYPES:
            _refuse("dtype must be float32, float16 or bfloat16")
        return like.new_empty((rows, cols), dtype=dtype), cols
    return out, _matrix(out, "out", rows, cols, like)


def mx_quantise(x, fmt: str = "fp8", out: MXTensor | None = None, stream=None) -> MXTensor:
    """MX form of x (rows x cols, float32/float16/bfloat16, any row stride)."""
    bits = _format(fmt)
    ld = _matrix(x, "x")
    at = x.get_device()
    if stream is not None or at != _current_device():
        with _on(x.device, stream, x, out):
            return mx_quantise(x, fmt, out)
    rows, cols = x.shape
    q = _mx_out(out, rows, cols, fmt, x)
    rc = lib().vcsrmc_mx_quantise(x.data_ptr(), TYPES[x.dtype], rows, cols, ld, bits,
                                  q.codes.data_ptr(), q.scales.data_ptr(), _current_stream(at))
    if rc:
        _check(rc, "mx_quantise")
    return q


def mx_dequantise(q: MXTensor, dtype=torch.float32, out=None, stream=None):
    """The values of q as a (q.rows, q.cols) matrix."""
    _mx(q, "q")
    at = q.codes.get_device()
    if stream is not None or at != _current_device():
        with _on(q.device, stream, q, out):
            return mx_dequantise(q, dtype, out)
    o, ld = _plain_out(out, q.rows, q.cols, dtype, q.codes)
    rc = lib().vcsrmc_mx_dequantise(q.codes.data_ptr(), q.scales.data_ptr(), q.rows, q.cols, q.bits,
                                    o.data_ptr(), TYPES[o.dtype], ld, _current_stream(at))
    if rc:
        _check(rc, "mx_dequantise")
    return o


def rms_norm_mx(x, weight, residual=None, eps: float = 1e-6, fmt: str = "fp8",
                out: MXTensor | None = None, residual_out=None, stream=None):
    """(MX of h / sqrt(mean(h^2) + eps) * weight, h) with h = x + residual, row by row in 32 bits;
    the second is h rounded to x's type, None without a residual.  residual_out may be x or
    residual themselves.  h carries no gradient: under a residual, x and residual that require one
    are refused."""
    bits = _format(fmt)
    ldx = _matrix(x, "x")
    rows, cols = x.shape
    at, dtype = x.get_device(), x.dtype
    if weight.shape != (cols,) or weight.get_device() != at or not weight.is_contiguous() \
            or (weight.dtype is not dtype and weight.dtype is not torch.float32):
        _refuse(f"weight must hold {cols} values of x's type or float32 on {x.device}")
    ldr = ldo = cols
    if residual is not None:
        ldr = _matrix(residual, "residual", rows, cols, x)
        if residual.dtype is not dtype:
            _refuse("residual must have x's type")
        _no_gradient("rms_norm_mx's sum", x, residual)
        if residual_out is not None:
            ldo = _matrix(residual_out, "residual_out", rows, cols, x)
            if residual_out.dtype is not dtype:
                _refuse("residual_out must have x's type")
    elif residual_out is not None:
        _refuse("residual_out needs a residual")
    if stream is not None or at != _current_device():
        with _on(x.device, stream, x, weight, residual, out, residual_out):
            return rms_norm_mx(x, weight, residual, eps, fmt, out, residual_out)
    q = _mx_out(out, rows, cols, fmt, x)
    h = residual_out
    if residual is not None and h is None:
        h = x.new_empty((rows, cols))
    rc = lib().vcsrmc_rms_norm_mx(
        x.data_ptr(), None if residual is None else residual.data_ptr(), weight.data_ptr(),
        TYPES[dtype], TYPES[weight.dtype], rows, cols, ldx, ldr, eps,
        None if h is None else h.data_ptr(), ldo, bits, q.codes.data_ptr(), q.scales.data_ptr(),
        _current_stream(at))
    if rc:
        _check(rc, "rms_norm_mx")
    return q, h


@functools.lru_cache(maxsize=4096)
def _moe_workspace(T: int, D: int, F: int, E: int, k: int) -> int:
    need = C.c_longlong()
    _check(lib().vcsrmc_mx_moe_workspace(T, D, F, E, k, C.byref(need)), "mx_moe")
    return need.value


def mx_matmul(x: MXTensor, w: MXTensor, dtype=torch.bfloat16, out=None, stream=None):
    """X.W^T (x.rows x w.rows), x in fp8 or fp4, w in fp4.  Sums are in 32 bits, but for an x in fp8
    the matrix cores add the products of 8 consecutive values cut to multiples of 2^-13 of the
    binade of the largest: near 4e-6 of the result for normal values, at most 7 * 2^-13 of
    sum |x||w|."""
    _mx(x, "x")
    _mx(w, "w", "fp4")
    xc, wc, M, N, K = x.codes, w.codes, x.rows, w.rows, x.cols
    at = xc.get_device()
    if K != w.cols or at != wc.get_device():
        _refuse(f"x has rows of {K} values on {x.device}, w of {w.cols} on {w.device}")
    if stream is not None or at != _current_device():
        with _on(x.device, stream, x, w, out):
            return mx_matmul(x, w, dtype, out)
    if N == 0:
        return xc.new_empty((M, 0), dtype=dtype)
    o, ld = _plain_out(out, M, N, dtype, xc)
    rc = lib().vcsrmc_mx_matmul(xc.data_ptr(), x.scales.data_ptr(), x.bits, M, wc.data_ptr(),
                                w.scales.data_ptr(), N, K, o.data_ptr(), TYPES[o.dtype], ld,
                                _current_stream(at))
    if rc:
        _check(rc, "mx_matmul")
    return o


def mx_moe(x: MXTensor, router, w13: MXTensor, w2: MXTensor, top_k: int, renormalise: bool = True,
           dtype=torch.bfloat16, out=None, stream=None):
    """A mixture-of-experts layer: x (T x D, fp8), router (E x D), w13 (E x 2F x D, fp4: F gate
    rows, then F up rows) and w2 (E x D x F, fp4).  Each token's top_k experts by router . x (ties
    to the lower index), weighted by softmax over them (renormalise) or over all experts.  For
    decoding batches: tokens are taken 64 at a time, each time with the weights of their experts.
    Logits, gate and up sums keep 32 bits; the down rows' are as mx_matmul's with fp8.
    No gradient: a router that requires one is refused."""
    _mx(x, "x", "fp8")
    _mx(w13, "w13", "fp4")
    _mx(w2, "w2", "fp4")
    T, D, F, top_k = x.rows, x.cols, w2.cols, int(top_k)
    xc, w13c, w2c, rs = x.codes, w13.codes, w2.codes, router.shape
    if len(rs) != 2 or rs[1] != D or router.dtype not in TYPES or not router.is_contiguous():
        _refuse(f"router must be a contiguous E x {D} float32, float16 or bfloat16 tensor")
    E = rs[0]
    if w13c.shape[:-1] != (E, 2 * F) or w13.cols != D or w2c.shape[:-1] != (E, D):
        _refuse(f"w13 must be {E} x {2 * F} x {D} and w2 {E} x {D} x {F}, not "
                f"{tuple(w13.shape)} and {tuple(w2.shape)}")
    at = xc.get_device()
    if not at == router.get_device() == w13c.get_device() == w2c.get_device():
        _refuse("x, router, w13 and w2 must be on the same GPU")
    _no_gradient("mx_moe", router)
    if not 1 <= E <= MAX_EXPERTS or not 1 <= top_k <= min(E, MAX_TOP_K):
        _refuse(f"experts must be 1 to {MAX_EXPERTS} and top_k 1 to experts (at most {MAX_TOP_K}), "
                f"not {E} and {top_k}")
    if stream is not None or at != _current_device():
        with _on(x.device, stream, x, router, w13, w2, out):
            return mx_moe(x, router, w13, w2, top_k, renormalise, dtype, out)
    o, ld = _plain_out(out, T, D, dtype, xc)
    need = _moe_workspace(T, D, F, E, top_k)
    ws = xc.new_empty((need,))
    rc = lib().vcsrmc_mx_moe(
        xc.data_ptr(), x.scales.data_ptr(), T, D, router.data_ptr(), TYPES[router.dtype], E,
        w13c.data_ptr(), w13.scales.data_ptr(), F, w2c.data_ptr(), w2.scales.data_ptr(), top_k,
        1 if renormalise else 0, o.data_ptr(), TYPES[o.dtype], ld, ws.data_ptr(), need,
        _current_stream(at))
    if rc:
        _check(rc, "mx_moe")
    return o
