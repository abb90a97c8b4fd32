"""Root-mean-square norm with the residual's addition, its rows in 32, 16 or 8 bits, and its backward pass, on the MI355X: what stands in
front of the products whose weights the step updates (RMSNorm, ancora/kernels/norm.py), and the gradient of the gains that AdamW steps.

    rms_norm(x, gain, si, y=y, residual=res, total=res2, rstd=r)        # res2 = x + res, y = res2 * r * gain
    rms_norm_grad(dy, res2, gain, r, si, dx, dgain, workspace, carry=dres)   # dx = gradient of res2 through the norm, + dres

8-bit rows (`fp8=`, `scale=` instead of `y=`) are MXFP8 as `Mxfp8WeightCache` holds the weights, blocks of 32 along the row, for a product over it that the
caller brings: the products here take bf16. Arithmetic is fp32 with one rounding per output.
"""
from . import _lib
from ._lib import api
from .devbuf import DevBuf
from .embed import _rows_of, _type

import numpy as np

B = 32          # MXFP8 scale block


def _gain(gain, H, who):
    if gain.size != H:
        raise ValueError(f"{who}: gain has {gain.size} elements, rows have {H}")
    return _type(gain, who)


def _rstd(rstd, T, who):
    if rstd.dtype != np.float32 or rstd.size < T:
        raise ValueError(f"{who}: rstd is {rstd.shape} {rstd.dtype}, ({T},) float32 expected")
    return rstd.ptr


def rms_norm(x, gain, si, y=None, residual=None, total=None, fp8=None, scale=None, rstd=None, eps=1e-6):
    """s = x + residual (or x), r = 1 / sqrt(mean(s^2) + eps) per row, result s * r * gain. x (T, H), gain (H,): float32 or bf16 bits;
    residual and total (s itself, rounded to their type; given together): float32 or bf16 bits, of one type. The result goes to y
    (T, H), float32 or bf16 bits, or to fp8 (T, H) and scale (T, H / 32) uint8. rstd (T,) float32 receives r for `rms_norm_grad`. H is
    a multiple of 8 (32 with fp8) up to 16384; a row whose squares add up beyond fp32 (values of 2^64 / sqrt(H)) becomes zeros. y or total may be x or residual itself; other overlaps are refused. Asynchronous on `si`."""
    T, H = x.shape if len(x.shape) == 2 else (-1, -1)
    if T < 0:
        raise ValueError(f"rms_norm: x is {x.shape}, (T, H) expected")
    if (y is None) == (fp8 is None) or (fp8 is None) != (scale is None):
        raise ValueError("rms_norm: either y, or fp8 and scale")
    if (residual is None) != (total is None):
        raise ValueError("rms_norm: residual and total go together")
    stream = _lib.BF16
    if residual is not None:
        _rows_of(residual, T, H, "rms_norm", "residual")
        _rows_of(total, T, H, "rms_norm", "total")
        stream = _type(residual, "rms_norm")
        if total.dtype != residual.dtype:
            raise ValueError(f"rms_norm: residual is {residual.dtype}, total {total.dtype}")
    if fp8 is None:
        _rows_of(y, T, H, "rms_norm", "y")
        out, kind, sc = y.ptr, _type(y, "rms_norm"), 0
    else:
        if H % B:
            raise ValueError(f"rms_norm: 8-bit rows of {H}: a multiple of {B}")
        _rows_of(fp8, T, H, "rms_norm", "fp8")
        _rows_of(scale, T, H // B, "rms_norm", "scale")
        if fp8.dtype != np.uint8 or scale.dtype != np.uint8:
            raise ValueError(f"rms_norm: fp8 is {fp8.dtype}, scale {scale.dtype}, uint8 expected")
        out, kind, sc = fp8.ptr, _lib.MXFP8, scale.ptr
    api.anc_rms_norm(x.ptr, _type(x, "rms_norm"), 0 if residual is None else residual.ptr, stream, gain.ptr, _gain(gain, H, "rms_norm"), T, H,
                     float(eps), out, kind, sc, 0 if total is None else total.ptr, 0 if rstd is None else _rstd(rstd, T, "rms_norm"), int(si))


class NormWorkspace:
    """Scratch of `rms_norm_grad` for rows of H, `rows` of them at most. One call at a time: work that overlaps on other streams (or replays
    of graphs) takes one each."""

    def __init__(self, rows, H):
        _lib.init()
        self.rows, self.H = int(rows), int(H)
        n = api.anc_rms_norm_grad_workspace_bytes(self.rows, self.H)
        if n < 0:
            raise ValueError("NormWorkspace: " + _lib.load().anc_last_error().decode())
        self.buf = DevBuf.empty((n // 4,), np.float32)

    def free(self):
        self.buf.free()


def rms_norm_grad(dy, x, gain, rstd, si, dx, dgain, workspace, carry=None, accumulate=False):
    """Gradients of `rms_norm` at what it normed: x is its `total` (or its x without residual), rstd its r. With a = dy * gain:
    dx = r * (a - x * r^2 * mean(a * x)) + carry, dgain (+)= the sum over rows of dy * x * r (fp32, `accumulate` adds onto it). dy
    (T, H) float32 or bf16 bits; x, dx and carry (the gradient that comes along the residual stream) of one type. dx may be dy, x or
    carry itself. The sum over rows is in a fixed order that hangs on T and H alone. Asynchronous on `si`."""
    who = "rms_norm_grad"
    T, H = dy.shape if len(dy.shape) == 2 else (-1, -1)
    if T < 0:
        raise ValueError(f"{who}: dy is {dy.shape}, (T, H) expected")
    for name, b in (("x", x), ("dx", dx), ("carry", carry)):
        if b is not None:
            _rows_of(b, T, H, who, name)
            if b.dtype != x.dtype:
                raise ValueError(f"{who}: {name} is {b.dtype}, x {x.dtype}")
    if dgain.dtype != np.float32 or dgain.size != H:
        raise ValueError(f"{who}: dgain is {dgain.shape} {dgain.dtype}, ({H},) float32 expected")
    api.anc_rms_norm_grad(dy.ptr, _type(dy, who), x.ptr, _type(x, who), gain.ptr, _gain(gain, H, who), _rstd(rstd, T, who),
                          0 if carry is None else carry.ptr, T, H, dx.ptr, dgain.ptr, int(bool(accumulate)), workspace.buf.ptr,
                          workspace.buf.nbytes, int(si))
