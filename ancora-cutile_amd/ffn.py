"""The gated feed-forward block (SwiGLU) on the MI355X, dense or over tokens that a `dispatch.RoutePlan` has sorted by expert: the products
between `dispatch` and `combine`, and the operands of the weight gradients (`grads.gemm_dW`, `grads.expert_dW`) on the way back.

    gated_ffn(x, Wg, Wu, si, h, gate=g, up=u, plan=plan)               # h = silu(x Wg) * (x Wu); g, u kept for the backward pass
    ffn_down(h, Wd, si, y, residual=None, plan=plan)                    # y = h Wd (+ residual)
    gated_ffn_grad(dy, g, u, Wd, si, dg, du, h=h, plan=plan)            # dg, du, and h once more for dWd
    gated_ffn_dx(dg, du, Wg, Wu, si, dx, plan=plan)                     # dx = dg Wg^T + du Wu^T (+ residual)
    expert_dW(plan, [dict(x=x, dy=dg, dW=dWg), dict(x=x, dy=du, dW=dWu), dict(x=h, dy=dy, dW=dWd)], si)

Weights are the bf16 copies that the optimizer refreshes, as they lie: (H, I) and (I, H), stacked per expert (E, H, I) or (E*H, I) with a
plan; no transposed copies are read. Mirrors SwiGLU and the grouped products of the reference's layers (ancora/kernels/activation.py,
ancora/kernels/moe.py). Products accumulate in fp32, each output is rounded once (h, dgate and dup in between too: they are
the caller's bf16 buffers). Without a plan every row of x is a row of the product; with
one, rows that fill up a segment or lie behind the last are neither read nor written. Each call may be captured into a graph, whose replays then
work on no more tokens than the plan held at the capture (`plan.active`), as its routing and dispatch do.
"""
import numpy as np

from . import _lib
from ._lib import api
from .embed import _type

_BITS = np.dtype(np.uint16)          # bf16 (buffers hold dtypes: comparing with a type costs each check 0.1 us)


def _call(who, rows_name, rows_buf, plan):
    """(rows, rows that are tokens' at most, experts, counts, offsets) of a call whose first operand is rows_buf (rows, K)."""
    if len(rows_buf.shape) != 2 or rows_buf.dtype != _BITS:
        raise ValueError(f"{who}: {rows_name} is {rows_buf.shape} {rows_buf.dtype}, rows of bf16 bits expected")
    if plan is None:
        return rows_buf.shape[0], rows_buf.shape[0], 0, 0, 0
    plan._used(who)
    counts, offsets = plan._at[:2]
    return plan.capacity, plan.active * plan.k, plan.E, counts, offsets


def _rows(who, name, b, rows, width, dtype=_BITS):
    if b is None:
        return 0
    shape = b.shape
    if len(shape) != 2 or shape[0] < rows or shape[1] != width or (dtype is not None and b.dtype != dtype):
        raise ValueError(f"{who}: {name} is {b.shape} {b.dtype}, ({rows}, {width}) "
                         f"{'of bf16 bits' if dtype == _BITS else '' if dtype is None else dtype} expected")
    return b.ptr


def _weight(who, name, w, E, K, N):
    shape, n = w.shape, E or 1
    if w.dtype != _BITS or (shape != (n * K, N) and shape != (n, K, N)):
        raise ValueError(f"{who}: {name} is {w.shape} {w.dtype}, {(E, K, N) if E else (K, N)} of bf16 bits expected")
    return w.ptr


def _dims(who, H, I):
    if H % 8 or I % 8:
        raise ValueError(f"{who}: widths {H} and {I} must be multiples of 8")


def _residual(who, residual, y, rows, width):
    _rows(who, "the result", y, rows, width, None)
    kind = _type(y, who)
    if residual is None:
        return 0, kind
    return _rows(who, "residual", residual, rows, width, y.dtype), kind


def gated_ffn(x, Wg, Wu, si, h, gate=None, up=None, plan=None):
    """h = silu(x Wg) * (x Wu): x (rows, H), Wg and Wu (H, I) or (E, H, I), h (rows, I), all bf16 bits; gate and up (rows, I)
    receive x Wg and x Wu where a backward pass will want them. With a plan rows is its capacity. Asynchronous on `si`."""
    who = "gated_ffn"
    rows, tokens, E, counts, offsets = _call(who, "x", x, plan)
    H, I = x.shape[1], h.shape[-1]
    _dims(who, H, I)
    api.anc_gated_ffn(_rows(who, "x", x, rows, H), _weight(who, "Wg", Wg, E, H, I), _weight(who, "Wu", Wu, E, H, I), counts, offsets, E,
                      rows, tokens, H, I, _rows(who, "h", h, rows, I), _rows(who, "gate", gate, rows, I), _rows(who, "up", up, rows, I), int(si))


def ffn_down(h, Wd, si, y, residual=None, plan=None):
    """y = h Wd + residual: h (rows, I) and Wd (I, H) or (E, I, H) bf16 bits; y (rows, H) and residual (or None) of one type, float32 or
    bf16 bits. residual may be y itself. Asynchronous on `si`."""
    who = "ffn_down"
    rows, tokens, E, counts, offsets = _call(who, "h", h, plan)
    I, H = h.shape[1], y.shape[-1]
    _dims(who, H, I)
    res, kind = _residual(who, residual, y, rows, H)
    api.anc_ffn_down(_rows(who, "h", h, rows, I), _weight(who, "Wd", Wd, E, I, H), counts, offsets, E, rows, tokens, I, H, res, y.ptr, kind, int(si))


def gated_ffn_grad(dy, gate, up, Wd, si, dgate, dup, h=None, plan=None):
    """From the gradient dy (rows, H) of the block's result to those of the pre-activations: with dh = dy Wd^T and
    s = sigmoid(gate), dgate = dh up s (1 + gate (1 - s)), dup = dh gate s, and h = gate s up where asked for (dWd = h^T dy): of gate and up as they were
    kept, rounded, so not the bits of the h that `gated_ffn` made before it rounded them; a caller who wants those in dWd keeps that h. gate, up, dgate,
    dup, h (rows, I) bf16 bits; dgate may be gate and dup up. Asynchronous on `si`."""
    who = "gated_ffn_grad"
    rows, tokens, E, counts, offsets = _call(who, "dy", dy, plan)
    H, I = dy.shape[1], gate.shape[-1]
    _dims(who, H, I)
    api.anc_gated_ffn_grad(_rows(who, "dy", dy, rows, H), _weight(who, "Wd", Wd, E, I, H), _rows(who, "gate", gate, rows, I),
                           _rows(who, "up", up, rows, I), counts, offsets, E, rows, tokens, H, I, _rows(who, "dgate", dgate, rows, I),
                           _rows(who, "dup", dup, rows, I), _rows(who, "h", h, rows, I), int(si))


def gated_ffn_dx(dgate, dup, Wg, Wu, si, dx, residual=None, plan=None):
    """dx = dgate Wg^T + dup Wu^T + residual: dgate and dup (rows, I), Wg and Wu (H, I) or (E, H, I) bf16 bits; dx (rows, H) and residual (the
    gradient along the residual stream, or None) of one type, float32 or bf16 bits. residual may be dx itself. Asynchronous on `si`."""
    who = "gated_ffn_dx"
    rows, tokens, E, counts, offsets = _call(who, "dgate", dgate, plan)
    I, H = dgate.shape[1], dx.shape[-1]
    _dims(who, H, I)
    res, kind = _residual(who, residual, dx, rows, H)
    api.anc_gated_ffn_dx(_rows(who, "dgate", dgate, rows, I), _rows(who, "dup", dup, rows, I), _weight(who, "Wg", Wg, E, H, I),
                         _weight(who, "Wu", Wu, E, H, I), counts, offsets, E, rows, tokens, H, I, res, dx.ptr, kind, int(si))
