"""A layer's norm and gated feed-forward block in 64 bits, and rows in MXFP8. Test infrastructure only."""
import numpy as np

from .quant_ref import e4m3_rne

f64 = np.float64


def rms_norm(s, gain, eps):
    """(rows, r) of s (T, H): s r gain with r = 1 / sqrt(mean(s^2) + eps)."""
    s = np.asarray(s, f64)
    r = 1.0 / np.sqrt((s * s).mean(1) + eps)
    return s * r[:, None] * gain, r


def rms_norm_grad(dy, s, gain, r):
    """(ds, dgain) for the norm's inputs s, gain and its r."""
    dy, s, r = np.asarray(dy, f64), np.asarray(s, f64), np.asarray(r, f64)[:, None]
    a, xh = dy * gain, s * r
    return r * (a - xh * (a * xh).mean(1, keepdims=True)), (dy * xh).sum(0)


def mx8_rows(y):
    """fp32 rows (T, H) -> (codes (T, H), scale bytes (T, H // 32)) by the rule of quant_ref.quant_mxfp8_w with the blocks along the row;
    elements that are not finite get the NaN code and count as infinitely large."""
    y = np.ascontiguousarray(y, np.float32)
    b = y.reshape(y.shape[0], -1, 32)
    ea = ((b.view(np.uint32) & 0x7FFFFFFF).max(2) >> 23).astype(np.int64)
    byte = np.where(ea >= 7, ea - 7, 0)
    with np.errstate(invalid="ignore", over="ignore"):
        codes = e4m3_rne(b.astype(f64) * np.exp2(127.0 - byte)[:, :, None])
    return codes.reshape(y.shape), byte.astype(np.uint8)


def sigmoid(g):
    return np.where(g >= 0, 1.0 / (1.0 + np.exp(-np.abs(g))), np.exp(-np.abs(g)) / (1.0 + np.exp(-np.abs(g))))


def by_segment(x, W, counts=None, offsets=None):
    """x W per row; with counts and offsets W is stacked by expert and rows outside the segments are zero."""
    x, W = np.asarray(x, f64), np.asarray(W, f64)
    if counts is None:
        return x @ W
    out = np.zeros((x.shape[0], W.shape[2]))
    for e, (c, o) in enumerate(zip(counts, offsets)):
        out[o:o + c] = x[o:o + c] @ W[e]
    return out


def gated(g, u):
    return g * sigmoid(g) * u


def gated_grad(dh, g, u):
    """(dg, du, h)."""
    s = sigmoid(g)
    return dh * u * s * (1.0 + g * (1.0 - s)), dh * g * s, g * s * u
