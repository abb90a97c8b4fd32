"""AdamW with moments in 8 bits, in numpy. Test infrastructure only. The step between the codes is adamw_ref's."""
import numpy as np

from .adamw_ref import adamw_step_div, adamw_step_ibc
from .bf16_ref import bf16_rne_bits, bf16_sr_bits

STATE_SEED = 0x3C6EF372


def sr_hash(i, seed):
    """The 32 bits whose low half is bf16_ref.sr_dither(i // 64, i % 64, seed)."""
    mask = np.uint64(0xFFFFFFFF)
    i = np.asarray(i, np.uint64)
    h = ((i >> np.uint64(6)) * np.uint64(73856093) & mask) ^ ((i & np.uint64(63)) * np.uint64(19349663) & mask) ^ np.uint64(int(seed) & 0xFFFFFFFF)
    h = h * np.uint64(0x9E3779B1) & mask
    h ^= h >> np.uint64(16)
    h = h * np.uint64(0x85EBCA6B) & mask
    return (h ^ (h >> np.uint64(13))).astype(np.int64)


def values(mantissa):
    """Magnitudes of the codes 0 .. 126 (E4M3: 3 mantissa bits) or 0 .. 123 (E5M2: 2)."""
    n = 127 if mantissa == 3 else 124
    e, m = np.divmod(np.arange(n), 1 << mantissa)
    bias = 7 if mantissa == 3 else 15
    return np.where(e == 0, m * 2.0 ** (1 - bias - mantissa), (1 + m * 2.0 ** -mantissa) * 2.0 ** (e - bias))


def decode(codes, scales, mantissa):
    """fp32 values of codes (R, 64) with scale bytes (R,); codes beyond the finite ones are NaN."""
    v = np.full(128, np.nan)
    t = values(mantissa)
    v[:t.size] = t
    codes = np.asarray(codes)
    x = np.where(codes & 0x80, -v[codes & 0x7F], v[codes & 0x7F])
    return (x * np.exp2(np.asarray(scales, np.float64) - 127)[:, None]).astype(np.float32)


def encode(x, mantissa, dither):
    """(codes, scales) of fp32 x (R, 64): by search among the format's values. The lower neighbour, plus one where the
    magnitude's place between the neighbours and dither / 2^16 make one or more."""
    x = np.asarray(x, np.float32)
    top, table = (7, values(3)) if mantissa == 3 else (14, values(2))
    a = np.abs(x)
    fin = np.isfinite(a)
    amax = np.where(fin, a, 0).max(1)
    _, e = np.frexp(amax.astype(np.float64))
    byte = np.where(amax > 0, np.maximum(e - 1 + 127 - top, 1), 1).astype(np.int64)
    y = np.where(fin, a, 0).astype(np.float64) * np.exp2(127.0 - byte)[:, None]
    at = np.clip(np.searchsorted(table, y, side="right") - 1, 0, table.size - 2)
    place = (y - table[at]) / (table[at + 1] - table[at])
    codes = at + (place * 65536.0 + dither >= 65536.0)
    codes = np.where(fin, codes, 0x7F) | (np.signbit(x).astype(np.int64) << 7)
    return codes.astype(np.uint8), byte.astype(np.uint8)


class Tensor8:
    """One tensor's state; `step` is one step with seed (seed_base + the tensor's own)."""

    def __init__(self, p):
        self.p = np.asarray(p, np.float32).reshape(-1, 64).copy()
        R = self.p.shape[0]
        self.m, self.v = np.zeros((R, 64), np.uint8), np.zeros((R, 64), np.uint8)
        self.ms, self.vs = np.zeros(R, np.uint8), np.zeros(R, np.uint8)

    def step(self, g, lr, b1, b2, eps, wd, t, seed, sr=False, clip=1.0, form="div"):
        m, v = decode(self.m, self.ms, 3), decode(self.v, self.vs, 2)
        g = np.asarray(g, np.float32).reshape(-1, 64)
        with np.errstate(all="ignore"):
            if form == "div":
                self.p, m, v = adamw_step_div(self.p, m, v, g, lr, b1, b2, eps, wd, t, clip)
            else:
                self.p, m, v = adamw_step_ibc(self.p, m, v, g, lr, b1, b2, eps, wd, 1 / (1 - b1 ** t), 1 / (1 - b2 ** t), clip)
        h = sr_hash(np.arange(self.p.size), (int(seed) ^ STATE_SEED) & 0xFFFFFFFF).reshape(-1, 64)
        self.m, self.ms = encode(m, 3, h & 0xFFFF)
        self.v, self.vs = encode(v, 2, h >> 16)
        self.v = np.where((v > 0) & (self.v == 0), 1, self.v).astype(np.uint8)
        self.p16 = bf16_sr_bits(self.p, seed) if sr else bf16_rne_bits(self.p).reshape(-1, 64)
