"""The norm and the feed-forward block where rows lie behind 2^31 elements: rows at the start, around that line and at the end hold values, all others zeros.

Bounds as in the tests of the single operators."""
import numpy as np
import pytest

from oracle import layer_ref as ref
from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from test_gpu_expert_dw import _plan_of
from util import bits_equal

pytestmark = pytest.mark.gpu
U16, F32 = np.uint16, np.float32
UNIT = 2.0 ** -23


def _bits(rng, shape, std=1.0):
    return bf16_rne_bits((std * rng.standard_normal(shape)).astype(F32)).reshape(shape)


def _wide(b):
    return bits_to_f32(b).reshape(b.shape).astype(np.float64)


def _row(buf, row):
    from ancora_cutile_amd import DevBuf
    return DevBuf(shape=(1, buf.shape[1]), dtype=buf.dtype, ptr=buf.ptr + row * buf.shape[1] * buf.dtype.itemsize)


def _put(buf, rows, values):
    for r, v in zip(rows, values):
        _row(buf, r).upload(v[None])


def _get(buf, rows):
    a = np.concatenate([_row(buf, r).to_numpy() for r in rows])
    return _wide(a) if a.dtype == U16 else a.astype(np.float64)


def test_norm(gpu):
    from ancora_cutile_amd import DevBuf, NormWorkspace, rms_norm, rms_norm_grad
    T, H = 2100008, 1024
    marks = (0, 1, 2097150, 2097151, 2097152, 2097153, T - 2, T - 1)
    rng = np.random.default_rng(1)
    x, res, dy, gain = _bits(rng, (len(marks), H)), _bits(rng, (len(marks), H)), _bits(rng, (len(marks), H)), rng.standard_normal(H).astype(F32)

    def run(T, at):
        xb, rb, total, y, d = [DevBuf.zeros((T, H), U16) for _ in range(5)]
        r, dg, g, ws = DevBuf.zeros((T,), F32), DevBuf.zeros((H,), F32), DevBuf(gain), NormWorkspace(T, H)
        for b, v in ((xb, x), (rb, res), (d, dy)):
            _put(b, at, v)
        rms_norm(xb, g, 0, y=y, residual=rb, total=total, rstd=r)
        rms_norm_grad(d, total, g, r, 0, xb, dg, ws, carry=rb)
        out = [_get(b, at) for b in (y, total, xb)] + [dg.to_numpy().astype(np.float64)]
        quiet = [not _get(b, (5, 2000000, T - 5)).any() for b in (y, total, xb)] if T > 100 else [True]
        for b in (xb, rb, total, y, d, r, dg, g, ws):
            b.free()
        assert all(quiet)
        return out
    far, near = run(T, marks), run(len(marks), range(len(marks)))
    for a, b in zip(far[:3], near):
        assert bits_equal(a, b)                        # (a row's results do not depend on the others)
    s = _wide(x) + _wide(res)
    r = 1.0 / np.sqrt((s * s).mean(1) + 1e-6)
    mag = (np.abs(_wide(dy)) * np.abs(s) * r[:, None]).sum(0)
    assert np.all(np.abs(far[3] - near[3]) <= 2 * (len(marks) + 3) * 2.0 ** -24 * mag)


@pytest.mark.parametrize("counts", [None, (261900, 300)])
def test_feed_forward(gpu, counts):
    from ancora_cutile_amd import DevBuf, ffn_down, gated_ffn, gated_ffn_dx, gated_ffn_grad
    H, I, R = 64, 8200, 262200
    plan, E = None, 1
    if counts is not None:
        plan, c, o = _plan_of(counts, 1)
        assert plan.capacity >= R and list(o[:2]) == [0, counts[0]]
        E = 2
    rows = R if plan is None else plan.capacity
    line = (1 << 31) // I
    marks = np.array([0, 300, line - 1, line, line + 1, 261899, 261900, 262000, R - 1])
    of = (marks >= 261900).astype(int) if E == 2 else np.zeros(len(marks), int)
    rng = np.random.default_rng(2)
    W = {n: _bits(rng, (E, a, b), a ** -0.5) for n, a, b in (("Wg", H, I), ("Wu", H, I), ("Wd", I, H))}
    x, dy = _bits(rng, (len(marks), H)), _bits(rng, (len(marks), H))
    dev = {n: DevBuf(b) for n, b in W.items()}
    xb, dyb, y, dx = DevBuf.zeros((rows, H), U16), DevBuf.zeros((rows, H), U16), DevBuf.zeros((rows, H), F32), DevBuf.zeros((rows, H), F32)
    g, u, h = [DevBuf.zeros((rows, I), U16) for _ in range(3)]
    _put(xb, marks, x)
    _put(dyb, marks, dy)

    def product(a, w, flip=False):
        w = [m.T if flip else m for m in _wide(W[w])]
        return (np.stack([v @ w[e] for v, e in zip(a, of)]), (a.shape[1] + 8) * UNIT * np.stack([np.abs(v) @ np.abs(w[e]) for v, e in zip(a, of)]))

    def near(buf, want, err, half=2.0 ** -8):
        got = _get(buf, marks)
        assert np.all(np.abs(got - want) <= err + half * (np.abs(want) + err) + 1e-30)
        assert not _get(buf, (7, line - 2, line + 5, R - 3)).any()
        return got
    gated_ffn(xb, dev["Wg"], dev["Wu"], 0, h, gate=g, up=u, plan=plan)
    (gv, ge), (uv, ue) = product(_wide(x), "Wg"), product(_wide(x), "Wu")
    a = np.abs(gv) * ref.sigmoid(gv)
    hv = near(h, ref.gated(gv, uv), 1.1 * ge * (np.abs(uv) + ue) + a * ue + a * np.abs(uv) * (np.abs(gv) + 10) * UNIT)
    gv, uv = near(g, gv, ge), near(u, uv, ue)
    ffn_down(h, dev["Wd"], 0, y, plan=plan)
    near(y, *product(hv, "Wd"), half=2.0 ** -24)
    gated_ffn_grad(dyb, g, u, dev["Wd"], 0, g, u, plan=plan)
    dh, de = product(_wide(dy), "Wd", True)
    s = ref.sigmoid(gv)
    wg, wu, _ = ref.gated_grad(dh, gv, uv)
    es, slope = (np.abs(gv) + 10) * UNIT, s * (1 + np.abs(gv))
    dg = near(g, wg, (1.1 * de + 2 * np.abs(dh) * es) * np.abs(uv) * slope)
    du = near(u, wu, (1.1 * de + np.abs(dh) * es) * np.abs(gv) * s)
    gated_ffn_dx(g, u, dev["Wg"], dev["Wu"], 0, dx, plan=plan)
    (v1, e1), (v2, e2) = product(dg, "Wg", True), product(du, "Wu", True)
    near(dx, v1 + v2, 2 * (e1 + e2), half=2.0 ** -24)
    for b in (*dev.values(), xb, dyb, y, dx, g, u, h, *([plan] if plan else [])):
        b.free()
