"""The norm with the residual's addition and its backward pass against 64 bits.

Bounds. fp32 sums of n values are off by at most n 2^-24 of the sum of magnitudes. r = 1 / sqrt(mean s^2 + eps): the squares are
positive, so the sum is off by (H + 2) 2^-24 of itself, the root by half of that, and division, root and reciprocal round once each; a
result takes two products more. Outputs round by 2^-8 (bf16) or 2^-24 (fp32) of the value; s itself is one addition, 2^-24."""
import ctypes

import numpy as np
import pytest

from oracle import layer_ref as ref
from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from util import bits_equal

pytestmark = pytest.mark.gpu
U16, F32 = np.uint16, np.float32
WIDTHS = [8, 64, 120, 128, 136, 256, 264, 512, 520, 1024, 2048, 2056, 4096, 5000, 8192, 16384]
EPS = 1e-6


def _make(rng, shape, dtype, std=1.0):
    """(what the device holds, its value in 64 bits)"""
    x = (std * rng.standard_normal(shape)).astype(F32)
    if dtype == F32:
        return x, x.astype(np.float64)
    b = bf16_rne_bits(x).reshape(shape)
    return b, bits_to_f32(b).reshape(shape).astype(np.float64)


def _val(b):
    return b.to_numpy().astype(np.float64) if b.dtype == F32 else bits_to_f32(b.to_numpy()).reshape(b.shape).astype(np.float64)


def _half(dtype):
    return 2.0 ** -8 if dtype == U16 else 2.0 ** -24


def _r_bound(H):
    return (H + 2) * 2.0 ** -25 + 4 * 2.0 ** -24


@pytest.mark.parametrize("H", WIDTHS)
@pytest.mark.parametrize("x,stream,gain,out", [(U16, U16, F32, U16), (U16, F32, U16, F32), (F32, F32, F32, F32), (F32, U16, U16, U16), (U16, None, F32, U16)])
def test_forward(gpu, H, x, stream, gain, out):
    from ancora_cutile_amd import DevBuf, rms_norm
    rng = np.random.default_rng(H)
    for T in (1, 2, 5, 33):
        xb, xv = _make(rng, (T, H), x, np.exp2(rng.integers(-6, 6, (T, 1))))
        gb, gv = _make(rng, (H,), gain)
        kw, s = {}, xv
        if stream is not None:
            rb, rv = _make(rng, (T, H), stream, 2.0)
            kw, s = dict(residual=DevBuf(rb), total=DevBuf.empty((T, H), stream)), xv + rv
        xd, gd, y, r = DevBuf(xb), DevBuf(gb), DevBuf.empty((T, H), out), DevBuf.empty((T,), F32)
        rms_norm(xd, gd, 0, y=y, rstd=r, eps=EPS, **kw)
        want, wr = ref.rms_norm(s, gv, EPS)
        e = _r_bound(H) + 2.0 ** -24                              # (s is rounded once)
        assert np.all(np.abs(_val(r) - wr) <= e * wr)
        e += 3 * 2.0 ** -24
        assert np.all(np.abs(_val(y) - want) <= np.abs(want) * (e + _half(out) * (1 + e))), T
        if stream is not None:
            got = _val(kw["total"])
            assert np.all(np.abs(got - s) <= np.abs(s) * (2.0 ** -24 + _half(stream) * 1.0001))
            first = y.to_numpy()
            rms_norm(xd, gd, 0, y=y, eps=EPS, residual=kw["residual"], total=kw["residual"])      # in place, without r: the same bits
            assert bits_equal(y.to_numpy(), first) and np.array_equal(_val(kw["residual"]), got)
        for b in (xd, gd, y, r, *kw.values()):
            b.free()


@pytest.mark.parametrize("H", [32, 96, 128, 256, 288, 1024, 2080, 4096, 16384])
def test_8_bit_rows(gpu, H):
    """Codes and scales are those of the fp32 rows that the same call gives, bit for bit, whatever the rows' magnitude."""
    from ancora_cutile_amd import DevBuf, rms_norm
    rng = np.random.default_rng(H)
    T = 37
    x, g = (rng.standard_normal((T, H)) * np.exp2(rng.integers(-12, 1, (T, H)))).astype(F32), rng.standard_normal(H).astype(F32)
    g[rng.random(H) < 0.1] = 0.0
    g[:32] *= 1e-37                                            # blocks whose scale byte is at its least
    x[5] = 0.0
    x[7, H // 2] = np.inf
    x[9, 3] = np.nan
    res, _ = _make(rng, (T, H), U16)
    res[5] = 0
    bufs = xd, gd, rd, td, y, q, s = (DevBuf(x), DevBuf(g), DevBuf(res), DevBuf.empty((T, H), U16), DevBuf.empty((T, H), F32), DevBuf.empty((T, H), np.uint8),
                                      DevBuf.empty((T, H // 32), np.uint8))
    rms_norm(xd, gd, 0, y=y, residual=rd, total=td)
    rms_norm(xd, gd, 0, fp8=q, scale=s, residual=rd, total=td)
    yv = y.to_numpy()
    assert np.isnan(yv[7, H // 2]) and np.isnan(yv[9]).all() and np.isfinite(np.delete(yv, [7, 9], 0)).all()
    codes, scale = ref.mx8_rows(yv)
    assert bits_equal(s.to_numpy(), scale)
    got, nan = q.to_numpy(), np.isnan(yv)
    assert bits_equal(got[~nan], codes[~nan]) and np.all(got[nan] & 0x7F == 0x7F)
    for b in bufs:
        b.free()


@pytest.mark.parametrize("H", WIDTHS)
@pytest.mark.parametrize("dy,stream,gain,carry", [(U16, U16, F32, True), (U16, F32, U16, False), (F32, F32, F32, True), (F32, U16, F32, False)])
def test_backward(gpu, H, dy, stream, gain, carry):
    """dx = r (a - xh c) + carry with a = dy gain, xh = x r, c = mean(a xh): c is a sum of H, off by (H + 4) 2^-24 of the mean of magnitudes; a, xh
    and the remaining operations round once each. dgain is a sum over T of products rounded twice."""
    from ancora_cutile_amd import DevBuf, NormWorkspace, rms_norm_grad
    rng = np.random.default_rng(H + 1)
    for T in (1, 7, 50, 1100 if H <= 264 else 131):
        db, dv = _make(rng, (T, H), dy, 0.1)
        sb, sv = _make(rng, (T, H), stream, np.exp2(rng.integers(-3, 3, (T, 1))))
        gb, gv = _make(rng, (H,), gain)
        cb, cv = _make(rng, (T, H), stream, 0.1)
        _, wr = ref.rms_norm(sv, gv, EPS)
        r32 = wr.astype(F32)
        bufs = d, s, g, c, r, dx, dg, base = (DevBuf(db), DevBuf(sb), DevBuf(gb), DevBuf(cb), DevBuf(r32), DevBuf.empty((T, H), stream), DevBuf.empty((H,), F32),
                                              DevBuf(np.arange(H, dtype=F32)))
        ws = NormWorkspace(T, H)
        rms_norm_grad(d, s, g, r, 0, dx, dg, ws, carry=c if carry else None)
        want, wdg = ref.rms_norm_grad(dv, sv, gv, r32)
        a, xh, u = np.abs(dv * gv), np.abs(sv * r32[:, None].astype(np.float64)), 2.0 ** -24
        mean = (a * xh).mean(1, keepdims=True)
        err = r32[:, None] * (4 * u * a + xh * mean * (H + 10) * u)
        if carry:
            want = want + cv
            err = err + u * (np.abs(want) + err)
        assert np.all(np.abs(_val(dx) - want) <= err + _half(stream) * (np.abs(want) + err) + 1e-38), T
        mag = (np.abs(dv) * xh).sum(0)
        assert np.all(np.abs(_val(dg) - wdg) <= (T + 3) * u * mag), T
        got = dg.to_numpy()
        rms_norm_grad(d, s, g, r, 0, dx, base, ws, carry=c if carry else None, accumulate=True)
        assert np.all(np.abs(base.to_numpy() - (np.arange(H) + got.astype(np.float64))) <= u * (np.arange(H) + np.abs(got)) * 1.0001)
        if dy == stream:                                         # over dy itself, and once more: the same bits
            first = dx.to_numpy()
            rms_norm_grad(d, s, g, r, 0, d, dg, ws, carry=c if carry else None)
            assert bits_equal(d.to_numpy(), first) and bits_equal(dg.to_numpy(), got)
        for b in (*bufs, ws):
            b.free()


@pytest.mark.parametrize("H", [64, 1024, 4096])
def test_one_workspace_for_batches_of_any_length(gpu, H):
    """Around the lengths where the number of partial sums changes, all with the workspace of the longest: a row of ones times ones counts the rows."""
    from ancora_cutile_amd import DevBuf, NormWorkspace, rms_norm_grad
    most = 8200 if H <= 1024 else 2060
    one = np.full((most, H), 0x3F80, U16)
    bufs = dy, x, g, r, dx, dg = DevBuf(one), DevBuf(one), DevBuf(np.ones(H, F32)), DevBuf(np.ones(most, F32)), DevBuf(one), DevBuf(np.zeros(H, F32))
    ws = NormWorkspace(most, H)
    for T in (most, most - 7, most - 8, most - 9, most // 2 + 1, most // 2, 1025, 1024, 1023, 17, 1):
        rms_norm_grad(dy.view((T, H)), x, g, r, 0, dx, dg, ws)
        assert (dg.to_numpy() == T).all(), T
    for b in (*bufs, ws):
        b.free()


def test_gradient_against_differences(gpu):
    """loss = sum(y w) in fp32. The device's central difference is within its own rounding (the bound of y, twice, over the step) of the formula's difference
    in 64 bits, and that is the gradient to the third order of the step, which is computed from two steps."""
    from ancora_cutile_amd import DevBuf, NormWorkspace, rms_norm, rms_norm_grad
    rng = np.random.default_rng(9)
    T, H, h = 3, 16, 2.0 ** -7
    x, g, w = (rng.standard_normal(s).astype(F32) for s in ((T, H), (H,), (T, H)))
    bufs = xd, gd, wd, y, r, dx, dg = (DevBuf(x), DevBuf(g), DevBuf(w), DevBuf.empty((T, H), F32), DevBuf.empty((T,), F32), DevBuf.empty((T, H), F32),
                                       DevBuf.empty((H,), F32))
    ws = NormWorkspace(T, H)
    rms_norm(xd, gd, 0, y=y, rstd=r)
    rms_norm_grad(wd, xd, gd, r, 0, dx, dg, ws)
    got = dx.to_numpy()

    def exact(v):
        return float((ref.rms_norm(v, g, EPS)[0] * w).sum())
    for i in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i] += F32(h)
        down[i] -= F32(h)
        vals = []
        for v in (up, down):
            xd.upload(v)
            rms_norm(xd, gd, 0, y=y)
            vals.append((y.to_numpy().astype(np.float64) * w).sum())
        step = float(up[i]) - float(down[i])
        diff, formula = (vals[0] - vals[1]) / step, (exact(up) - exact(down)) / step
        noise = 2 * (_r_bound(H) + 4 * 2.0 ** -24) * np.abs(ref.rms_norm(x, g, EPS)[0] * w).sum() * 1.1 / step
        assert abs(diff - formula) <= noise
        wide = [x.astype(np.float64), x.astype(np.float64)]
        wide[0][i] += 2 * h
        wide[1][i] -= 2 * h
        third = abs((exact(wide[0]) - exact(wide[1])) / (4 * h) - formula)          # three times the step's own error, and higher orders
        assert abs(formula - got[i]) <= third + 1e-5 * np.abs(got).max()
    for b in (*bufs, ws):
        b.free()


def test_captured_and_replayed(gpu):
    """Forward and backward in one graph on a stream of its own, replayed on new inputs between eager calls with a workspace of their own."""
    from ancora_cutile_amd import DevBuf, NormWorkspace, rms_norm, rms_norm_grad
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng(10)
    T, H = 700, 264
    s = gpu.stream_create()
    x, g, dy = DevBuf.zeros((T, H), U16), DevBuf(rng.standard_normal(H).astype(F32)), DevBuf.zeros((T, H), U16)
    sets = [dict(y=DevBuf.zeros((T, H), U16), r=DevBuf.zeros((T,), F32), dx=DevBuf.zeros((T, H), U16), dg=DevBuf.zeros((H,), F32), ws=NormWorkspace(T, H)) for _ in range(2)]

    def go(b, si):
        rms_norm(x, g, si, y=b["y"], rstd=b["r"])
        rms_norm_grad(dy, x, g, b["r"], si, b["dx"], b["dg"], b["ws"])
    graph, graph_exec = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(ctypes.c_void_p(s), 0) == 0
    go(sets[0], s)
    assert hip.hipStreamEndCapture(ctypes.c_void_p(s), ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(3):
        x.upload(_make(rng, (T, H), U16)[0])
        dy.upload(_make(rng, (T, H), U16)[0])
        go(sets[1], 0)
        gpu.stream_sync(0)
        assert hip.hipGraphLaunch(graph_exec, ctypes.c_void_p(s)) == 0
        gpu.stream_sync(s)
        for k in ("y", "r", "dx", "dg"):
            assert bits_equal(sets[0][k].to_numpy(), sets[1][k].to_numpy()), k
    hip.hipGraphExecDestroy(graph_exec)
    hip.hipGraphDestroy(graph)
    for b in (x, g, dy, *(v for q in sets for v in q.values())):
        b.free()
    gpu.api.anc_stream_destroy(s)


@pytest.mark.parametrize("T,H", [(4500, 200), (9000, 520), (4200, 1000), (2100, 1544), (2300, 4096), (1300, 5000), (1100, 16384)])
def test_backward_of_many_rows(gpu, T, H):
    """Three rows and more to every group of lanes, at each number of lanes: the bounds of `test_backward`."""
    from ancora_cutile_amd import DevBuf, NormWorkspace, rms_norm_grad
    rng = np.random.default_rng(T)
    (db, dv), (sb, sv), (gb, gv), (cb, cv) = _make(rng, (T, H), U16, 0.1), _make(rng, (T, H), U16), _make(rng, (H,), F32), _make(rng, (T, H), U16, 0.1)
    r32 = ref.rms_norm(sv, gv, EPS)[1].astype(F32)
    bufs = d, s, g, c, r, dx, dg = (DevBuf(db), DevBuf(sb), DevBuf(gb), DevBuf(cb), DevBuf(r32), DevBuf.empty((T, H), U16), DevBuf.empty((H,), F32))
    ws, u = NormWorkspace(T, H), 2.0 ** -24
    rms_norm_grad(d, s, g, r, 0, dx, dg, ws, carry=c)
    first = dx.to_numpy(), dg.to_numpy()
    want, wdg = ref.rms_norm_grad(dv, sv, gv, r32)
    a, xh = np.abs(dv * gv), np.abs(sv * r32[:, None].astype(np.float64))
    err = r32[:, None] * (4 * u * a + xh * (a * xh).mean(1, keepdims=True) * (H + 10) * u)
    want = want + cv
    err = err + u * (np.abs(want) + err)
    assert np.all(np.abs(_val(dx) - want) <= err + _half(U16) * (np.abs(want) + err) + 1e-38)
    assert np.all(np.abs(_val(dg) - wdg) <= (T + 3) * u * (np.abs(dv) * xh).sum(0))
    rms_norm_grad(d, s, g, r, 0, dx, dg, ws, carry=c)
    assert bits_equal(dx.to_numpy(), first[0]) and bits_equal(dg.to_numpy(), first[1])
    for b in (*bufs, ws):
        b.free()
