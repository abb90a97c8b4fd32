"""The gated feed-forward block, dense and by expert, against the products in 64 bits.

Bounds. Products of bf16 are exact in fp32; K of them (and seven partial sums, where wavefronts share k) are added, each addition off by at most
one unit in the last place: (K + 8) 2^-23 of the sum of magnitudes. sigmoid(g) is off by (|g| + 8) 2^-23 of itself: the exponent's argument is rounded
(|g| 2^-24), exponential, sum and reciprocal are good to two units. An output rounds by 2^-8 (bf16) or 2^-24 (fp32) of the value."""
import ctypes

import numpy as np
import pytest

from oracle import layer_ref as ref
from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from test_gpu_expert_dw import _dirty, _plan_of
from util import bits_equal

pytestmark = pytest.mark.gpu
U16, F32 = np.uint16, np.float32
UNIT = 2.0 ** -23


def _bits(rng, shape, std=1.0):
    return bf16_rne_bits((std * rng.standard_normal(shape)).astype(F32)).reshape(shape)


def _wide(b):
    return np.nan_to_num(bits_to_f32(b).reshape(b.shape).astype(np.float64), posinf=0, neginf=0)


def _val(b):
    return b.to_numpy().astype(np.float64) if b.dtype == F32 else bits_to_f32(b.to_numpy()).reshape(b.shape).astype(np.float64)


def _half(b):
    return 2.0 ** -8 if b.dtype == U16 else 2.0 ** -24


def _near(buf, want, err, mine, what):
    got = _val(buf)
    assert np.isfinite(got[mine]).all(), what
    bad = (np.abs(got - want) - (err + _half(buf) * (np.abs(want) + err) + 1e-30))[mine]
    assert np.all(bad <= 0), (what, float(bad.max()))


class Case:
    """One block's weights and rows, on the device and in 64 bits. counts None: dense, `rows` rows."""

    def __init__(self, rng, H, I, rows=None, counts=None, align=1, spare=3):
        from ancora_cutile_amd import DevBuf
        self.H, self.I, self.plan, self.counts, self.offsets = H, I, None, None, None
        lead = ()
        if counts is not None:
            self.plan, self.counts, o = _plan_of(counts, align, spare)
            self.offsets, rows, lead = o[:-1], self.plan.capacity, (len(counts),)
        self.rows = rows
        self.mine = np.ones(rows, bool)
        if counts is not None:
            self.mine[:] = False
            for c, o in zip(self.counts, self.offsets):
                self.mine[o:o + c] = True
        self.host, self.dev = {}, {}
        for n, shape in (("Wg", (H, I)), ("Wu", (H, I)), ("Wd", (I, H))):
            b = _bits(rng, lead + shape, shape[0] ** -0.5)
            if counts is not None:                              # an expert without tokens may hold anything
                b[np.asarray(counts) == 0] = 0x7FFF
            self.put(n, b)
        for n, w in (("x", H), ("h", I), ("gate", I), ("up", I), ("dy", H), ("dgate", I), ("dup", I), ("res", H)):
            b = _bits(rng, (rows, w), 2.0 if n == "gate" else 1.0)
            self.put(n, b if counts is None else _dirty(b, self.counts, list(self.offsets) + [0]))
        self.put("res32", np.where(self.mine[:, None], rng.standard_normal((rows, H)), np.nan).astype(F32))
        self.new = lambda w, t=U16: DevBuf(np.full((rows, w), 0x7FC1 if t == U16 else np.nan, t))

    def put(self, name, a):
        from ancora_cutile_amd import DevBuf
        self.dev[name] = DevBuf(a)
        self.host[name] = _wide(a) if a.dtype == U16 else np.nan_to_num(a.astype(np.float64))

    def product(self, a, w, flip=False):
        """(a W, its error) per segment; flip: W transposed."""
        x, W = self.host[a], self.host[w]
        W = np.swapaxes(W, -1, -2) if flip else W
        K = W.shape[-2]
        return (ref.by_segment(x, W, self.counts, self.offsets),
                (K + 8) * UNIT * ref.by_segment(np.abs(x), np.abs(W), self.counts, self.offsets))

    def free(self):
        for b in self.dev.values():
            b.free()
        if self.plan is not None:
            self.plan.free()


def _untouched(buf, mine):
    a = buf.to_numpy()
    assert (np.isnan(a[~mine]).all() if buf.dtype == F32 else (a[~mine] == 0x7FC1).all())


def _check_all(c, si=0):
    """All four calls on one case; the bits of every result."""
    from ancora_cutile_amd import ffn_down, gated_ffn, gated_ffn_dx, gated_ffn_grad
    d, H, I, m, plan, out = c.dev, c.H, c.I, c.mine, c.plan, {}
    bufs = h, g, u, h2 = [c.new(I) for _ in range(4)]
    gated_ffn(d["x"], d["Wg"], d["Wu"], si, h, gate=g, up=u, plan=plan)
    gated_ffn(d["x"], d["Wg"], d["Wu"], si, h2, plan=plan)
    assert bits_equal(h.to_numpy(), h2.to_numpy())
    (gv, ge), (uv, ue) = c.product("x", "Wg"), c.product("x", "Wu")
    _near(g, gv, ge, m, "gate")
    _near(u, uv, ue, m, "up")
    a = np.abs(gv) * ref.sigmoid(gv)
    _near(h, ref.gated(gv, uv), 1.1 * ge * (np.abs(uv) + ue) + a * ue + a * np.abs(uv) * (np.abs(gv) + 10) * UNIT, m, "h")
    out.update(h=h.to_numpy(), gate=g.to_numpy(), up=u.to_numpy())

    v, e = c.product("h", "Wd")
    for t, res in ((U16, None), (U16, "res"), (F32, None), (F32, "res32")):
        y = c.new(H, t)
        bufs.append(y)
        ffn_down(d["h"], d["Wd"], si, y, residual=d[res] if res else None, plan=plan)
        want = v + (c.host[res] if res else 0.0)
        _near(y, want, e + (2.0 ** -24 * (np.abs(want) + e) if res else 0.0), m, ("down", t, res))
        out["y", t, res] = y.to_numpy()

    bufs += [c.new(I) for _ in range(3)]
    dg, du, h3 = bufs[-3:]
    gated_ffn_grad(d["dy"], d["gate"], d["up"], d["Wd"], si, dg, du, h=h3, plan=plan)
    dh, de = c.product("dy", "Wd", True)
    gv, uv = c.host["gate"], c.host["up"]
    s = ref.sigmoid(gv)
    wg, wu, wh = ref.gated_grad(dh, gv, uv)
    slope, es = np.abs(s * (1 + gv * (1 - s))), (np.abs(gv) + 10) * UNIT
    _near(dg, wg, de * np.abs(uv) * (slope + s * (1 + np.abs(gv)) * 2 * es) + np.abs(dh * uv) * (s * (1 + np.abs(gv)) * 2 * es), m, "dgate")
    _near(du, wu, de * np.abs(gv) * s * (1 + es) + np.abs(wu) * es, m, "dup")
    _near(h3, wh, np.abs(wh) * es, m, "h of the backward pass")
    out.update(dgate=dg.to_numpy(), dup=du.to_numpy(), h3=h3.to_numpy())

    (v1, e1), (v2, e2) = c.product("dgate", "Wg", True), c.product("dup", "Wu", True)
    v, e = v1 + v2, 2 * (e1 + e2)
    for t, res in ((U16, None), (U16, "res"), (F32, "res32")):
        dx = c.new(H, t)
        bufs.append(dx)
        gated_ffn_dx(d["dgate"], d["dup"], d["Wg"], d["Wu"], si, dx, residual=d[res] if res else None, plan=plan)
        want = v + (c.host[res] if res else 0.0)
        _near(dx, want, e + (2.0 ** -24 * (np.abs(want) + e) if res else 0.0), m, ("dx", t, res))
        out["dx", t, res] = dx.to_numpy()
    for b in bufs:
        _untouched(b, m)
        b.free()
    return out


SIZES = [(8, 8), (64, 264), (136, 1000), (640, 392), (264, 72), (40, 2056)]


@pytest.mark.parametrize("H,I", SIZES)
@pytest.mark.parametrize("rows", [1, 2, 16, 17, 33, 48, 49, 64, 130, 300])
def test_dense(gpu, H, I, rows):
    c = Case(np.random.default_rng(H + I + rows), H, I, rows=rows)
    _check_all(c)
    c.free()


@pytest.mark.parametrize("H,I", SIZES)
@pytest.mark.parametrize("counts,align", [((0, 1, 31, 32, 33), 1), ((64, 0, 100, 5, 0, 95, 96, 97), 16), ((3,), 128), ((400, 1, 257), 32), ((0, 0, 0, 200), 1)])
def test_by_expert(gpu, H, I, counts, align):
    c = Case(np.random.default_rng(H + I + len(counts)), H, I, counts=counts, align=align)
    _check_all(c)
    c.free()


@pytest.mark.parametrize("H,I", [(72, 8200), (8200, 72)])
def test_the_largest_tiles(gpu, H, I):
    c = Case(np.random.default_rng(1), H, I, rows=2049)
    _check_all(c)
    c.free()
    c = Case(np.random.default_rng(2), H, I, counts=(1000, 0, 1, 1047), align=16)
    _check_all(c)
    c.free()


@pytest.mark.parametrize("H,I,rows", [(520, 2816, 700), (520, 4104, 70), (4104, 264, 70), (72, 520, 4100), (520, 72, 4100), (2056, 520, 2050), (520, 2056, 2050), (2200, 2040, 8100),
                                      (2040, 2200, 8100), (4104, 2040, 200), (4088, 4088, 200), (136, 2816, 8100)])
def test_every_size_of_tile(gpu, H, I, rows):
    """Sizes at which each kernel that a call can take is the cheapest for one of the four calls (2200 and 2040: whole rounds of the largest tiles, with ragged
    edges): some rows, the first and the last among them, against 64 bits."""
    from ancora_cutile_amd import DevBuf, ffn_down, gated_ffn, gated_ffn_dx, gated_ffn_grad
    rng = np.random.default_rng(H + I + rows)
    pick = np.unique(np.concatenate([[0, 31, 32, 127, 128, 255, 256, rows - 1], rng.integers(0, rows, 60)]) % rows)
    host, dev = {}, {}
    for n, shape, std in (("Wg", (H, I), H ** -0.5), ("Wu", (H, I), H ** -0.5), ("Wd", (I, H), I ** -0.5), ("x", (rows, H), 1.0), ("h", (rows, I), 1.0),
                          ("gate", (rows, I), 1.0), ("up", (rows, I), 1.0), ("dy", (rows, H), 1.0)):
        b = bf16_rne_bits((std * rng.standard_normal(shape, dtype=F32))).reshape(shape)
        dev[n], host[n] = DevBuf(b), _wide(b if n[0] == "W" else b[pick])
    out = {n: DevBuf(np.full((rows, w), np.nan, t) if t == F32 else np.full((rows, w), 0x7FC1, t)) for n, w, t in
           (("h", I, U16), ("y", H, F32), ("dgate", I, U16), ("dup", I, U16), ("dx", H, U16))}

    def product(a, w):
        return a @ w, (a.shape[1] + 8) * UNIT * (np.abs(a) @ np.abs(w))

    def near(name, want, err):
        got = _val(out[name])
        assert np.isfinite(got).all(), name
        assert np.all(np.abs(got[pick] - want) <= err + _half(out[name]) * (np.abs(want) + err) + 1e-30), name
    gated_ffn(dev["x"], dev["Wg"], dev["Wu"], 0, out["h"])
    (g, ge), (u, ue) = product(host["x"], host["Wg"]), product(host["x"], host["Wu"])
    a = np.abs(g) * ref.sigmoid(g)
    near("h", ref.gated(g, u), 1.1 * ge * (np.abs(u) + ue) + a * ue + a * np.abs(u) * (np.abs(g) + 10) * UNIT)
    ffn_down(dev["h"], dev["Wd"], 0, out["y"])
    near("y", *product(host["h"], host["Wd"]))
    gated_ffn_grad(dev["dy"], dev["gate"], dev["up"], dev["Wd"], 0, out["dgate"], out["dup"])
    dh, de = product(host["dy"], host["Wd"].T)
    g, u = host["gate"], host["up"]
    s = ref.sigmoid(g)
    wg, wu, _ = ref.gated_grad(dh, g, u)
    es, slope = (np.abs(g) + 10) * UNIT, s * (1 + np.abs(g))
    near("dgate", wg, (1.1 * de + 2 * np.abs(dh) * es) * np.abs(u) * slope)
    near("dup", wu, (1.1 * de + np.abs(dh) * es) * np.abs(g) * s)
    gated_ffn_dx(dev["gate"], dev["up"], dev["Wg"], dev["Wu"], 0, out["dx"])
    (v1, e1), (v2, e2) = product(g, host["Wg"].T), product(u, host["Wu"].T)
    near("dx", v1 + v2, 2 * (e1 + e2))
    for b in (*dev.values(), *out.values()):
        b.free()


@pytest.mark.parametrize("E", [65, 130, 512])
def test_many_experts(gpu, E):
    rng = np.random.default_rng(E)
    counts = np.where(rng.random(E) < 0.5, 0, rng.integers(0, 5, E))
    counts[-1] = 2
    c = Case(rng, 40, 24, counts=tuple(counts))
    _check_all(c)
    c.free()
    if E == 65:
        c = Case(rng, 40, 24, counts=tuple(rng.integers(0, 140, E)), align=4)
        _check_all(c)
        c.free()


def test_bits_repeat_and_results_may_lie_on_their_inputs(gpu):
    from ancora_cutile_amd import DevBuf, ffn_down, gated_ffn_dx, gated_ffn_grad
    for c in (Case(np.random.default_rng(3), 136, 264, rows=20), Case(np.random.default_rng(4), 136, 264, counts=(200, 0, 90), align=8)):
        a, b = _check_all(c), _check_all(c)
        assert all(bits_equal(a[k], b[k]) for k in a)
        d, m = c.dev, c.mine
        ffn_down(d["h"], d["Wd"], 0, d["res32"], residual=d["res32"], plan=c.plan)
        assert bits_equal(d["res32"].to_numpy()[m], a["y", F32, "res32"][m])
        y = DevBuf(d["res"].to_numpy())
        gated_ffn_dx(d["dgate"], d["dup"], d["Wg"], d["Wu"], 0, y, residual=y, plan=c.plan)
        assert bits_equal(y.to_numpy()[m], a["dx", U16, "res"][m])
        gated_ffn_grad(d["dy"], d["gate"], d["up"], d["Wd"], 0, d["gate"], d["up"], plan=c.plan)
        assert bits_equal(d["gate"].to_numpy()[m], a["dgate"][m]) and bits_equal(d["up"].to_numpy()[m], a["dup"][m])
        y.free()
        c.free()


def test_what_is_not_finite_stays_in_its_row(gpu):
    from ancora_cutile_amd import ffn_down, gated_ffn
    for kw in (dict(rows=5), dict(rows=200), dict(counts=(3, 0, 2)), dict(counts=(150, 2, 100))):
        c = Case(np.random.default_rng(5), 72, 40, **kw)
        x, h = c.dev["x"].to_numpy(), c.dev["h"].to_numpy()
        row = int(np.flatnonzero(c.mine)[-1])                    # the last row of the last segment
        x[row, 71], h[row, 0] = 0x7F80, 0x7FFF
        c.dev["x"].upload(x)
        c.dev["h"].upload(h)
        ho, y = c.new(40), c.new(72)
        gated_ffn(c.dev["x"], c.dev["Wg"], c.dev["Wu"], 0, ho, plan=c.plan)
        ffn_down(c.dev["h"], c.dev["Wd"], 0, y, plan=c.plan)
        others = c.mine.copy()
        others[row] = False
        assert np.isfinite(_val(ho)[others]).all() and np.isfinite(_val(y)[others]).all()
        assert not np.isfinite(_val(ho)[row]).any() and np.isnan(_val(y)[row]).all()
        for b in (ho, y):
            b.free()
        c.free()


def test_large_pre_activations(gpu):
    """sigmoid at both ends: nothing becomes NaN, a gate far below zero gives zeros."""
    from ancora_cutile_amd import DevBuf, gated_ffn, gated_ffn_grad
    H = I = 8
    g = np.array([-1e4, -200, -90, -1, 0, 1, 90, 1e4], F32)
    x, Wg, Wu = np.ones((3, H), F32), np.diag(g) + 0 * np.ones((H, I), F32), np.eye(H, dtype=F32)
    to = lambda a: DevBuf(bf16_rne_bits(a.astype(F32)).reshape(a.shape))  # noqa: E731
    bufs = xd, gd, ud, h, gate, up = to(x), to(Wg), to(Wu), DevBuf.empty((3, I), U16), DevBuf.empty((3, I), U16), DevBuf.empty((3, I), U16)
    gated_ffn(xd, gd, ud, 0, h, gate=gate, up=up)
    gv = _val(gate)[0]
    want = gv * ref.sigmoid(gv)
    assert np.all(np.abs(_val(h) - want) <= np.abs(want) * (2.0 ** -8 + 200 * UNIT) + 1e-30)
    dg, du = DevBuf.empty((3, I), U16), DevBuf.empty((3, I), U16)
    gated_ffn_grad(xd, gate, up, ud, 0, dg, du)
    s = ref.sigmoid(gv)
    assert np.all(np.abs(_val(du) - want) <= np.abs(want) * (2.0 ** -8 + 200 * UNIT) + 1e-30)
    slope = s * (1 + gv * (1 - s))
    assert np.all(np.abs(_val(dg) - slope) <= np.abs(slope) * 2.0 ** -8 + s * (1 + np.abs(gv)) * (np.minimum(np.abs(gv), 200) + 10) * 2 * UNIT + 1e-30)
    for b in (*bufs, dg, du):
        b.free()


def test_gradient_against_differences(gpu):
    """sum(y w) with y = h Wd + residual in fp32 is linear in h: moving one value by 1/2 each way gives w Wd^T to the accuracy of fp32."""
    from ancora_cutile_amd import DevBuf, ffn_down, gated_ffn_grad
    rng = np.random.default_rng(6)
    T, I, H = 4, 16, 24
    h, Wd, w = _bits(rng, (T, I)), _bits(rng, (I, H)), _bits(rng, (T, H))
    one, zero = np.full((T, I), 0x3F80, U16), np.full((T, I), 0x42C8, U16)            # up = 1; gate = 100, where silu is the identity
    bufs = hd, Wdd, wd, up, gate, dg, du, y = (DevBuf(h), DevBuf(Wd), DevBuf(w), DevBuf(one), DevBuf(zero), DevBuf.empty((T, I), U16), DevBuf.empty((T, I), U16),
                                               DevBuf.empty((T, H), F32))
    gated_ffn_grad(wd, gate, up, Wdd, 0, dg, du)
    got, wv = _val(dg), bits_to_f32(w).reshape(T, H).astype(np.float64)
    for i in range(I):
        vals = []
        for to in (0x4000, 0x3F80):                                                  # 2 and 1
            b = h.copy()
            b[:, i] = to
            hd.upload(b)
            ffn_down(hd, Wdd, 0, y)
            vals.append(_val(y))
        diff = ((vals[0] - vals[1]) * wv).sum(1)
        mag = np.abs(_wide(Wd)).sum(0) * 4.0 * np.abs(_wide(h)).max()
        noise = 2 * (I + 8) * UNIT * (mag * np.abs(wv)).sum(1)
        assert np.all(np.abs(diff - got[:, i]) <= noise + 2.0 ** -8 * np.abs(got[:, i]) + 1e-5), i
    for b in bufs:
        b.free()


def test_captured_and_replayed_on_new_segments(gpu):
    from ancora_cutile_amd import DevBuf, RoutePlan, ffn_down, gated_ffn, gated_ffn_dx, gated_ffn_grad
    hip = ctypes.CDLL("libamdhip64.so")
    T, k, E, H, I = 300, 2, 6, 72, 136
    rng = np.random.default_rng(7)
    s = gpu.stream_create()
    W = [DevBuf(_bits(rng, (E, a, b), a ** -0.5)) for a, b in ((H, I), (H, I), (I, H))]
    sets = []
    for _ in range(2):
        p = RoutePlan(T, k, E, 4)
        S = p.capacity
        sets.append(dict(plan=p, **{n: DevBuf.zeros((S, w), U16) for n, w in (("h", I), ("g", I), ("u", I), ("y", H), ("dg", I), ("du", I), ("dx", H))}))
    x, e = DevBuf(_bits(rng, (S, H))), DevBuf(np.zeros((T, k), np.int32))

    def go(b, si):
        b["plan"].route(e, si)
        gated_ffn(x, W[0], W[1], si, b["h"], gate=b["g"], up=b["u"], plan=b["plan"])
        ffn_down(b["h"], W[2], si, b["y"], plan=b["plan"])
        gated_ffn_grad(b["y"], b["g"], b["u"], W[2], si, b["dg"], b["du"], plan=b["plan"])
        gated_ffn_dx(b["dg"], b["du"], W[0], W[1], si, b["dx"], plan=b["plan"])
    graph, graph_exec = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(ctypes.c_void_p(s), 0) == 0
    go(sets[0], s)
    assert hip.hipStreamEndCapture(ctypes.c_void_p(s), ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, ctypes.c_size_t(0)) == 0
    for r in range(4):
        e.upload(np.minimum((E * rng.random((T, k)) ** (r + 1)).astype(np.int32), E - 1) - (r == 3))
        go(sets[1], 0)
        gpu.stream_sync(0)
        assert hip.hipGraphLaunch(graph_exec, ctypes.c_void_p(s)) == 0
        gpu.stream_sync(s)
        for n in ("h", "g", "u", "y", "dg", "du", "dx"):
            assert bits_equal(sets[0][n].to_numpy(), sets[1][n].to_numpy()), (r, n)
    hip.hipGraphExecDestroy(graph_exec)
    hip.hipGraphDestroy(graph)
    for b in (x, e, *W, *(v for q in sets for v in q.values())):
        b.free()
    gpu.api.anc_stream_destroy(s)


def test_no_tokens_at_all(gpu):
    from ancora_cutile_amd import DevBuf, RoutePlan, ffn_down, gated_ffn
    plan, ids = RoutePlan(20, 2, 3, 16), DevBuf(np.zeros((20, 2), np.int32))
    plan.route(ids, 0, 0)
    S = plan.capacity
    bufs = x, W, Wd, h, y = (DevBuf(np.full((S, 16), 0x7FFF, U16)), DevBuf(np.full((3, 16, 24), 0x7FFF, U16)), DevBuf(np.full((3, 24, 16), 0x7FFF, U16)),
                             DevBuf(np.full((S, 24), 7, U16)), DevBuf(np.full((S, 16), 7, U16)))
    gated_ffn(x, W, W, 0, h, plan=plan)
    ffn_down(h, Wd, 0, y, plan=plan)
    assert (h.to_numpy() == 7).all() and (y.to_numpy() == 7).all()
    for b in (*bufs, plan, ids):
        b.free()


@pytest.mark.parametrize("H,I,E,tokens", [(72, 2056, 2, 3000), (2056, 40, 2, 3000), (264, 264, 6, 16000), (520, 520, 2, 16000), (2056, 520, 2, 700),
                                          (520, 4104, 2, 1500), (1544, 1032, 2, 5000)])
def test_every_size_of_tile_over_segments(gpu, H, I, E, tokens):
    """Uneven segments at sizes where each of the kernels is the cheapest for one of the four calls: rows at the tiles' edges and some others of every segment
    against 64 bits, nothing else written."""
    from ancora_cutile_amd import DevBuf, ffn_down, gated_ffn, gated_ffn_dx, gated_ffn_grad
    rng = np.random.default_rng(H + I + tokens)
    counts = rng.multinomial(tokens, np.linspace(0.6, 1.4, E) / E)
    plan, counts, offsets = _plan_of(counts, 8, 5)
    rows, mine = plan.capacity, np.zeros(plan.capacity, bool)
    pick, of = [], []
    for e, (n, o) in enumerate(zip(counts, offsets)):
        mine[o:o + n] = True
        p = np.unique(np.concatenate([[0, 31, 63, 64, 127, 128, 255, 256, n - 1], rng.integers(0, n, 25)]) % n)
        pick.append(o + p)
        of.append(np.full(p.size, e))
    pick, of = np.concatenate(pick), np.concatenate(of)
    host, dev = {}, {}
    for n, shape, std in (("Wg", (E, H, I), H ** -0.5), ("Wu", (E, H, I), H ** -0.5), ("Wd", (E, I, H), I ** -0.5), ("x", (rows, H), 1.0), ("h", (rows, I), 1.0),
                          ("gate", (rows, I), 1.0), ("up", (rows, I), 1.0), ("dy", (rows, H), 1.0), ("res", (rows, H), 1.0)):
        b = bf16_rne_bits((std * rng.standard_normal(shape, dtype=F32))).reshape(shape)
        if n[0] != "W":
            b[~mine] = 0x7FFF
        dev[n], host[n] = DevBuf(b), _wide(b if n[0] == "W" else b[pick])
    out = {n: DevBuf(np.full((rows, w), np.nan, t) if t == F32 else np.full((rows, w), 0x7FC1, t)) for n, w, t in
           (("h", I, U16), ("g", I, U16), ("u", I, U16), ("y", H, F32), ("dgate", I, U16), ("dup", I, U16), ("h2", I, U16), ("dx", H, U16))}

    def product(a, w):
        v, m = np.empty((a.shape[0], w.shape[2])), np.empty((a.shape[0], w.shape[2]))
        for e in range(E):
            v[of == e], m[of == e] = a[of == e] @ w[e], np.abs(a[of == e]) @ np.abs(w[e])
        return v, (a.shape[1] + 8) * UNIT * m

    def near(name, want, err):
        got = _val(out[name])
        assert np.isfinite(got[mine]).all(), name
        assert np.all(np.abs(got[pick] - want) <= err + _half(out[name]) * (np.abs(want) + err) + 1e-30), name
        _untouched(out[name], mine)
    gated_ffn(dev["x"], dev["Wg"], dev["Wu"], 0, out["h"], gate=out["g"], up=out["u"], plan=plan)
    (g, ge), (u, ue) = product(host["x"], host["Wg"]), product(host["x"], host["Wu"])
    a = np.abs(g) * ref.sigmoid(g)
    near("h", ref.gated(g, u), 1.1 * ge * (np.abs(u) + ue) + a * ue + a * np.abs(u) * (np.abs(g) + 10) * UNIT)
    near("g", g, ge)
    near("u", u, ue)
    ffn_down(dev["h"], dev["Wd"], 0, out["y"], plan=plan)
    near("y", *product(host["h"], host["Wd"]))
    gated_ffn_grad(dev["dy"], dev["gate"], dev["up"], dev["Wd"], 0, out["dgate"], out["dup"], h=out["h2"], plan=plan)
    flip = lambda w: np.swapaxes(w, 1, 2)  # noqa: E731
    dh, de = product(host["dy"], flip(host["Wd"]))
    g, u = host["gate"], host["up"]
    s = ref.sigmoid(g)
    wg, wu, wh = ref.gated_grad(dh, g, u)
    es, slope = (np.abs(g) + 10) * UNIT, s * (1 + np.abs(g))
    near("dgate", wg, (1.1 * de + 2 * np.abs(dh) * es) * np.abs(u) * slope)
    near("dup", wu, (1.1 * de + np.abs(dh) * es) * np.abs(g) * s)
    near("h2", wh, np.abs(wh) * es)
    gated_ffn_dx(dev["gate"], dev["up"], dev["Wg"], dev["Wu"], 0, out["dx"], residual=dev["res"], plan=plan)
    (v1, e1), (v2, e2) = product(g, flip(host["Wg"])), product(u, flip(host["Wu"]))
    want = v1 + v2 + host["res"]
    near("dx", want, 2 * (e1 + e2) + 2.0 ** -24 * (np.abs(want) + 2 * (e1 + e2)))
    for b in (*dev.values(), *out.values(), plan):
        b.free()
