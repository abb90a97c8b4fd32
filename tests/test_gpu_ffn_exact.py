"""The feed-forward block on small whole numbers, whose sums fp32 holds exactly in any order: every product's outputs are the whole sum's rounding and nothing
else, so that one k dropped, doubled or taken from another row shows, however long k is.

Operands within 3, up within 4, residuals within 100: sums of up to 8200 products stay below 2^18, what the epilogues multiply onto them below 2^24. The
backward epilogue is exact where the gate is 0 (sigmoid 1/2, its slope 1/2, silu 0) or 32 (1 + e^-32 is 1 in fp32: sigmoid 1, slope 1, silu 32). The sizes
are such that every kernel that the call's rule can choose is taken by each of the four calls, dense and by expert, where the rule takes it at all, with all
optional results and both types of residual; K ends inside a step of 32 or 64 and in a whole one, N inside a tile."""
import numpy as np
import pytest

from oracle import layer_ref as ref
from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from test_gpu_expert_dw import _plan_of

pytestmark = pytest.mark.gpu
U16, F32 = np.uint16, np.float32


def _bits(a):
    return bf16_rne_bits(np.ascontiguousarray(a, F32)).reshape(a.shape)


def _rounded(a):
    return bits_to_f32(_bits(a)).reshape(a.shape)


def _same(buf, want, mine, what):
    a = buf.to_numpy()
    got = a if a.dtype == F32 else bits_to_f32(a).reshape(a.shape)
    assert np.array_equal(got[mine], (want if a.dtype == F32 else _rounded(want))[mine]), what
    assert np.isnan(got[~mine]).all(), what


@pytest.mark.parametrize("rows,E,H,I", [
    (1, 0, 72, 72), (1, 2, 72, 72), (1653, 0, 72, 72), (1, 2, 328, 328), (165, 2, 392, 392), (2891, 0, 328, 72), (2483, 0, 136, 72), (8363, 0, 200, 72),
    (4230, 0, 72, 1544), (3461, 9, 72, 1544), (1688, 5, 1032, 72), (3743, 0, 2056, 72), (2314, 9, 2568, 136), (4253, 2, 8200, 72), (6336, 0, 1288, 72),
    (763, 3, 648, 8200), (5869, 0, 2056, 1032), (5811, 2, 2200, 2056), (5514, 0, 520, 2200), (5, 0, 8200, 72), (40, 0, 4104, 8200), (300, 0, 8200, 1024),
    (2000, 0, 128, 8192)])
def test_whole_numbers(gpu, rows, E, H, I):
    from ancora_cutile_amd import DevBuf, ffn_down, gated_ffn, gated_ffn_dx, gated_ffn_grad
    rng = np.random.default_rng(rows + H + I)
    whole = lambda shape, most: rng.integers(-most, most + 1, shape, np.int8).astype(F32)  # noqa: E731
    plan = counts = offsets = None
    lead, mine = (), np.ones(rows, bool)
    if E:
        counts = rng.multinomial(rows, np.linspace(0.5, 1.5, E) / E)
        plan, counts, offsets = _plan_of(counts, 8, 3)
        lead, mine = (E,), np.zeros(plan.capacity, bool)
        for c, o in zip(counts, offsets):
            mine[o:o + c] = True
    S = mine.size
    host = {n: whole(lead + s, 3) for n, s in dict(Wg=(H, I), Wu=(H, I), Wd=(I, H)).items()}
    host.update(x=whole((S, H), 3), h=whole((S, I), 3), dy=whole((S, H), 3), dg=whole((S, I), 3), du=whole((S, I), 3), res=whole((S, H), 100),
                gate=np.where(rng.random((S, I)) < 0.5, 0, 32).astype(F32), up=np.exp2(rng.integers(0, 3, (S, I))).astype(F32) * np.where(rng.random((S, I)) < 0.5, 1, -1))
    dev = {}
    for n, a in host.items():
        b = _bits(a)
        if n[0] != "W":
            b[~mine] = 0x7FFF                             # what is nobody's may hold anything
        dev[n] = DevBuf(b)
    dev["res32"] = DevBuf(np.where(mine[:, None], host["res"], F32(np.nan)))
    new = lambda w, t=U16: DevBuf(np.full((S, w), 0x7FC1 if t == U16 else np.nan, t))  # noqa: E731

    def product(a, w, flip=False):
        x, W = host[a], np.swapaxes(host[w], -1, -2) if flip else host[w]
        if not E:
            return x @ W
        out = np.zeros((S, W.shape[2]), F32)
        for e, (c, o) in enumerate(zip(counts, offsets)):
            out[o:o + c] = x[o:o + c] @ W[e]
        return out
    outs = h, g, u = new(I), new(I), new(I)
    gated_ffn(dev["x"], dev["Wg"], dev["Wu"], 0, h, gate=g, up=u, plan=plan)
    gv, uv = product("x", "Wg"), product("x", "Wu")
    _same(g, gv, mine, "gate")
    _same(u, uv, mine, "up")
    got, want = bits_to_f32(h.to_numpy()).reshape(S, I)[mine], ref.gated(gv.astype(np.float64), uv)[mine]
    e = np.abs(want) * (np.abs(gv[mine]) + 10) * 2.0 ** -23     # (sigmoid's: the exponent's rounding, and two units of exponential, sum and reciprocal each)
    assert np.all(np.abs(got - want) <= e + 2.0 ** -8 * (np.abs(want) + e) + 1e-30), "h"
    for b in outs:
        b.free()
    v = product("h", "Wd")
    for t, res in ((U16, None), (U16, "res"), (F32, None), (F32, "res32")):
        y = new(H, t)
        ffn_down(dev["h"], dev["Wd"], 0, y, residual=dev[res] if res else None, plan=plan)
        _same(y, v + host["res"] if res else v, mine, ("down", t, res))
        y.free()
    outs = dg, du, h = new(I), new(I), new(I)
    gated_ffn_grad(dev["dy"], dev["gate"], dev["up"], dev["Wd"], 0, dg, du, h=h, plan=plan)
    dh, big = product("dy", "Wd", True), host["gate"] > 0
    _same(dg, dh * host["up"] * np.where(big, F32(1), F32(0.5)), mine, "dgate")
    _same(du, dh * host["gate"], mine, "dup")
    _same(h, host["gate"] * host["up"], mine, "h of the backward pass")
    for b in outs:
        b.free()
    v = product("dg", "Wg", True) + product("du", "Wu", True)
    for t, res in ((U16, None), (U16, "res"), (F32, None), (F32, "res32")):
        dx = new(H, t)
        gated_ffn_dx(dev["dg"], dev["du"], dev["Wg"], dev["Wu"], 0, dx, residual=dev[res] if res else None, plan=plan)
        _same(dx, v + host["res"] if res else v, mine, ("dx", t, res))
        dx.free()
    for b in (*dev.values(), *([plan] if E else [])):
        b.free()
