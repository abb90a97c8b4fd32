"""Every result that may lie on an input does: the bits of the call with buffers of their own, at sizes that take each kernel of the rule."""
import numpy as np
import pytest

from oracle.bf16_ref import bf16_rne_bits
from util import bits_equal

pytestmark = pytest.mark.gpu
U16, F32 = np.uint16, np.float32


def _bits(rng, shape, std=1.0):
    return bf16_rne_bits((std * rng.standard_normal(shape, dtype=F32))).reshape(shape)


@pytest.mark.parametrize("T,H", [(5, 136), (33, 1000), (300, 2056), (70, 8200)])
@pytest.mark.parametrize("t", [U16, F32])
def test_norm(gpu, T, H, t):
    from ancora_cutile_amd import DevBuf, NormWorkspace, rms_norm, rms_norm_grad
    rng = np.random.default_rng(H)
    make = lambda: _bits(rng, (T, H)) if t == U16 else rng.standard_normal((T, H), dtype=F32)  # noqa: E731
    x, res, dy = make(), make(), make()
    g, r, dg, ws = DevBuf(rng.standard_normal(H).astype(F32)), DevBuf(np.zeros(T, F32)), DevBuf(np.zeros(H, F32)), NormWorkspace(T, H)
    a, b, y, total = DevBuf(x), DevBuf(res), DevBuf(np.zeros_like(x)), DevBuf(np.zeros_like(x))
    rms_norm(a, g, 0, y=y, residual=b, total=total, rstd=r)
    wy, wt, wr = y.to_numpy(), total.to_numpy(), r.to_numpy()
    for on_y, on_total in ((a, b), (b, a), (a, total), (y, a), (b, total), (y, b)):
        a.upload(x)
        b.upload(res)
        rms_norm(a, g, 0, y=on_y, residual=b, total=on_total, rstd=r)
        assert bits_equal(on_y.to_numpy(), wy) and bits_equal(on_total.to_numpy(), wt) and bits_equal(r.to_numpy(), wr)
    a.upload(x)
    rms_norm(a, g, 0, y=y)
    rms_norm(a, g, 0, y=a)
    assert bits_equal(a.to_numpy(), y.to_numpy())
    d, s, c, dx = DevBuf(dy), DevBuf(x), DevBuf(res), DevBuf(np.zeros_like(x))
    rms_norm_grad(d, s, g, r, 0, dx, dg, ws, carry=c)
    wdx, wdg = dx.to_numpy(), dg.to_numpy()
    for on in (d, s, c):
        for buf, v in ((d, dy), (s, x), (c, res)):
            buf.upload(v)
        rms_norm_grad(d, s, g, r, 0, on, dg, ws, carry=c)
        assert bits_equal(on.to_numpy(), wdx) and bits_equal(dg.to_numpy(), wdg)
    for buf, v in ((s, x), (d, dy)):
        buf.upload(v)
    rms_norm_grad(d, s, g, r, 0, dx, dg, ws, carry=d)             # the same buffer for two inputs, and then for the result too
    want = dx.to_numpy()
    rms_norm_grad(d, s, g, r, 0, d, dg, ws, carry=d)
    assert bits_equal(d.to_numpy(), want)
    for o in (g, r, dg, ws, a, b, y, total, d, s, c, dx):
        o.free()


# which of the eight kernels take (down, dx, grad): (6, 6, 6), (1, 0, 4), (2, 2, 5), (3, 3, 0), (0, 0, 1), (5, 5, 6), (7, 7, 7), (4, 4, 2), (1, 1, 3)
@pytest.mark.parametrize("rows,H,I", [(1653, 72, 72), (6336, 1288, 72), (3743, 2056, 72), (5514, 520, 2200), (5869, 2056, 1032), (2483, 136, 72), (1, 72, 72), (4230, 72, 1544),
                                      (8363, 200, 72)])
@pytest.mark.parametrize("t", [U16, F32])
def test_feed_forward(gpu, rows, H, I, t):
    from ancora_cutile_amd import DevBuf, ffn_down, gated_ffn_dx, gated_ffn_grad
    rng = np.random.default_rng(rows)
    dev = {n: DevBuf(_bits(rng, s, std)) for n, s, std in (("Wg", (H, I), H ** -0.5), ("Wu", (H, I), H ** -0.5), ("Wd", (I, H), I ** -0.5), ("h", (rows, I), 1.0),
                                                            ("dy", (rows, H), 1.0), ("gate", (rows, I), 1.0), ("up", (rows, I), 1.0))}
    res = _bits(rng, (rows, H)) if t == U16 else rng.standard_normal((rows, H), dtype=F32)
    own, on = DevBuf(np.zeros_like(res)), DevBuf(res)
    r = DevBuf(res)
    ffn_down(dev["h"], dev["Wd"], 0, own, residual=r)
    ffn_down(dev["h"], dev["Wd"], 0, on, residual=on)
    assert bits_equal(on.to_numpy(), own.to_numpy())
    on.upload(res)
    gated_ffn_dx(dev["gate"], dev["up"], dev["Wg"], dev["Wu"], 0, own, residual=r)
    gated_ffn_dx(dev["gate"], dev["up"], dev["Wg"], dev["Wu"], 0, on, residual=on)
    assert bits_equal(on.to_numpy(), own.to_numpy())
    if t == U16:
        dg, du, h, h2 = (DevBuf(np.zeros((rows, I), U16)) for _ in range(4))
        gated_ffn_grad(dev["dy"], dev["gate"], dev["up"], dev["Wd"], 0, dg, du, h=h)
        gated_ffn_grad(dev["dy"], dev["gate"], dev["up"], dev["Wd"], 0, dev["gate"], dev["up"], h=h2)
        assert bits_equal(dev["gate"].to_numpy(), dg.to_numpy()) and bits_equal(dev["up"].to_numpy(), du.to_numpy()) and bits_equal(h.to_numpy(), h2.to_numpy())
        for b in (dg, du, h, h2):
            b.free()
    for b in (*dev.values(), own, on, r):
        b.free()
