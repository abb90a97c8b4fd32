"""The oracles of the norm, the gated block and the 8-bit moments against differences, closed forms and their own definitions."""
import numpy as np
import pytest

from oracle import adamw8_ref as a8
from oracle import layer_ref as ref
from oracle.bf16_ref import sr_dither
from oracle.quant_ref import e4m3_table, quant_mxfp8_w


def test_norm_gradient_against_differences():
    rng = np.random.default_rng(0)
    s, gain, dy = rng.standard_normal((3, 8)), 1 + 0.1 * rng.standard_normal(8), rng.standard_normal((3, 8))
    _, r = ref.rms_norm(s, gain, 1e-3)
    ds, dgain = ref.rms_norm_grad(dy, s, gain, r)
    f, h = lambda s, g: (ref.rms_norm(s, g, 1e-3)[0] * dy).sum(), 1e-5
    for i in np.ndindex(s.shape):
        d = np.zeros_like(s)
        d[i] = h
        assert abs((f(s + d, gain) - f(s - d, gain)) / (2 * h) - ds[i]) < 1e-7
    for i in range(8):
        d = np.zeros(8)
        d[i] = h
        assert abs((f(s, gain + d) - f(s, gain - d)) / (2 * h) - dgain[i]) < 1e-7


def test_gated_gradient_against_differences():
    rng = np.random.default_rng(1)
    x, Wg, Wu, Wd, dy = (rng.standard_normal(n) for n in ((4, 6), (6, 5), (6, 5), (5, 6), (4, 6)))
    f = lambda x: ((ref.gated(x @ Wg, x @ Wu) @ Wd) * dy).sum()  # noqa: E731
    dg, du, h = ref.gated_grad(dy @ Wd.T, x @ Wg, x @ Wu)
    dx = dg @ Wg.T + du @ Wu.T
    assert np.allclose(h, ref.gated(x @ Wg, x @ Wu), rtol=1e-13)
    for i in np.ndindex(x.shape):
        d = np.zeros_like(x)
        d[i] = 1e-5
        assert abs((f(x + d) - f(x - d)) / 2e-5 - dx[i]) < 1e-7
    assert np.allclose(ref.sigmoid(np.array([-800.0, 0.0, 800.0])), [0, 0.5, 1])


def test_segments_are_products_of_their_own_rows():
    rng = np.random.default_rng(2)
    x, W = rng.standard_normal((9, 4)), rng.standard_normal((3, 4, 5))
    got = ref.by_segment(x, W, (2, 0, 3), (1, 4, 4))
    assert np.array_equal(got[1:3], x[1:3] @ W[0]) and np.array_equal(got[4:7], x[4:7] @ W[2]) and not got[[0, 3, 7, 8]].any()


def test_mx8_rows_are_the_weights_format_along_the_row():
    rng = np.random.default_rng(3)
    bits = ((rng.standard_normal((64, 96)) * np.exp2(rng.integers(-30, 30, (64, 1)))).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    y = (bits.astype(np.uint32) << 16).view(np.float32)
    codes, scale = ref.mx8_rows(y)
    wc, ws = quant_mxfp8_w(np.ascontiguousarray(bits.T))
    assert np.array_equal(codes, wc.T) and np.array_equal(scale, ws.T)


def test_8_bit_values_and_hash():
    assert np.array_equal(a8.values(3), e4m3_table()[:127])
    assert a8.values(2)[-1] == 57344 and a8.values(2)[1] == 2.0 ** -16 and a8.values(2)[4] == 2.0 ** -14
    i = np.arange(5000)
    assert np.array_equal(a8.sr_hash(i, 77) & 0xFFFF, sr_dither(i // 64, i % 64, 77))


@pytest.mark.parametrize("mantissa", [3, 2])
def test_stored_moments_are_unbiased_neighbours(mantissa):
    """Every stored value is one of the two neighbours of the exact one, itself if it is a code's, and the mean over all dithers is the
    exact value to the width of the dither."""
    rng = np.random.default_rng(4)
    x = (np.abs(rng.standard_normal((1, 64))) * np.exp2(-rng.integers(0, 24, (1, 64)))).astype(np.float32)
    step = 1 << 8
    mean = np.zeros((1, 64))
    for d in range(0, 65536, step):
        codes, scale = a8.encode(x, mantissa, np.full((1, 64), d))
        got = a8.decode(codes, scale, mantissa).astype(np.float64)
        mean += got * step / 65536
        up = np.exp2(float(scale[0]) - 127)
        t = a8.values(mantissa) * up
        lo = t[np.searchsorted(t, x, side="right") - 1]
        hi = t[np.searchsorted(t, x, side="right")]
        assert np.all((got == lo) | (got == hi))
    assert np.all(np.abs(mean - x) <= (hi - lo) * 1.02 * step / 65536)
    codes, scale = a8.encode(got.astype(np.float32), mantissa, np.full((1, 64), 65535))
    assert np.array_equal(a8.decode(codes, scale, mantissa), got.astype(np.float32)) or scale[0] != a8.encode(x, mantissa, 0)[1][0]


def test_a_decaying_moment_keeps_moving():
    """1000 steps without gradient: the mean of many second moments falls as beta2^t does (nearest rounding would leave it where it is)."""
    t = a8.Tensor8(np.ones(64 * 200))
    t.step(np.ones(64 * 200), 0.0, 0.9, 0.999, 1e-8, 0.0, 1, 1)
    v0 = a8.decode(t.v, t.vs, 2).mean()
    for s in range(2, 202):
        t.step(np.zeros(64 * 200), 0.0, 0.9, 0.999, 1e-8, 0.0, s, 1 + 1000003 * s)
    # 12800 elements, each with a relative spread of at most sqrt(step / 2) = 0.36 (a code's distance is a quarter): the mean's is 0.0032
    assert abs(a8.decode(t.v, t.vs, 2).mean() / v0 - 0.999 ** 200) < 5 * 0.0032


def test_not_finite_moments_stay_alone():
    x = np.ones((2, 64), np.float32)
    x[0, 3], x[1, 5] = np.nan, -np.inf
    codes, scale = a8.encode(x, 3, np.zeros((2, 64), np.int64))
    assert codes[0, 3] & 0x7F == 0x7F and codes[1, 5] == 0xFF and (scale == 127 - 7).all()
    v = a8.decode(codes, scale, 3)
    assert np.isnan(v).sum() == 2 and np.nanmax(np.abs(v - 1)) == 0
