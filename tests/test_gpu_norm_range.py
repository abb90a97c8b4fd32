"""Where the norm's squares leave fp32: a row is right up to squares that add up to 2^128, whatever its width, and zeros beyond."""
import numpy as np
import pytest

from oracle import layer_ref as ref

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.mark.parametrize("H", [8, 1024, 16384])
def test_both_sides_of_the_limit(gpu, H):
    """Magnitudes of 2^64 / sqrt(H), a hundredth less (1 - 2 / 100 of the limit; 16384 additions round up by 2^-10 of the sum at most) and a hundredth more; the bound
    of a row below is that of the norm's own tests: (H + 2) 2^-25 + 7 2^-24 and the output's half step."""
    from ancora_cutile_amd import DevBuf, rms_norm
    rng = np.random.default_rng(H)
    T, limit = 6, 2.0 ** 64 / H ** 0.5
    x = np.where(rng.random((T, H)) < 0.5, -1.0, 1.0) * limit * np.where(np.arange(T) % 2, 1.01, 0.99)[:, None]
    x, gain = x.astype(F32), (1 + 0.1 * rng.standard_normal(H)).astype(F32)
    bufs = xd, g, y, r = DevBuf(x), DevBuf(gain), DevBuf(np.full((T, H), 7, F32)), DevBuf(np.full(T, 7, F32))
    rms_norm(xd, g, 0, y=y, rstd=r)
    want, wr = ref.rms_norm(x, gain, 1e-6)
    got, e = y.to_numpy(), (H + 2) * 2.0 ** -25 + 8 * 2.0 ** -24
    assert np.all(np.abs(got[::2] - want[::2]) <= e * np.abs(want[::2])) and np.all(np.abs(r.to_numpy()[::2] - wr[::2]) <= e * wr[::2])
    assert not got[1::2].any() and not r.to_numpy()[1::2].any()
    for b in bufs:
        b.free()
