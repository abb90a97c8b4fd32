"""AdamW with 8-bit moments at both ends of fp32's range: the step is the 32-bit kernel's, operation by operation, wherever the corrected
moments fall. Everything is compared with the numpy oracle bit for bit."""
import numpy as np
import pytest

from oracle import adamw8_ref as ref
from util import bits_equal, max_ulp

pytestmark = pytest.mark.gpu
F32 = np.float32


def _run(p, g, steps, eps, lr, wd, betas=(0.9, 0.95), form="div"):
    from ancora_cutile_amd import AdamW
    opt, r = AdamW({"p": p}, state_bits=8, lr=lr, betas=betas, eps=eps, wd=wd, form=form), ref.Tensor8(p)
    for t in range(1, steps + 1):
        opt.step({"p": g}, 0)
        r.step(g, lr, *betas, eps, wd, t, 1000003 * t, form=form)
        s = opt.st["p"]
        got, ok = s["p32"].to_numpy(), np.isfinite(r.p)
        assert np.array_equal(np.isfinite(got), ok) and ok.mean() > 0.9, t
        assert max_ulp(got[ok], r.p[ok]) == 0, t
        for k, want in (("ms", r.ms), ("vs", r.vs)):
            assert bits_equal(s[k].to_numpy(), want), (t, k)
        for k, want in (("m", r.m), ("v", r.v), ("p16", r.p16.reshape(-1, 64))):
            assert bits_equal(s[k].to_numpy()[ok], want[ok]), (t, k)
    opt.free()


@pytest.mark.parametrize("form", ["div", "ibc"])
def test_a_second_moment_whose_correction_overflows(gpu, form):
    """v = 0.05 g^2 is finite up to |g| = 8.2e19, v / bc2 = g^2 from 1.8e19 on is not: the update is m / infinity = 0, as in fp32, until v itself has grown
    beyond fp32. Gradients on both sides, alone among small ones and by whole blocks."""
    rng = np.random.default_rng(1)
    n = 64 * 70
    g = rng.standard_normal(n).astype(F32)
    big = rng.random(n) < 0.3
    big[:128] = True
    g[big] = (np.exp2(rng.uniform(63.0, 65.9, n)) * np.where(rng.random(n) < 0.5, -1, 1)).astype(F32)[big]        # 9.2e18 .. 6.9e19
    _run(rng.standard_normal(n).astype(F32), g, 3, 1e-8, 1e-3, 0.01, form=form)


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.9, 0.999999)])
def test_moments_whose_remainders_leave_the_range(gpu, betas):
    """Gradients from the least fp32 on, with an eps so small that the quotients' last bits reach the weights."""
    rng = np.random.default_rng(2)
    n = 64 * 300
    g = (np.exp2(rng.uniform(-148, -30, n)) * np.where(rng.random(n) < 0.5, -1, 1)).astype(F32)
    g[64:128] = 0.0
    p = np.where(rng.random(n) < 0.5, 0.0, 1e-3 * rng.standard_normal(n)).astype(F32)
    _run(p, g, 4, 1e-30, 1e-3, 0.0, betas)
