"""What storing moments in 8 bits does to them over many steps, on the oracle."""
import numpy as np

from oracle import adamw8_ref as a8

N = 64 * 40


def _run(seed_of, steps, b1=0.9, b2=0.999, g=1.0):
    t = a8.Tensor8(np.zeros(N))
    for s in range(1, steps + 1):
        t.step(np.full(N, g, np.float32), 0.0, b1, b2, 1e-8, 0.0, s, seed_of(s))
    return a8.decode(t.m, t.ms, 3).astype(np.float64), a8.decode(t.v, t.vs, 2).astype(np.float64)


def test_one_dither_for_every_step_freezes_the_moments():
    """300 steps of a constant gradient. With a dither of each step's own the moments' means are the exact ones: a second moment's relative spread is at most
    sqrt(1/4 / (1 + b2)) = 0.36 (the variance of a store is at most the code's distance, a quarter, times the step, and steps add up to (1 - b2) / (1 - b2^2)),
    its mean over 2560 elements within five times 0.36 / sqrt(2560) = 0.036. With one dither for all steps, as replays of a captured launch would have, a
    moment stops where its step no longer reaches over its own threshold: half of them stay below a fifth of the exact value."""
    exact = 1 - 0.999 ** 300
    m, v = _run(lambda s: 1000003 * s, 300)
    assert abs(v.mean() / exact - 1) < 0.036 and abs(m.mean() - 1) < 0.036
    m, v = _run(lambda s: 1000003, 300)
    assert np.median(v) < 0.2 * exact and v.mean() < 0.5 * exact and m.mean() < 0.9
