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


def test_a_second_moment_stops_at_the_least_code_of_its_block():
    """Every block holds one element whose gradient stays; the others had one at the first step only. Theirs decay as b2^t does while they lie above the block's least
    code, 2^-31 to 2^-30 of its largest, and then stay at that code, not at zero. Rows: first gradients of 2^-2 and of 2^-16 of the lasting one (v from 2^-4 and
    from 2^-32, at the least code from the start)."""
    g = np.full((40, 64), 2.0 ** -2, np.float32)
    g[20:] = 2.0 ** -16
    g[:, 0] = 1.0
    t, b2 = a8.Tensor8(np.zeros(g.size)), 0.95
    kept = np.zeros_like(g)
    kept[:, 0] = 1.0
    for s in range(1, 701):
        t.step(g if s == 1 else kept, 0.0, 0.9, b2, 1e-8, 0.0, s, 1000003 * s)
        if s == 41:
            v = a8.decode(t.v, t.vs, 2).astype(np.float64)[:20, 1:]
            # (a store's relative variance is at most the code's distance, a quarter, times the step's size, 0.05: over 40 steps 1.0125^40 - 1 = 0.64)
            assert abs(v.mean() / ((1 - b2) * 2.0 ** -4 * b2 ** 40) - 1) < 5 * 0.8 / v.size ** 0.5
    least = np.exp2(t.vs.astype(np.float64) - 127 - 16)
    v = a8.decode(t.v, t.vs, 2).astype(np.float64)
    assert np.array_equal(v[:, 1:], np.broadcast_to(least[:, None], (40, 63)))
    assert np.all((least >= 2.0 ** -31 * v[:, 0]) & (least <= 2.0 ** -30 * v[:, 0]))


def test_how_far_8_bit_moments_are_from_32_bit_ones():
    """400 steps of random gradients of one size against moments kept in 64 bits. A store's variance is at most the code's distance (a quarter of v, an eighth of |m|) times
    the step's size. v: steps of (1 - b2) |g^2 - v|, 0.97 v on average for Gaussian ones, add up to a relative variance of 0.25 * 0.97 (1 - b2) / (1 - b2^2), 0.35^2
    with v's own spread on top, below 0.4^2. m: 0.1 |g - m| of some 0.8, |m| 0.18 on average, m^2 0.053: 0.125 * 0.1 * 0.8 * 0.18 / 0.19 / 0.053 = 0.42^2. Means are
    those of the exact ones."""
    rng = np.random.default_rng(5)
    for b2 in (0.95, 0.999):
        t, m, v = a8.Tensor8(np.zeros(N)), np.zeros(N), np.zeros(N)
        for s in range(1, 401):
            g = rng.standard_normal(N).astype(np.float32)
            t.step(g, 0.0, 0.9, b2, 1e-8, 0.0, s, 1000003 * s)
            m, v = 0.9 * m + 0.1 * g, b2 * v + (1 - b2) * g.astype(np.float64) ** 2
        m8, v8 = a8.decode(t.m, t.ms, 3).reshape(-1), a8.decode(t.v, t.vs, 2).reshape(-1).astype(np.float64)
        dv, dm = np.sqrt(np.mean((v8 / v - 1) ** 2)), np.sqrt(np.mean((m8 - m) ** 2) / np.mean(m ** 2))
        assert dv < 0.4 and abs((v8 / v).mean() - 1) < 5 * 0.4 / N ** 0.5
        assert dm < 0.45
