"""8-bit AdamW on both sides of the line between its two launches, 2048 blocks of 4096 elements: the same bits for every tensor, whatever shares its launch."""
import numpy as np
import pytest

from util import bits_equal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [np.float32, np.uint16])
def test_a_tensor_s_bits_do_not_hang_on_the_launch(gpu, grad):
    from ancora_cutile_amd import AdamW, DevBuf
    rng = np.random.default_rng(4)
    small = {"a": 64 * 65, "b": 4096 * 3 - 64, "c": 64}
    p = {n: (0.02 * rng.standard_normal(s)).astype(np.float32) for n, s in small.items()}
    fill = {n: np.zeros(4096 * k, np.float32) for n, k in (("d", 2041), ("e", 2042))}          # with a, b, c (2, 3, 1 blocks): 2047 and 2048 of them
    results = []
    for extra in ({}, {"d": fill["d"]}, {"e": fill["e"]}):
        params = {**p, **extra}
        opt = AdamW(params, state_bits=8, sr=True, seed=3, grad_dtype=grad)
        g = {n: DevBuf((np.random.default_rng(len(n) + i).standard_normal(x.size)).astype(np.float32) if grad == np.float32
                       else np.random.default_rng(len(n) + i).integers(0x3C00, 0x3E00, x.size).astype(np.uint16)) for i, (n, x) in enumerate(params.items())}
        for _ in range(2):
            opt.step(g, 0)
        assert opt._total_blocks == 6 + sum(x.size // 4096 for x in extra.values())
        results.append({(n, k): opt.st[n][k].to_numpy() for n in small for k in ("p32", "p16", "m", "v", "ms", "vs")})
        for b in g.values():
            b.free()
        opt.free()
    for other in results[1:]:
        assert all(bits_equal(results[0][k], other[k]) for k in other)
