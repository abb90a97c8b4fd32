"""Fills write their words and no others, whatever their place and number."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_fill_around_alignments(gpu):
    from ancora_cutile_amd import DevBuf
    rng = np.random.default_rng(0)
    host = rng.integers(0, 2 ** 32, 6000, dtype=np.uint64).astype(np.uint32)
    b = DevBuf(host)
    for at in range(9):
        for n in (0, 1, 2, 3, 4, 5, 7, 8, 63, 1024, 1025, 4099):
            b.upload(host)
            gpu.api.anc_fill_u32(b.ptr + 4 * at, 0xABCD1234, n, 0)
            want = host.copy()
            want[at:at + n] = 0xABCD1234
            assert np.array_equal(b.to_numpy(), want), (at, n)
    b.free()
    big = DevBuf.empty((50_000_003,), np.uint32)
    gpu.api.anc_fill_u32(big.ptr, 7, big.size, 0)
    assert np.all(big.to_numpy() == 7)
    big.free()
