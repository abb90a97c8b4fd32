"""The 64-bit restatement of tokens by expert against its defining properties."""
import numpy as np
import pytest

from oracle import route_ref as ref


@pytest.mark.parametrize("T,k,E,align,seed", [(1, 1, 1, 1, 0), (17, 3, 5, 1, 1), (40, 2, 7, 8, 2), (9, 4, 3, 16, 3)])
def test_route_and_row_movers(T, k, E, align, seed):
    rng = np.random.default_rng(seed)
    experts = rng.integers(-1, E, (T, k))
    counts, offsets, slot, src = ref.route(experts, E, align)
    assert np.all(offsets % align == 0) and counts.sum() == np.count_nonzero(experts >= 0)
    for e in range(E):
        mine = slot[experts == e]
        assert np.array_equal(np.sort(mine), mine) and np.array_equal(mine, offsets[e] + np.arange(counts[e]))
        assert offsets[e + 1] - offsets[e] - counts[e] < align
    assert np.all(slot[experts < 0] == -1)
    H, S = 5, int(offsets[-1]) + 3
    x, ys, dy = rng.standard_normal((T, H)), rng.standard_normal((S, H)), rng.standard_normal((T, H))
    w = rng.standard_normal((T, k))
    # <dispatch(x), ys> = <x, dispatch's gradient of ys>
    xs = ref.dispatch(slot, x, np.zeros((S, H)))
    assert np.isclose(np.sum(xs * ys), np.sum(x * ref.combine(slot, ys)))
    # <combine(ys), dy> = <ys, dys>, and its derivative in one weight
    dys, dw = ref.combine_grad(slot, dy, ys, w)
    assert np.isclose(np.sum(ref.combine(slot, ys, w) * dy), np.sum(ys * dys))
    eps = 1e-4
    for t, j in ((0, 0), (T - 1, k - 1)):
        d = np.zeros_like(w)
        d[t, j] = eps
        diff = np.sum((ref.combine(slot, ys, w + d) - ref.combine(slot, ys, w - d)) * dy) / (2 * eps)
        assert np.isclose(diff, dw[t, j], atol=1e-9)
    # <x W, dy> = <W, dW> per expert
    W = rng.standard_normal((E, H, H))
    dW = ref.expert_dw(counts, offsets, xs, ys)
    total = sum(np.sum((xs[o:o + c] @ W[e]) * ys[o:o + c]) for e, (o, c) in enumerate(zip(offsets, counts)))
    assert np.isclose(total, np.sum(W * dW))
