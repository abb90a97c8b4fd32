"""The experts' weight gradients over ragged segments against the product in 64 bits.

Bound: bf16 products are exact in fp32; c of them are added onto one accumulator, each addition off by at most one unit in the last place of the
partial sum (the matrix instruction need not round to nearest): c 2^-23 of the sum of magnitudes, and one rounding more where it
is added onto an old gradient. The bf16 copy is the rounded fp32 result bit for bit."""
import ctypes

import numpy as np
import pytest

from oracle import route_ref as ref
from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from util import bits_equal

pytestmark = pytest.mark.gpu


def _bits(rng, shape, std=1.0):
    return bf16_rne_bits((std * rng.standard_normal(shape)).astype(np.float32)).reshape(shape)


def _plan_of(counts, align, spare=0):
    """A routed plan whose experts hold `counts` tokens, and its arrays on the host."""
    from ancora_cutile_amd import DevBuf, RoutePlan
    ids = np.repeat(np.arange(len(counts)), counts)
    ids = np.concatenate([np.random.default_rng(0).permutation(ids), np.full(spare + 1, -1)]).astype(np.int32).reshape(-1, 1)
    plan, buf = RoutePlan(ids.shape[0], 1, len(counts), align), DevBuf(ids)
    plan.route(buf, 0)
    c, o = plan.counts.to_numpy(), plan.offsets.to_numpy()
    buf.free()
    assert np.array_equal(c, counts)
    return plan, c, o


def _dirty(bits, counts, offsets):
    """NaN in every row that is not a token's."""
    bits = bits.copy()
    mine = np.zeros(bits.shape[0], bool)
    for c, o in zip(counts, offsets[:-1]):
        mine[o:o + c] = True
    bits[~mine] = 0x7FFF
    return bits


def _check(got, counts, offsets, x, dy, base=None):
    xv, dv = (np.nan_to_num(bits_to_f32(a).reshape(a.shape)) for a in (x, dy))
    want, mag = ref.expert_dw(counts, offsets, xv, dv), ref.expert_dw(counts, offsets, np.abs(xv), np.abs(dv))
    bound = counts[:, None, None] * 2.0 ** -23 * mag
    if base is not None:
        want = want + base
        bound = bound + 2.0 ** -24 * (np.abs(want) + bound)
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) - bound).max())


@pytest.mark.parametrize("K,N", [(8, 8), (1536, 2304), (64, 264), (128, 256), (136, 1000), (640, 392), (264, 72), (1024, 512)])
@pytest.mark.parametrize("counts,align", [((0, 1, 31, 32, 33), 1), ((64, 0, 100, 5, 0, 95, 96, 97), 16), ((3,), 128), ((1000, 1, 257), 32)])
def test_against_64_bits(gpu, K, N, counts, align):
    from ancora_cutile_amd import DevBuf, expert_dW
    rng = np.random.default_rng(K + N + len(counts))
    plan, c, o = _plan_of(counts, align, spare=7)
    E = len(counts)
    x, dy = _dirty(_bits(rng, (plan.capacity, K)), c, o), _dirty(_bits(rng, (plan.capacity, N), 1e-2), c, o)
    base = rng.standard_normal((E, K, N)).astype(np.float32)
    gx, gdy, gW, gA = DevBuf(x), DevBuf(dy), DevBuf(np.full((E, K, N), np.nan, np.float32)), DevBuf(base)
    g16 = DevBuf.zeros((E, K, N), np.uint16)
    expert_dW(plan, [dict(x=gx, dy=gdy, dW=gW, g16=g16), dict(x=gx, dy=gdy, dW=gA, accumulate=True)], 0)
    got = gW.to_numpy()
    _check(got, c, o, x, dy)
    assert not got[c == 0].any()
    assert bits_equal(g16.to_numpy(), bf16_rne_bits(got).reshape(got.shape))
    _check(gA.to_numpy(), c, o, x, dy, base)
    assert bits_equal(gA.to_numpy()[c == 0], base[c == 0])
    # run to run, and each weight by itself: the bits are the expert's own
    gW.upload(base)
    expert_dW(plan, [dict(x=gx, dy=gdy, dW=gW)], 0)
    assert bits_equal(gW.to_numpy(), got)
    for b in (plan, gx, gdy, gW, gA, g16):
        b.free()


def test_an_experts_bits_do_not_depend_on_the_others(gpu):
    from ancora_cutile_amd import DevBuf, expert_dW
    K, N = 136, 264
    rng = np.random.default_rng(5)
    rows = 321
    x, dy = _bits(rng, (rows, K)), _bits(rng, (rows, N))
    seen = []
    for counts, at in (((rows,), 0), ((500, 3, rows, 0, 64), 2), ((rows, 900), 0)):
        plan, c, o = _plan_of(counts, 16)
        fx, fdy = _bits(rng, (plan.capacity, K)), _bits(rng, (plan.capacity, N))
        fx[o[at]:o[at] + rows], fdy[o[at]:o[at] + rows] = x, dy
        gx, gdy, gW = DevBuf(fx), DevBuf(fdy), DevBuf.empty((len(counts) * K, N), np.float32)
        expert_dW(plan, [dict(x=gx, dy=gdy, dW=gW)], 0)
        seen.append(gW.to_numpy().reshape(len(counts), K, N)[at])
        for b in (plan, gx, gdy, gW):
            b.free()
    assert bits_equal(seen[0], seen[1]) and bits_equal(seen[0], seen[2])


def test_more_weights_than_one_call_takes_and_non_finite_rows(gpu):
    from ancora_cutile_amd import DevBuf, expert_dW
    rng = np.random.default_rng(6)
    plan, c, o = _plan_of((40, 70, 9), 8)
    x, dy = _bits(rng, (plan.capacity, 72)), _bits(rng, (plan.capacity, 40))
    x[o[1] + 4, 7] = 0x7F80                          # one infinity: a row of expert 1's gradient
    gx, gdy = DevBuf(x), DevBuf(dy)
    outs = [DevBuf.empty((3, 72, 40), np.float32) for _ in range(19)]
    expert_dW(plan, [dict(x=gx, dy=gdy, dW=w) for w in outs], 0)
    got = [w.to_numpy() for w in outs]
    assert all(bits_equal(g, got[0]) for g in got[1:])
    bad = ~np.isfinite(got[0])
    assert bad[1, 7].all() and np.count_nonzero(bad) == 40
    xv = x.copy()
    xv[o[1] + 4, 7] = 0
    keep = got[0].copy()
    keep[1, 7] = ref.expert_dw(c, o, bits_to_f32(xv).reshape(x.shape), bits_to_f32(dy).reshape(dy.shape))[1, 7]
    _check(keep, c, o, xv, dy)
    for b in (plan, gx, gdy, *outs):
        b.free()


def test_no_tokens_at_all(gpu):
    from ancora_cutile_amd import DevBuf, RoutePlan, expert_dW
    plan, ids = RoutePlan(20, 2, 3, 16), DevBuf(np.zeros((20, 2), np.int32))
    plan.route(ids, 0, 0)
    x, dy = DevBuf(np.full((plan.capacity, 16), 0x7FFF, np.uint16)), DevBuf(np.full((plan.capacity, 24), 0x7FFF, np.uint16))
    base = np.arange(3 * 16 * 24, dtype=np.float32).reshape(3, 16, 24)
    W, A, g16 = DevBuf(base), DevBuf(base), DevBuf.zeros((3, 16, 24), np.uint16)
    expert_dW(plan, [dict(x=x, dy=dy, dW=W), dict(x=x, dy=dy, dW=A, g16=g16, accumulate=True)], 0)
    assert not W.to_numpy().any() and bits_equal(A.to_numpy(), base) and bits_equal(g16.to_numpy(), bf16_rne_bits(base).reshape(base.shape))
    for b in (plan, ids, x, dy, W, A, g16):
        b.free()


def test_captured_and_replayed_on_new_segments(gpu):
    from ancora_cutile_amd import DevBuf, RoutePlan, expert_dW
    hip = ctypes.CDLL("libamdhip64.so")
    T, k, E, K, N = 400, 2, 6, 200, 304
    rng = np.random.default_rng(7)
    s = gpu.stream_create()
    plans = [RoutePlan(T, k, E, 4) for _ in range(2)]
    S = plans[0].capacity
    e, gx, gdy = DevBuf(np.zeros((T, k), np.int32)), DevBuf(_bits(rng, (S, K))), DevBuf(_bits(rng, (S, N)))
    outs = [DevBuf.zeros((E, K, N), np.float32) for _ in range(2)]

    def go(i, si):
        plans[i].route(e, si)
        expert_dW(plans[i], [dict(x=gx, dy=gdy, dW=outs[i])], si)

    graph, graph_exec = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(ctypes.c_void_p(s), 0) == 0
    go(0, s)
    assert hip.hipStreamEndCapture(ctypes.c_void_p(s), ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, ctypes.c_size_t(0)) == 0
    for r in range(4):
        e.upload(np.minimum((E * rng.random((T, k)) ** (r + 1)).astype(np.int32), E - 1) - (r == 3))
        go(1, 0)
        gpu.stream_sync(0)
        assert hip.hipGraphLaunch(graph_exec, ctypes.c_void_p(s)) == 0
        gpu.stream_sync(s)
        assert bits_equal(outs[0].to_numpy(), outs[1].to_numpy()), r
    hip.hipGraphExecDestroy(graph_exec)
    hip.hipGraphDestroy(graph)
    for b in (*plans, e, gx, gdy, *outs):
        b.free()
    gpu.api.anc_stream_destroy(s)


@pytest.mark.parametrize("counts,align", [((1100, 1, 0, 31), 1), ((33, 700, 0, 320), 64)])
def test_large_ragged_weights_with_long_and_short_segments(gpu, counts, align):
    """Enough outputs and long enough segments for the widest tiles, which reach over the weight's edges here."""
    test_against_64_bits(gpu, 2296, 2056, counts, align)
