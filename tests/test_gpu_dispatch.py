"""Tokens by expert and back against the 64-bit restatement: the routing exactly, rows that are moved bit for bit, sums within
their bounds.

Bounds: y is k fused products in fp32, at most (k + 1) 2^-24 of the sum of magnitudes, and one rounding to its type; dw is H
products summed in fp32 in some order, at most (H + 1) 2^-24 of the sum of magnitudes; dys is one fp32 product rounded to its type, bit
for bit."""
import ctypes

import numpy as np
import pytest

from oracle import route_ref as ref
from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from util import bits_equal

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _rows(rng, shape, kind):
    x = rng.standard_normal(shape).astype(np.float32)
    if kind == "f32":
        return x, x
    b = bf16_rne_bits(x).reshape(shape)
    return b, bits_to_f32(b).reshape(shape)


def _values(a):
    return bits_to_f32(a).reshape(a.shape) if a.dtype == np.uint16 else a


def _rounded(x, kind):
    x = np.asarray(x, np.float32)
    return bf16_rne_bits(x).reshape(x.shape) if kind == "bf16" else x


def _experts(rng, T, k, E, how):
    if how == "even":
        e = rng.integers(0, E, (T, k))                         # the same expert may come twice
    elif how == "masked":
        e = rng.integers(0, E, (T, k))
        e[rng.random(T) < 0.4] = -1                            # tokens without any expert
        e[rng.random((T, k)) < 0.1] = E                        # choices that name none
    elif how == "one":
        e = np.full((T, k), E - 1)
    elif how == "none":
        e = np.full((T, k), -1)
    else:
        e = np.minimum((E * rng.random((T, k)) ** 4).astype(np.int64), E - 1)
    return e


ROUTES = [(1, 1, 1, 1), (32768, 1, 16, 16), (16385, 2, 3, 1), (4096, 8, 512, 2), (2049, 1, 1, 256), (1, 8, 128, 16), (3, 2, 5, 128), (700, 3, 7, 1), (1000, 4, 512, 4), (2048, 8, 64, 256), (5000, 8, 31, 16),
          (33, 512, 300, 2), (500, 3, 256, 8), (9000, 2, 256, 1), (9000, 3, 257, 1), (60000, 2, 512, 1), (9001, 8, 160, 128)]


@pytest.mark.parametrize("T,k,E,align", ROUTES)
def test_route(gpu, T, k, E, align):
    from ancora_cutile_amd import DevBuf, RoutePlan
    rng = np.random.default_rng(T + E)
    plan = RoutePlan(T, k, E, align)
    assert plan.capacity == T * k + min(E, T * k) * (align - 1)
    for how, dtype in (("even", np.int32), ("masked", np.int64), ("one", np.int32), ("none", np.int64), ("skewed", np.int32)):
        e = _experts(rng, T, k, E, how).astype(dtype)
        if dtype == np.int64 and how == "masked":
            e[0, 0] = 1 << 32                                  # (zero in 32 bits)
        buf = DevBuf(e)
        for n in {T, (T + 1) // 2, 0}:
            before = plan.slot.to_numpy()
            plan.route(buf, 0, n)
            counts, offsets, slot, src = ref.route(np.where((e[:n] >= 0) & (e[:n] < E), e[:n], -1), E, align)
            assert np.array_equal(plan.counts.to_numpy(), counts), (how, n)
            assert np.array_equal(plan.offsets.to_numpy(), offsets), (how, n)
            assert np.array_equal(plan.order.to_numpy(), np.argsort(-counts, kind="stable") if E <= 256 else np.arange(E)), (how, n)
            got = plan.slot.to_numpy()
            assert np.array_equal(got[:n], slot) and np.array_equal(got[n:], before[n:]), (how, n)
            full = np.full(plan.capacity, -1)
            full[:src.size] = src
            assert np.array_equal(plan.src.to_numpy(), full), (how, n)
        buf.free()
    plan.free()


@pytest.mark.parametrize("T,k,E,H,align", [(1, 1, 1, 1, 1), (1, 2, 4, 1024, 16), (5, 3, 4, 7, 128), (130, 2, 6, 64, 1), (257, 8, 40, 130, 4),
                                           (600, 5, 3, 1000, 64), (64, 70, 5, 24, 2), (2500, 8, 16, 392, 16)])
@pytest.mark.parametrize("kind,out", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
def test_there_and_back(gpu, T, k, E, H, align, kind, out):
    from ancora_cutile_amd import DevBuf, RoutePlan, combine, combine_grad, dispatch_grad
    from ancora_cutile_amd.dispatch import dispatch
    rng = np.random.default_rng(T + H)
    plan = RoutePlan(T + 1, k, E, align)                       # (room for one token more than the batch has)
    S = plan.capacity
    for how in ("even", "masked", "none"):
        e = _experts(rng, T, k, E, how)
        ge = DevBuf(e.astype(np.int32))
        plan.route(ge, 0)
        counts, offsets, slot, src = ref.route(np.where(e < E, e, -1), E, align)
        end = int(offsets[-1])
        filling = np.nonzero(src < 0)[0]
        # there
        x, xv = _rows(rng, (T, H), kind)
        before, _ = _rows(rng, (S, H), kind)
        gx, gxs = DevBuf(x), DevBuf(before)
        dispatch(plan, gx, 0, gxs)
        got = gxs.to_numpy()
        want = before.copy()
        want[filling] = 0
        for j in range(k):
            want[slot[slot[:, j] >= 0, j]] = x[slot[:, j] >= 0]
        assert bits_equal(got, want), how
        # back, weighted and plain; rows without a slot hold NaN and must not be met
        ys, yv = _rows(rng, (S, H), kind)
        ys = ys.copy()
        ys[end:] = 0x7FFF if kind == "bf16" else np.nan
        ys[filling] = 0x7FFF if kind == "bf16" else np.nan
        yv = np.nan_to_num(_values(ys), nan=0.0)
        w = rng.random((T, k)).astype(np.float32)
        tail, _ = _rows(rng, (T + 1, H), out)
        gys, gw, gy = DevBuf(ys), DevBuf(w), DevBuf(tail)
        for weights, call in ((w, lambda: combine(plan, gys, gw, 0, gy)), (None, lambda: dispatch_grad(plan, gys, 0, gy))):
            call()
            y = gy.to_numpy()
            assert bits_equal(y[T:], tail[T:])
            exact = ref.combine(slot, yv, weights)
            mag = ref.combine(slot, np.abs(yv), weights)
            bound = (k + 1) * U * mag + (2.0 ** -8 * np.abs(exact) + 2.0 ** -8 * (k + 1) * U * mag if out == "bf16" else 0.0)
            assert np.all(np.abs(_values(y[:T]) - exact) <= bound), how
        # gradients
        dy, dv = _rows(rng, (T, H), out)
        dys0, _ = _rows(rng, (S, H), kind)
        gdy, gdys, gdw = DevBuf(dy), DevBuf(dys0), DevBuf(np.full((T, k), 9.0, np.float32))
        combine_grad(plan, gdy, gys, gw, 0, gdys, gdw)
        want = dys0.copy()
        want[filling] = 0
        for j in range(k):
            at = slot[:, j] >= 0
            want[slot[at, j]] = _rounded(w[at, j, None] * dv[at], kind)
        assert bits_equal(gdys.to_numpy(), want), how
        _, dw = ref.combine_grad(slot, dv, yv, w)
        _, mag = ref.combine_grad(slot, np.abs(dv), np.abs(yv), w)
        got_dw = gdw.to_numpy()
        assert np.all(np.abs(got_dw - dw) <= (H + 1) * U * mag) and not got_dw[slot < 0].any(), how
        for b in (ge, gx, gxs, gys, gw, gy, gdy, gdys, gdw):
            b.free()
    plan.free()


def test_a_choice_without_a_slot_is_not_read_and_nan_goes_only_where_it_belongs(gpu):
    from ancora_cutile_amd import DevBuf, RoutePlan, combine, combine_grad
    T, k, E, H = 6, 2, 3, 16
    e = np.array([[0, 1], [-1, -1], [2, -1], [0, 2], [1, 1], [-1, 0]], np.int32)
    plan = RoutePlan(T, k, E, 4)
    ge = DevBuf(e)
    plan.route(ge, 0)
    slot = plan.slot.to_numpy()
    ys = np.ones((plan.capacity, H), np.float32)
    ys[slot[3, 1]] = np.nan
    w = np.full((T, k), 0.5, np.float32)
    w[1], w[2, 1], w[5, 0] = np.nan, np.inf, np.nan            # weights of choices without a slot
    w[3, 1] = 0.0                                              # zero times NaN is NaN
    gys, gw, gy = DevBuf(ys), DevBuf(w), DevBuf.zeros((T, H), np.float32)
    combine(plan, gys, gw, 0, gy)
    y = gy.to_numpy()
    assert np.all(np.isnan(y[3])) and np.array_equal(y[[0, 1, 2, 4, 5], 0], np.float32([1.0, 0.0, 0.5, 1.0, 0.5]))
    dy, gdys, gdw = DevBuf(np.ones((T, H), np.float32)), DevBuf.zeros((plan.capacity, H), np.float32), DevBuf.zeros((T, k), np.float32)
    combine_grad(plan, dy, gys, gw, 0, gdys, gdw)
    dw = gdw.to_numpy()
    assert np.isnan(dw[3, 1]) and np.count_nonzero(np.isnan(dw)) == 1 and not dw[slot < 0].any()
    assert np.all(np.isfinite(gdys.to_numpy()))
    for b in (plan, ge, gys, gw, gy, dy, gdys, gdw):
        b.free()


def test_rows_beyond_32_bit_offsets(gpu):
    """One expert's segment lies behind 2^31 elements of another's filling up: rows there and back by 64-bit offsets."""
    from ancora_cutile_amd import DevBuf, RoutePlan, combine
    from ancora_cutile_amd.dispatch import dispatch
    T, H = 40000, 65536                                        # 2.6e9 elements of xs, 5 GB
    plan = RoutePlan(T, 1, 2)
    e = np.ones((T, 1), np.int32)
    ge, gx, gxs = DevBuf(e), DevBuf.empty((T, H), np.uint16), DevBuf.empty((T, H), np.uint16)
    marks = {0: 11, 32767: 12, 32768: 13, T - 1: 14}
    gx.fill_zero(0)
    for t, v in marks.items():
        DevBuf(shape=(H,), dtype=np.uint16, ptr=gx.ptr + t * H * 2).upload(np.full(H, 0x3F80 + v, np.uint16))
    plan.route(ge, 0)
    dispatch(plan, gx, 0, gxs)
    gx.fill_zero(0)
    combine(plan, gxs, None, 0, gx)
    for t, v in marks.items():
        got = DevBuf(shape=(H,), dtype=np.uint16, ptr=gx.ptr + t * H * 2).to_numpy()
        assert np.all(got == 0x3F80 + v), t
    assert not DevBuf(shape=(H,), dtype=np.uint16, ptr=gx.ptr + 20000 * H * 2).to_numpy().any()
    for b in (plan, ge, gx, gxs):
        b.free()


def test_slots_and_segments_that_hold_anything_touch_no_other_row(gpu):
    from ancora_cutile_amd import DevBuf, RoutePlan, combine, combine_grad, expert_dW
    from ancora_cutile_amd.dispatch import dispatch
    T, k, E, H, align, guard = 500, 3, 7, 40, 8, 64
    rng = np.random.default_rng(1)
    plan = RoutePlan(T, k, E, align)
    S = plan.capacity
    ge = DevBuf(np.zeros((T, k), np.int32))
    plan.route(ge, 0)
    outer = {n: DevBuf(np.full((S + 2 * guard, H), 0x4040, np.uint16)) for n in ("xs", "dys")}
    inner = {n: DevBuf(shape=(S, H), dtype=np.uint16, ptr=b.ptr + guard * H * 2) for n, b in outer.items()}
    x, y, w = DevBuf.zeros((T, H), np.uint16), DevBuf.zeros((T, H), np.float32), DevBuf(np.ones((T, k), np.float32))
    dw, dW = DevBuf.zeros((T, k), np.float32), DevBuf.zeros((E, H, H), np.float32)
    for _ in range(3):
        for a in (plan.slot, plan.counts, plan.offsets, plan.order):
            r = rng.integers(-2 ** 31, 2 ** 31 - 1, a.shape) >> rng.integers(0, 31, a.shape)
            a.upload(r.astype(np.int32))
        dispatch(plan, x, 0, inner["xs"])
        combine(plan, inner["xs"], w, 0, y)
        combine_grad(plan, y, inner["xs"], w, 0, inner["dys"], dw)
        expert_dW(plan, [dict(x=inner["xs"], dy=inner["dys"], dW=dW)], 0)
    gpu.stream_sync(0)
    for b in outer.values():
        host = b.to_numpy()
        assert np.all(host[:guard] == 0x4040) and np.all(host[guard + S:] == 0x4040)
    for b in (plan, ge, x, y, w, dw, dW, *outer.values()):
        b.free()


@pytest.mark.parametrize("T", [50, 6000])
def test_captured_and_replayed_on_new_routes(gpu, T):
    from ancora_cutile_amd import DevBuf, RoutePlan, combine, combine_grad, dispatch_grad
    from ancora_cutile_amd.dispatch import dispatch
    hip = ctypes.CDLL("libamdhip64.so")
    k, E, H, align = 4, 9, 72, 16
    rng = np.random.default_rng(T)
    s = gpu.stream_create()
    plans = [RoutePlan(T, k, E, align) for _ in range(2)]
    S = plans[0].capacity
    e, w = DevBuf(np.zeros((T, k), np.int32)), DevBuf(rng.random((T, k)).astype(np.float32))
    x, dy = DevBuf(_rows(rng, (T, H), "bf16")[0]), DevBuf(_rows(rng, (T, H), "bf16")[0])
    outs = [[DevBuf.zeros(sh, dt) for sh, dt in (((S, H), np.uint16), ((T, H), np.uint16), ((S, H), np.uint16), ((T, k), np.float32),
                                                 ((T, H), np.uint16))] for _ in range(2)]

    def go(i, si):
        xs, y, dys, dw, dx = outs[i]
        plans[i].route(e, si)
        dispatch(plans[i], x, si, xs)
        combine(plans[i], xs, w, si, y)
        combine_grad(plans[i], dy, xs, w, si, dys, dw)
        dispatch_grad(plans[i], dys, si, dx)

    graph, graph_exec = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(ctypes.c_void_p(s), 0) == 0
    go(0, s)
    assert hip.hipStreamEndCapture(ctypes.c_void_p(s), ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, ctypes.c_size_t(0)) == 0
    for r in range(4):
        e.upload(_experts(rng, T, k, E, ("even", "masked", "one", "skewed")[r]).astype(np.int32))
        for o in outs:
            for b in o:
                b.fill_zero(0)
        go(1, 0)
        gpu.stream_sync(0)
        assert hip.hipGraphLaunch(graph_exec, ctypes.c_void_p(s)) == 0
        gpu.stream_sync(s)
        for a, b in zip(*outs):
            assert bits_equal(a.to_numpy(), b.to_numpy()), r
        assert np.array_equal(plans[0].src.to_numpy(), plans[1].src.to_numpy())
    hip.hipGraphExecDestroy(graph_exec)
    hip.hipGraphDestroy(graph)
    for b in (*plans, e, w, x, dy, *outs[0], *outs[1]):
        b.free()
    gpu.api.anc_stream_destroy(s)


def test_weight_gradient_against_differences(gpu):
    """The loss sum(y * dy) is linear in every weight: its difference over a step of 1/8 in one weight is the gradient to
    the accuracy of fp32 sums."""
    from ancora_cutile_amd import DevBuf, RoutePlan, combine, combine_grad
    T, k, E, H = 12, 3, 5, 48
    rng = np.random.default_rng(0)
    plan = RoutePlan(T, k, E)
    e, w = rng.integers(-1, E, (T, k)).astype(np.int32), rng.random((T, k)).astype(np.float32)
    ys, dy = rng.standard_normal((plan.capacity, H)).astype(np.float32), rng.standard_normal((T, H)).astype(np.float32)
    ge, gw, gys, gdy = DevBuf(e), DevBuf(w), DevBuf(ys), DevBuf(dy)
    gy, gdys, gdw = DevBuf.zeros((T, H), np.float32), DevBuf.zeros(ys.shape, np.float32), DevBuf.zeros((T, k), np.float32)
    plan.route(ge, 0)
    combine_grad(plan, gdy, gys, gw, 0, gdys, gdw)
    dw = gdw.to_numpy()

    def loss(w):
        gw.upload(w)
        combine(plan, gys, gw, 0, gy)
        return np.sum(gy.to_numpy().astype(np.float64) * dy, axis=1)

    for j in range(k):
        d = np.zeros_like(w)
        d[:, j] = 0.125
        diff = (loss(w + d) - loss(w - d)) / ((w + d)[:, j].astype(np.float64) - (w - d)[:, j])
        scale = 2 * (k + 1) * U * np.sum(np.abs(dy), axis=1) * np.abs(ys).max() * 2 * k / 0.125
        assert np.all(np.abs(diff - dw[:, j]) <= scale + (H + 1) * U * np.sum(np.abs(dy), axis=1) * np.abs(ys).max())
    for b in (plan, ge, gw, gys, gdy, gy, gdys, gdw):
        b.free()
