"""AdamW with 8-bit moments under graph capture: a launch that carries its own step's dither is refused, one that takes the count of steps from the
device is a step of its own at every replay."""
import ctypes

import numpy as np
import pytest

from oracle import adamw8_ref as ref
from util import bits_equal, max_ulp

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.mark.parametrize("sr", [False, True])
def test_a_launch_with_its_own_dither_is_refused(gpu, sr):
    from ancora_cutile_amd import AdamW, DevBuf
    from ancora_cutile_amd._lib import AncoraError
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng(8)
    p, g = rng.standard_normal(64 * 33).astype(F32), rng.standard_normal(64 * 33).astype(F32)
    opt, wide, r = AdamW({"p": p}, state_bits=8, wd=0.0, sr=sr), AdamW({"p": p}, wd=0.0, sr=sr), ref.Tensor8(p)
    gb, s = DevBuf(g), gpu.stream_create()
    for o in (opt, wide):
        o.step({"p": gb}, s)
    r.step(g, 3e-4, 0.9, 0.95, 1e-8, 0.0, 1, 1000003, sr)
    graph, error = ctypes.c_void_p(), None
    assert hip.hipStreamBeginCapture(ctypes.c_void_p(s), 0) == 0
    try:
        opt.launch({"p": gb}, s)
    except AncoraError as e:
        error = e
    wide.launch({"p": gb}, s)                       # (moments of 32 bits have no dither: the one node of the graph)
    assert hip.hipStreamEndCapture(ctypes.c_void_p(s), ctypes.byref(graph)) == 0
    nodes = ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(graph, None, ctypes.byref(nodes)) == 0 and nodes.value == 1
    hip.hipGraphDestroy(graph)
    assert error is not None and "captured" in str(error) and opt.t == 1
    for t in (2, 3):
        opt.step({"p": gb}, s)
        r.step(g, 3e-4, 0.9, 0.95, 1e-8, 0.0, t, t * 1000003, sr)
        st = opt.st["p"]
        assert max_ulp(st["p32"].to_numpy(), r.p) == 0 and bits_equal(st["m"].to_numpy(), r.m) and bits_equal(st["v"].to_numpy(), r.v)
    for o in (opt, wide, gb):
        o.free()
    gpu.api.anc_stream_destroy(s)


def test_replays_of_steps_counted_on_the_device(gpu):
    """A guarded step in a graph, replayed between eager steps of another optimizer on the same gradients: the same bits after every one, and moments that go on
    moving (the means of a constant gradient's, as the oracle's own test bounds them)."""
    from ancora_cutile_amd import DevBuf, HybridOptimizer
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng(9)
    params = {"embed": (0.02 * rng.standard_normal((50, 64))).astype(F32), "gain_norm": np.ones(64 * 9, F32)}
    host = {n: np.full(p.shape, 2.0 ** -10, F32) for n, p in params.items()}
    grads = {n: DevBuf(g) for n, g in host.items()}

    def make():
        return HybridOptimizer(params, max_grad_norm=1e9, adamw_kw=dict(lr=1e-4, betas=(0.9, 0.999), wd=0.1, sr=True, seed=5, state_bits=8))
    eager, captured, s = make(), make(), gpu.stream_create()
    eager.step(grads, s)
    captured.step(grads, s)
    graph, graph_exec = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(ctypes.c_void_p(s), 0) == 0
    captured.step(grads, s, sync=False)
    assert hip.hipStreamEndCapture(ctypes.c_void_p(s), ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in range(299):
        eager.step(grads, s)
        assert hip.hipGraphLaunch(graph_exec, ctypes.c_void_p(s)) == 0
        if i < 4 or i == 298:
            gpu.stream_sync(s)
            for n in params:
                a, b = eager.adamw.st[n], captured.adamw.st[n]
                assert all(bits_equal(a[k].to_numpy(), b[k].to_numpy()) for k in ("p32", "p16", "m", "v", "ms", "vs")), (i, n)
    assert captured.guard.read(s)["t"] == 300
    v = np.concatenate([v.reshape(-1) for _, v in captured.adamw.moments().values()]).astype(np.float64)
    assert abs(v.mean() / ((1 - 0.999 ** 300) * 2.0 ** -20) - 1) < 5 * 0.36 / v.size ** 0.5
    hip.hipGraphExecDestroy(graph_exec)
    hip.hipGraphDestroy(graph)
    for o in (eager, captured, *grads.values()):
        o.free()
    gpu.api.anc_stream_destroy(s)
