"""AdamW with 8-bit moments against the numpy oracle: everything it writes, bit for bit."""
import ctypes

import numpy as np
import pytest

from oracle import adamw8_ref as ref
from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from util import bf16_grad, bits_equal, max_ulp

pytestmark = pytest.mark.gpu


def _same(opt, refs, where):
    for n, r in refs.items():
        s = opt.st[n]
        assert max_ulp(s["p32"].to_numpy(), r.p) == 0, (where, n)
        for k, want in (("m", r.m), ("v", r.v), ("ms", r.ms), ("vs", r.vs), ("p16", r.p16.reshape(-1, 64))):
            assert bits_equal(s[k].to_numpy(), want), (where, n, k)


@pytest.mark.parametrize("form", ["div", "ibc"])
@pytest.mark.parametrize("grad", [np.float32, np.uint16])
@pytest.mark.parametrize("sr", [False, True])
def test_steps_against_the_oracle(gpu, form, grad, sr):
    from ancora_cutile_amd import AdamW
    rng = np.random.default_rng(3)
    sizes = {"a": (64,), "b": (128,), "c": (5, 64 * 13), "d": (4096,), "e": (64, 65), "f": (9000 * 64,)}
    p = {n: (0.02 * rng.standard_normal(s)).astype(np.float32) for n, s in sizes.items()}
    lr, b1, b2, eps, wd = 1e-3, 0.9, 0.95, 1e-8, 0.1
    opt = AdamW(p, lr=lr, betas=(b1, b2), eps=eps, wd=wd, no_decay=("b",), form=form, sr=sr, seed=99, grad_dtype=grad, state_bits=8)
    refs = {n: ref.Tensor8(x) for n, x in p.items()}
    for t in range(1, 6):
        g = {}
        for n, s in sizes.items():
            x = (rng.standard_normal(s) * np.exp2(rng.integers(-20, 1, s))).astype(np.float32)
            x[rng.random(s) < 0.2] = 0.0
            g[n] = x if grad == np.float32 else bf16_rne_bits(x).reshape(s)
        opt.step(g, 0)
        for i, n in enumerate(sizes):
            gv = g[n] if grad == np.float32 else bits_to_f32(g[n])
            refs[n].step(gv, lr, b1, b2, eps, 0.0 if n == "b" else wd, t, 99 + 1000003 * t + i, sr, form=form)
        _same(opt, refs, t)
    for n, (m, v) in opt.moments().items():
        assert bits_equal(m.reshape(-1, 64), ref.decode(refs[n].m, refs[n].ms, 3)) and bits_equal(v.reshape(-1, 64), ref.decode(refs[n].v, refs[n].vs, 2))
    opt.free()


def test_extreme_moments(gpu):
    """Gradients from the smallest to the largest that leave a finite step, zeros, infinities and NaN; blocks of one size and mixed ones. A NaN
    stays with its element, the block's others go on."""
    from ancora_cutile_amd import AdamW
    rng = np.random.default_rng(5)
    n = 64 * 70
    g = (np.exp2(rng.uniform(-40, 30, n)) * np.where(rng.random(n) < 0.5, -1, 1)).astype(np.float32)
    g[:64] = 0.0
    g[64:128] = 1e-30
    g[128:192] = 1e-22                                    # squares are subnormal
    g[192:256] = 1.8e19
    g[300], g[400], g[500] = np.inf, -np.inf, np.nan
    p = rng.standard_normal(n).astype(np.float32)
    opt, r = AdamW({"p": p}, state_bits=8, lr=1e-3, wd=0.0), ref.Tensor8(p)
    for t in range(1, 4):
        opt.step({"p": g}, 0)
        r.step(g, 1e-3, 0.9, 0.95, 1e-8, 0.0, t, 1000003 * t)
        s = opt.st["p"]
        got, ok = s["p32"].to_numpy(), np.isfinite(r.p)
        assert np.array_equal(np.isfinite(got), ok) and max_ulp(got[ok], r.p[ok]) == 0
        for k in ("ms", "vs"):
            assert bits_equal(s[k].to_numpy(), getattr(r, k)), (t, k)
        fm = r.m & 0x7F != 0x7F
        assert bits_equal(s["m"].to_numpy()[fm], r.m[fm]) and np.all(s["m"].to_numpy()[~fm] & 0x7F == 0x7F)
        assert bits_equal(s["v"].to_numpy() & 0x7F, r.v & 0x7F)
        assert not ok.all() and np.count_nonzero(~ok) == 3
    opt.free()


def test_guarded_steps_counted_on_the_device(gpu):
    """Unsynchronised steps of the hybrid optimizer, one of them skipped: as the oracle's steps without it, and a resumed run goes on."""
    from ancora_cutile_amd import DevBuf, HybridOptimizer
    rng = np.random.default_rng(6)
    p = {"embed": (0.02 * rng.standard_normal((50, 64))).astype(np.float32), "gain_norm": np.ones(64, np.float32)}
    kw = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, wd=0.1, state_bits=8, seed=5)

    def make():
        return HybridOptimizer(p, adamw_kw=dict(kw), max_grad_norm=1e9, grad_dtype=np.uint16)
    opt, refs, t = make(), {n: ref.Tensor8(x) for n, x in p.items()}, 0
    saved = None
    for step in range(5):
        bits = {n: bf16_grad(rng, x.shape, 0.1) for n, x in p.items()}
        if step == 2:
            bits["embed"][0][3, 3] = 0x7F80
        grads = {n: DevBuf(b[0]) for n, b in bits.items()}
        opt.step(grads, 0, sync=False)
        if step != 2:
            t += 1
            for i, n in enumerate(p):
                refs[n].step(bits[n][1], 1e-2, 0.9, 0.95, 1e-8, 0.1 if n == "embed" else 0.0, t, 5 + 1000003 * t + i)
        assert opt.last_skipped == (step == 2)
        _same(opt.adamw, refs, step)
        for b in grads.values():
            b.free()
        if step == 3:
            saved = opt.state_dict()
            other = make()
            other.load_state_dict(saved)
            opt.free()
            opt = other
    wide = HybridOptimizer(p, adamw_kw=dict(lr=1e-2), max_grad_norm=1e9, grad_dtype=np.uint16)
    with pytest.raises(ValueError):
        wide.load_state_dict(saved)
    opt.free()
    wide.free()


def test_captured_and_replayed(gpu):
    """A captured launch carries its step's number and is repeated as it was: every replay against the oracle's same step from there."""
    from ancora_cutile_amd import AdamW, DevBuf
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng(8)
    p, g = rng.standard_normal(64 * 33).astype(np.float32), rng.standard_normal(64 * 33).astype(np.float32)
    opt, r, gb, s = AdamW({"p": p}, state_bits=8, wd=0.0), ref.Tensor8(p), DevBuf(g), gpu.stream_create()
    opt.step({"p": gb}, s)                                # (the table of addresses is uploaded by the first)
    r.step(g, 3e-4, 0.9, 0.95, 1e-8, 0.0, 1, 1000003)
    graph, graph_exec = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(ctypes.c_void_p(s), 0) == 0
    opt.launch({"p": gb}, s)
    assert hip.hipStreamEndCapture(ctypes.c_void_p(s), ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(3):
        assert hip.hipGraphLaunch(graph_exec, ctypes.c_void_p(s)) == 0
        gpu.stream_sync(s)
        r.step(g, 3e-4, 0.9, 0.95, 1e-8, 0.0, 2, 2 * 1000003)
        _same(opt, {"p": r}, "replay")
    hip.hipGraphExecDestroy(graph_exec)
    hip.hipGraphDestroy(graph)
    opt.free()
    gb.free()
    gpu.api.anc_stream_destroy(s)
