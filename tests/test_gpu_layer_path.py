"""A layer's feed-forward half as a training step runs it: norm, tokens to their experts, the experts' gated block, the way back onto the
residual stream, every gradient on the way back, and AdamW with 8-bit moments on what they belong to. Every result is compared with the
64-bit formula of what the device itself read; bounds as in the operators' own tests."""
import numpy as np
import pytest

from oracle import adamw8_ref as a8
from oracle import layer_ref as lay
from oracle import route_ref as ref
from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from util import bits_equal, max_ulp

pytestmark = pytest.mark.gpu
U16, F32, U = np.uint16, np.float32, 2.0 ** -23


def _val(b):
    a = b.to_numpy()
    return a.astype(np.float64) if a.dtype == F32 else bits_to_f32(a).reshape(a.shape).astype(np.float64)


def _close(buf, want, err, rows=slice(None)):
    half = 2.0 ** -8 if buf.dtype == U16 else 2.0 ** -24
    d = np.abs(_val(buf) - want) - (err + half * (np.abs(want) + err) + 1e-30)
    assert np.all(d[rows] <= 0), float(d[rows].max())


def _product(x, W, counts, offsets):
    K = W.shape[-2]
    return lay.by_segment(x, W, counts, offsets), (K + 8) * U * lay.by_segment(np.abs(x), np.abs(W), counts, offsets)


@pytest.mark.parametrize("E", [0, 4])
def test_training_steps_of_a_layer(gpu, E):
    from ancora_cutile_amd import (AdamW, DevBuf, DwWorkspace, NormWorkspace, RoutePlan, combine, combine_grad, dispatch_grad, expert_dW, ffn_down, gated_ffn,
                                   gated_ffn_dx, gated_ffn_grad, gemm_dW, rms_norm, rms_norm_grad)
    from ancora_cutile_amd.dispatch import dispatch
    T, H, I, k = 192, 256, 256, 2
    rng = np.random.default_rng(21)
    lead = (E,) if E else ()
    params = {"gain": np.ones(H, F32), "Wg": (H ** -0.5 * rng.standard_normal(lead + (H, I))).astype(F32),
              "Wu": (H ** -0.5 * rng.standard_normal(lead + (H, I))).astype(F32), "Wd": (I ** -0.5 * rng.standard_normal(lead + (I, H))).astype(F32)}
    opt = AdamW(params, lr=1e-3, wd=0.01, no_decay=("gain",), state_bits=8, seed=3)
    refs = {n: a8.Tensor8(p) for n, p in params.items()}
    si = gpu.stream_create()
    plan = RoutePlan(T, k, E, 16) if E else None
    S = plan.capacity if E else T
    new = lambda n, w, t=U16: DevBuf.zeros((n, w), t)  # noqa: E731
    n_ = {n: new(T, H) for n in ("y", "dnorm")}
    n_.update(total=new(T, H, F32), rstd=DevBuf.zeros((T,), F32), out=new(T, H, F32), dx=new(T, H, F32), dgain=DevBuf.zeros((H,), F32), dw=new(T, k, F32),
              add=new(T, H, F32))
    n_.update({n: new(S, H) for n in ("xs", "ys", "dys", "dxs")})
    n_.update({n: new(S, I) for n in ("h", "gate", "up", "dgate", "dup", "h2")})
    grads = {n: DevBuf.zeros(p.shape, F32) for n, p in params.items() if n != "gain"}
    ws, dws = NormWorkspace(T, H), [DwWorkspace() for _ in range(3)]
    gpu.stream_sync(0)
    for step in range(1, 4):
        W16 = {}
        for n in ("Wg", "Wu", "Wd"):                          # the forward reads the optimizer's bf16 copies
            s = opt.st[n]
            if step == 1:
                s["p16"].upload(bf16_rne_bits(params[n]).reshape(s["p16"].shape))
            W16[n] = s["p16"].view(params[n].shape)
        Wv = {n: _val(b) for n, b in W16.items()}
        x, res = rng.standard_normal((T, H)).astype(F32), rng.standard_normal((T, H)).astype(F32)
        dy = (0.1 * rng.standard_normal((T, H))).astype(F32)
        experts, w = rng.integers(-1, max(E, 1), (T, k)).astype(np.int32), rng.random((T, k)).astype(F32)
        up = {n: DevBuf(a) for n, a in dict(x=bf16_rne_bits(x).reshape(T, H), res=res, dy=dy, dyb=bf16_rne_bits(dy).reshape(T, H), experts=experts, w=w).items()}
        gain = opt.st["gain"]["p32"]
        # forwards
        rms_norm(up["x"], gain, si, y=n_["y"], residual=up["res"], total=n_["total"], rstd=n_["rstd"])
        counts = offsets = slot = None
        rows = np.ones(S, bool)
        if E:
            plan.route(up["experts"], si)
            dispatch(plan, n_["y"], si, n_["xs"])
            counts, offsets, slot, _ = ref.route(experts, E, 16)
            rows[:] = False
            for c, o in zip(counts, offsets):
                rows[o:o + c] = True
        xs = n_["xs"] if E else n_["y"]
        gated_ffn(xs, W16["Wg"], W16["Wu"], si, n_["h"], gate=n_["gate"], up=n_["up"], plan=plan)
        if E:
            ffn_down(n_["h"], W16["Wd"], si, n_["ys"], plan=plan)
            combine(plan, n_["ys"], up["w"], si, n_["out"])
        else:
            ffn_down(n_["h"], W16["Wd"], si, n_["out"], residual=n_["total"])
        # backwards
        dys = n_["dys"] if E else up["dyb"]
        if E:
            combine_grad(plan, up["dy"], n_["ys"], up["w"], si, n_["dys"], n_["dw"])
        gated_ffn_grad(dys, n_["gate"], n_["up"], W16["Wd"], si, n_["dgate"], n_["dup"], h=n_["h2"], plan=plan)
        gated_ffn_dx(n_["dgate"], n_["dup"], W16["Wg"], W16["Wu"], si, n_["dxs"] if E else n_["dnorm"], plan=plan)
        pairs = (("Wg", xs, n_["dgate"]), ("Wu", xs, n_["dup"]), ("Wd", n_["h2"], dys))
        if E:
            expert_dW(plan, [dict(x=a, dy=b, dW=grads[n]) for n, a, b in pairs], si)
            dispatch_grad(plan, n_["dxs"], si, n_["dnorm"])
        else:
            gemm_dW([dict(x=a, dy=b, dW=grads[n], T=T, K=a.shape[1], N=b.shape[1], workspace=q) for (n, a, b), q in zip(pairs, dws)], si)
        rms_norm_grad(n_["dnorm"], n_["total"], gain, n_["rstd"], si, n_["dx"], n_["dgain"], ws, carry=up["dy"])
        gpu.stream_sync(si)
        # what the device made, against the formulas of what it read
        gv = _val(gain).reshape(-1)
        total = _val(up["x"]) + res
        _close(n_["total"], total, 0.0)
        yv, rv = lay.rms_norm(total, gv, 1e-6)
        _close(n_["y"], yv, np.abs(yv) * (H + 20) * 2.0 ** -24)
        xv = _val(xs)
        if E:
            assert np.array_equal(xv[rows], ref.dispatch(slot, _val(n_["y"]), np.zeros((S, H)))[rows])
        (g, ge), (u, ue) = _product(xv, Wv["Wg"], counts, offsets), _product(xv, Wv["Wu"], counts, offsets)
        _close(n_["gate"], g, ge, rows)
        _close(n_["up"], u, ue, rows)
        a = np.abs(g) * lay.sigmoid(g)
        _close(n_["h"], lay.gated(g, u), 1.1 * ge * (np.abs(u) + ue) + a * ue + a * np.abs(u) * (np.abs(g) + 10) * U, rows)
        d, de = _product(_val(n_["h"]), Wv["Wd"], counts, offsets)
        if E:
            _close(n_["ys"], d, de, rows)
            mag = ref.combine(slot, np.abs(_val(n_["ys"])), w)
            _close(n_["out"], ref.combine(slot, _val(n_["ys"]), w), (k + 1) * 2.0 ** -24 * mag)
        else:
            _close(n_["out"], d + _val(n_["total"]), de + U * np.abs(d + _val(n_["total"])))
        dyv, gv2, uv2 = _val(dys), _val(n_["gate"]), _val(n_["up"])
        dh, dhe = _product(dyv, np.swapaxes(Wv["Wd"], -1, -2), counts, offsets)
        s = lay.sigmoid(gv2)
        wg, wu, wh = lay.gated_grad(dh, gv2, uv2)
        es, slope = (np.abs(gv2) + 10) * U, s * (1 + np.abs(gv2))
        _close(n_["dgate"], wg, (dhe * 1.1 + np.abs(dh) * 2 * es) * np.abs(uv2) * slope, rows)
        _close(n_["dup"], wu, (dhe * 1.1 + np.abs(dh) * es) * np.abs(gv2) * s, rows)
        _close(n_["h2"], wh, np.abs(wh) * es, rows)
        (v1, e1), (v2, e2) = (_product(_val(n_[a]), np.swapaxes(Wv[b], -1, -2), counts, offsets) for a, b in (("dgate", "Wg"), ("dup", "Wu")))
        _close(n_["dxs"] if E else n_["dnorm"], v1 + v2, 2 * (e1 + e2), rows)
        for n, x_, b_ in pairs:
            xw, dw = _val(x_), _val(b_)
            c1, o1 = (counts, offsets) if E else (np.array([T]), np.array([0, T]))
            want, mag = ref.expert_dw(c1, o1, xw, dw), ref.expert_dw(c1, o1, np.abs(xw), np.abs(dw))
            assert np.all(np.abs(_val(grads[n]).reshape(want.shape) - want) <= c1[:, None, None] * U * mag), n
        wdx, wdg = lay.rms_norm_grad(_val(n_["dnorm"]), _val(n_["total"]), gv, _val(n_["rstd"]))
        mean = np.abs(_val(n_["dnorm"]) * gv).mean(1, keepdims=True) * 8
        _close(n_["dx"], wdx + dy, (np.abs(wdx) + np.abs(dy) + rv[:, None] * mean * (1 + np.abs(total))) * (H + 12) * 2.0 ** -24)
        assert np.all(np.abs(_val(n_["dgain"]) - wdg) <= (T + 3) * 2.0 ** -24 * (np.abs(_val(n_["dnorm"]) * _val(n_["total"])) * rv[:, None]).sum(0) * 1.001)
        # the step
        host = {n: b.to_numpy() for n, b in {**grads, "gain": n_["dgain"]}.items()}
        opt.launch({**grads, "gain": n_["dgain"]}, si)
        gpu.stream_sync(si)
        for i, n in enumerate(params):
            refs[n].step(host[n], 1e-3, 0.9, 0.95, 1e-8, 0.0 if n == "gain" else 0.01, step, 3 + 1000003 * step + i)
            st = opt.st[n]
            assert max_ulp(st["p32"].to_numpy(), refs[n].p) == 0 and bits_equal(st["m"].to_numpy(), refs[n].m) and bits_equal(st["v"].to_numpy(), refs[n].v), n
        for b in up.values():
            b.free()
    for b in (opt, ws, *dws, *n_.values(), *grads.values()):
        b.free()
    if E:
        plan.free()
    gpu.api.anc_stream_destroy(si)
