"""The operators indexed by token in a run, as a training step uses them: lookup, tokens by expert, the experts' products, the
way back, all gradients, and the optimizers that read them."""
import numpy as np
import pytest

from oracle import route_ref as ref
from oracle.adamw_ref import adamw_step_div, adamw_step_ibc
from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from util import bits_equal, max_ulp

pytestmark = pytest.mark.gpu


def _bits(x):
    return bf16_rne_bits(np.asarray(x, np.float32)).reshape(np.shape(x))


def _val(b):
    return bits_to_f32(b).reshape(b.shape).astype(np.float64)


def test_one_training_step_of_an_embedding_and_an_expert_layer(gpu):
    """Three micro-batches of ragged length. Every result of the device is compared with the 64-bit formula of what the device read;
    bounds are one bf16 rounding (2^-8) of a value, or fp32 sums (terms times 2^-23 of the magnitudes)."""
    from ancora_cutile_amd import (DevBuf, DeviceIdGroups, ExpertOptimizer, RoutePlan, combine, combine_grad, dispatch_grad, embed_dw,
                                   embed_lookup, expert_dW)
    from ancora_cutile_amd.dispatch import dispatch
    from ancora_cutile_amd.embed import RowSparseAdamW
    V, H, Ie, E, k, T, align, scale = 900, 128, 128, 4, 2, 150, 16, 11.25
    rng = np.random.default_rng(12)
    table0 = (0.02 * rng.standard_normal((V, H))).astype(np.float32)
    W0 = {n: (0.05 * rng.standard_normal((E, H, Ie))).astype(np.float32) for n in ("gate_proj", "up_proj", "down_proj")}
    emb = RowSparseAdamW(table0, lr=1e-2, wd=0.0)
    opt = ExpertOptimizer(W0, optimizer="adamw")
    plan, groups = RoutePlan(T, k, E, align), DeviceIdGroups(T, V)
    S = plan.capacity
    u16, f32 = np.uint16, np.float32
    x, xs, y = DevBuf.zeros((T, H), u16), DevBuf.zeros((S, H), u16), DevBuf.zeros((T, H), f32)
    dys, dw, dx, rows = DevBuf.zeros((S, H), u16), DevBuf.zeros((T, k), f32), DevBuf.zeros((T, H), f32), DevBuf.zeros((T, H), f32)
    dW = {n: DevBuf.zeros((E, H, Ie), f32) for n in W0}
    table, m, v = table0.copy(), np.zeros_like(table0), np.zeros_like(table0)
    for step, n in enumerate((T, 97, 1), 1):
        ids = (V * rng.random(n) ** 2).astype(np.int64)
        ids[rng.random(n) < 0.1] = -1
        experts = rng.integers(0, E - 1, (n, k))                      # the last expert gets nothing
        experts[ids < 0] = -1
        w = rng.random((n, k)).astype(f32)
        gids, gex, gw = DevBuf(ids), DevBuf(experts.astype(np.int32)), DevBuf(w)
        emb.catch_up(ids, 0)
        embed_lookup(gids, emb.p32, 0, x, scale=scale)
        xb = x.to_numpy()
        want = np.zeros((n, H), f32)
        want[ids >= 0] = table[ids[ids >= 0]] * f32(scale)
        assert bits_equal(xb[:n], _bits(want))
        plan.route(gex, 0)
        counts, offsets, slot, _ = ref.route(experts, E, align)
        dispatch(plan, x, 0, xs)
        xsv = _val(xs.to_numpy())
        end = int(offsets[-1])
        assert np.array_equal(xsv[:end], ref.dispatch(slot, _val(xb[:n]), np.zeros((end, H))))
        # the experts' products are the caller's: here on the host, rounded to bf16 as its kernels would
        masters = opt.master()
        h, ys = np.zeros((S, Ie)), np.zeros((S, H))
        gate, up = np.zeros((S, Ie)), np.zeros((S, Ie))
        for e in range(E):
            seg = slice(int(offsets[e]), int(offsets[e + 1]))
            gate[seg], up[seg] = xsv[seg] @ masters["gate_proj"][e], xsv[seg] @ masters["up_proj"][e]
            h[seg] = _val(_bits(gate[seg] * up[seg]))
            ys[seg] = _val(_bits(h[seg] @ masters["down_proj"][e]))
        gh, gys = DevBuf(_bits(h)), DevBuf(_bits(ys))
        combine(plan, gys, gw, 0, y)
        mag = ref.combine(slot, np.abs(ys), w)
        assert np.all(np.abs(y.to_numpy()[:n] - ref.combine(slot, ys, w)) <= (k + 1) * 2.0 ** -24 * mag)
        # backwards from a gradient of y
        dy = (0.1 * rng.standard_normal((n, H))).astype(f32)
        gdy = DevBuf(dy)
        combine_grad(plan, gdy, gys, gw, 0, dys, dw)
        want_dys, want_dw = ref.combine_grad(slot, dy, ys, w)
        dysv = _val(dys.to_numpy())
        assert np.all(np.abs(dysv[:end] - want_dys[:end]) <= 2.0 ** -8 * np.abs(want_dys[:end]) + 1e-30)
        _, mag = ref.combine_grad(slot, np.abs(dy), np.abs(ys), w)
        assert np.all(np.abs(dw.to_numpy()[:n] - want_dw) <= (H + 1) * 2.0 ** -24 * mag)
        dgate, dup, dxs = np.zeros((S, Ie)), np.zeros((S, Ie)), np.zeros((S, H))
        for e in range(E):
            seg = slice(int(offsets[e]), int(offsets[e + 1]))
            dh = dysv[seg] @ masters["down_proj"][e].T
            dgate[seg], dup[seg] = dh * up[seg], dh * gate[seg]
            dxs[seg] = dgate[seg] @ masters["gate_proj"][e].T + dup[seg] @ masters["up_proj"][e].T
        gdg, gdu, gdxs = DevBuf(_bits(dgate)), DevBuf(_bits(dup)), DevBuf(_bits(dxs))
        problems = {"gate_proj": (xs, gdg), "up_proj": (xs, gdu), "down_proj": (gh, dys)}
        expert_dW(plan, [dict(x=a, dy=b, dW=dW[name]) for name, (a, b) in problems.items()], 0)
        grads = {}
        for name, (a, b) in problems.items():
            av, bv = _val(a.to_numpy()), _val(b.to_numpy())
            want, mag = ref.expert_dw(counts, offsets, av, bv), ref.expert_dw(counts, offsets, np.abs(av), np.abs(bv))
            grads[name] = dW[name].to_numpy()
            assert np.all(np.abs(grads[name] - want) <= counts[:, None, None] * 2.0 ** -23 * mag), name
        # <dy, y> does not change to first order along (x, W): the gradients belong to the forward
        dispatch_grad(plan, gdxs, 0, dx)
        want_dx = ref.combine(slot, _val(gdxs.to_numpy()))
        mag = ref.combine(slot, np.abs(_val(gdxs.to_numpy())))
        dxv = dx.to_numpy()
        assert np.all(np.abs(dxv[:n] - want_dx) <= k * 2.0 ** -24 * mag)
        groups.group(gids, 0)
        embed_dw(groups, dx, 0, compact=rows, scale=scale)
        # the optimizers read what was produced
        emb.step(groups.gid, n, rows, 0)
        opt.step(dW, 0, lr=1e-2)
        G = np.zeros((V, H), f32)
        got = int(groups.count.to_numpy()[0])
        gid = groups.gid.to_numpy().reshape(-1)[:got]
        assert np.array_equal(gid, np.unique(ids[ids >= 0]))
        G[gid] = rows.to_numpy()[:got]
        exact = np.zeros((V, H))
        np.add.at(exact, ids[ids >= 0], scale * dxv[:n][ids >= 0].astype(np.float64))
        assert np.all(np.abs(G - exact) <= (n + 2) * 2.0 ** -24 * scale * np.abs(dxv[:n]).sum(0) + 1e-30)
        table, m, v = adamw_step_div(table, m, v, G, 1e-2, 0.9, 0.95, 1e-8, 0.0, step)
        for b in (gids, gex, gw, gh, gys, gdy, gdg, gdu, gdxs):
            b.free()
    emb.flush(0)
    assert max_ulp(emb.master(), table) == 0
    after = opt.master()
    assert all(np.isfinite(after[n]).all() and np.abs(after[n][:E - 1] - W0[n][:E - 1]).max() > 0 for n in W0)
    assert all(bits_equal(after[n][E - 1], W0[n][E - 1]) for n in W0)              # no token, no decay: not moved
    for b in (emb, opt, plan, groups, x, xs, y, dys, dw, dx, rows, *dW.values()):
        b.free()


def test_embedding_gradient_against_differences(gpu):
    """sum(lookup * dy) is linear in the table: moving one element by 1/2 each way gives its gradient to the accuracy of fp32."""
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_dw, embed_lookup
    V, H, M, scale = 12, 24, 60, 1.5
    rng = np.random.default_rng(2)
    table, dy = rng.standard_normal((V, H)).astype(np.float32), rng.standard_normal((M, H)).astype(np.float32)
    ids = rng.integers(-1, V, M).astype(np.int32)
    gi, gt, gdy, go, dE = DevBuf(ids), DevBuf(table), DevBuf(dy), DevBuf.zeros((M, H), np.float32), DevBuf.zeros((V, H), np.float32)
    groups = DeviceIdGroups(M, V)
    groups.group(gi, 0)
    embed_dw(groups, gdy, 0, out=dE, scale=scale)
    got = dE.to_numpy()

    def loss(t):
        gt.upload(t)
        embed_lookup(gi, gt, 0, go, scale=scale)
        return go.to_numpy().astype(np.float64) * dy

    for r in range(V):
        up, down = table.copy(), table.copy()
        up[r] += 0.5
        down[r] -= 0.5
        diff = (loss(up) - loss(down)).sum(0) / (up[r].astype(np.float64) - down[r])
        bound = (M + 4) * 2.0 ** -23 * scale * np.abs(dy).sum(0) * (np.abs(table).max() + 1.0)
        assert np.all(np.abs(diff - got[r]) <= bound), r
    for b in (gi, gt, gdy, go, dE, groups):
        b.free()
