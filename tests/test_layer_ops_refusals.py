"""Calls of the norm, the gated feed-forward block and AdamW with 8-bit moments that would read or write beside their buffers or answer
wrongly are refused before a launch, by the C entries and by the Python ones."""
import ctypes

import numpy as np
import pytest

from test_token_ops_refusals import P, _but, _refused

U16, F32 = np.uint16, np.float32


def _buf(shape, dtype):
    from ancora_cutile_amd import DevBuf
    return DevBuf(shape=shape, dtype=dtype)


def _lib():
    from ancora_cutile_amd import _lib
    return _lib.load()


def test_norm_entry():
    lib, a = _lib(), [P * (16 + i) for i in range(10)]
    T, H, n = 100, 64, 6400
    # x, x_type, residual, stream_type, gain, gain_type, T, H, eps, y, y_type, scale, total, rstd, stream
    ok = (a[0], 1, a[1], 0, a[2], 0, T, H, 1e-6, a[3], 1, 0, a[4], a[5], 0)
    for at, value, word in ((1, 2, "types"), (3, 5, "types"), (5, -1, "types"), (10, 3, "types"), (7, 60, "multiple of 8"), (7, 0, "multiple of 8"),
                            (7, 16392, "multiple of 8"), (6, -1, "rows"), (6, 1 << 31, "rows"), (0, 0, "null"), (4, 0, "null"), (9, 0, "null"), (11, a[6], "null"),
                            (12, 0, "null"), (2, 0, "null"), (0, a[0] + 8, "misaligned"), (2, a[1] + 4, "misaligned"), (9, a[3] + 2, "misaligned"),
                            (13, a[5] + 2, "misaligned")):
        _refused(lib, "anc_rms_norm", _but(ok, at, value), word)
    mx = _but(_but(ok, 10, 2), 11, a[6])
    _refused(lib, "anc_rms_norm", _but(mx, 11, 0), "null")
    _refused(lib, "anc_rms_norm", _but(mx, 7, 72), "multiple of 32")
    for at, other in ((9, a[0] + 16), (9, a[0] - 2 * n + 16), (9, a[1]), (9, a[1] + 4 * n - 16), (12, a[0]), (12, a[1] + 16), (13, a[2] + 252), (13, a[3] + 2 * n - 4),
                      (9, a[4] + 16), (9, a[2]), (4, a[3])):
        _refused(lib, "anc_rms_norm", _but(ok, at, other), "overlap")
    for at, other in ((9, a[0]), (11, a[0] + 2 * n - 4), (11, a[3] + n - 4)):           # 8-bit rows on top of the input
        _refused(lib, "anc_rms_norm", _but(mx, at, other), "overlap")
    assert lib.anc_rms_norm(*_but(ok, 6, 0)) == 0                                       # no rows: nothing to do
    for rows, width in ((1 << 28, 8), (1 << 26, 264), (1 << 24, 2056)):                  # more lanes than one launch has
        _refused(lib, "anc_rms_norm", _but(_but(ok, 6, rows), 7, width), "too large")


def test_a_workspace_for_many_rows_serves_fewer():
    lib = _lib()
    for H in (64, 512, 4096):
        sizes = [lib.anc_rms_norm_grad_workspace_bytes(T, H) for T in (0, 1, 7, 100, 1000, 4095, 4096, 4097, 8191, 8192, 8193, 8194, 65536, 65537, 1 << 20)]
        assert sizes == sorted(sizes) and sizes[0] == 4 * H


def test_norm_gradient_entry():
    lib, a = _lib(), [P * (16 + i) for i in range(10)]
    T, H, n = 3000, 64, 192000
    ws = lib.anc_rms_norm_grad_workspace_bytes(T, H)
    assert ws > 0 and lib.anc_rms_norm_grad_workspace_bytes(T, 60) == -1 and lib.anc_rms_norm_grad_workspace_bytes(-1, 64) == -1
    # dy, dy_type, x, stream_type, gain, gain_type, rstd, carry, T, H, dx, dgain, accumulate, workspace, bytes, stream
    ok = (a[0], 1, a[1], 1, a[2], 0, a[3], a[4], T, H, a[5], a[6], 0, a[7], ws, 0)
    for at, value, word in ((1, 2, "types"), (3, 7, "types"), (5, 2, "types"), (9, 12, "multiple"), (9, 32768, "multiple"), (8, -5, "rows"), (0, 0, "null"), (2, 0, "null"),
                            (4, 0, "null"), (6, 0, "null"), (10, 0, "null"), (11, 0, "null"), (13, 0, "workspace"), (14, ws - 4, "workspace"),
                            (7, a[4] + 2, "misaligned"), (11, a[6] + 4, "misaligned"), (13, a[7] + 4, "misaligned")):
        _refused(lib, "anc_rms_norm_grad", _but(ok, at, value), word)
    for at, other in ((10, a[0] + 16), (10, a[4] - 2 * n + 16), (11, a[0]), (11, a[3] + 4 * T - 16 - 4 * T % 16), (13, a[1] + 2 * n - 16), (13, a[6]), (11, a[5] + 2 * n - 16), (10, a[2])):
        _refused(lib, "anc_rms_norm_grad", _but(ok, at, other), "overlap")


def test_ffn_entries():
    lib, a = _lib(), [P * (64 + 16 * i) for i in range(14)]
    rows, H, I, E = 1000, 64, 128, 3
    hi, ii, w = rows * H * 2, rows * I * 2, E * H * I * 2
    calls = {
        # x, Wg, Wu, counts, offsets, experts, rows, tokens, H, I, h, gate, up, stream
        "anc_gated_ffn": ((a[0], a[1], a[2], a[3], a[4], E, rows, rows, H, I, a[5], a[6], a[7], 0), (0, 1, 2, 10), (11, 12), (3, 4, 5), (6, 7, 8, 9),
                          ((10, a[0]), (10, a[0] + hi - 16), (11, a[1] + w - 16), (12, a[4]), (11, a[5]), (12, a[6] + ii - 16), (10, a[3] - ii + 16))),
        # h, Wd, counts, offsets, experts, rows, tokens, I, H, residual, y, y_type, stream
        "anc_ffn_down": ((a[0], a[1], a[2], a[3], E, rows, rows, I, H, a[4], a[5], 0, 0), (0, 1, 10), (9,), (2, 3, 4), (5, 6, 7, 8),
                         ((10, a[0]), (10, a[1] + w - 16), (10, a[2]), (10, a[4] + 16), (9, a[5] + 2 * hi - 16))),
        # dy, Wd, gate, up, counts, offsets, experts, rows, tokens, H, I, dgate, dup, h, stream
        "anc_gated_ffn_grad": ((a[0], a[1], a[2], a[3], a[4], a[5], E, rows, rows, H, I, a[6], a[7], a[8], 0), (0, 1, 2, 3, 11, 12), (13,), (4, 5, 6), (7, 8, 9, 10),
                               ((11, a[3]), (12, a[2]), (13, a[2]), (13, a[3]), (11, a[0]), (12, a[1] + w - 16), (11, a[7] + 16), (13, a[6]), (11, a[2] + 16), (13, a[4] - ii + 16))),
        # dgate, dup, Wg, Wu, counts, offsets, experts, rows, tokens, H, I, residual, dx, dx_type, stream
        "anc_gated_ffn_dx": ((a[0], a[1], a[2], a[3], a[4], a[5], E, rows, rows, H, I, a[6], a[7], 1, 0), (0, 1, 2, 3, 12), (11,), (4, 5, 6), (7, 8, 9, 10),
                             ((12, a[0]), (12, a[1] + ii - 16), (12, a[3]), (12, a[5] - hi + 16), (12, a[6] + 16))),
    }
    for name, (ok, needed, optional, (counts, offsets, experts), (nrows, ntok, d1, d2), overlaps) in calls.items():
        for at in needed:
            _refused(lib, name, _but(ok, at, 0), "null")
        for at in needed + optional:
            _refused(lib, name, _but(ok, at, ok[at] + 8), "misaligned")
        for at, value in ((counts, 0), (offsets, 0), (experts, 0), (experts, 513), (experts, -1), (counts, ok[counts] + 2)):
            _refused(lib, name, _but(ok, at, value), "segments")
        for at in (d1, d2):
            for value in (0, 60, -8, (1 << 17) + 8):
                _refused(lib, name, _but(ok, at, value), "%")
        for value in (-1, 1 << 31):
            _refused(lib, name, _but(ok, nrows, value), "rows")
        for at, other in overlaps:
            _refused(lib, name, _but(ok, at, other), "overlap")
        for value in (-1, rows + 1):
            _refused(lib, name, _but(ok, ntok, value), "rows")
        _refused(lib, name, _but(_but(_but(_but(ok, ntok, rows - 1), experts, 0), counts, 0), offsets, 0), "rows")
        assert getattr(lib, name)(*_but(ok, ntok, 0)) == 0
    _refused(lib, "anc_ffn_down", _but(calls["anc_ffn_down"][0], 11, 2), "y_type")
    _refused(lib, "anc_gated_ffn_dx", _but(calls["anc_gated_ffn_dx"][0], 13, 2), "dx_type")


def test_adamw8_entry():
    from ancora_cutile_amd._lib import AdamWHyper
    lib = _lib()
    h = lambda **kw: ctypes.byref(AdamWHyper(**{**dict(form=0, sr=0), **kw}))  # noqa: E731
    ok = (P, 2, 10, h(), 0, 0)
    for at, value, word in ((0, 0, "empty"), (0, P + 4, "empty"), (1, 0, "empty"), (2, 0, "total_blocks"), (2, 1 << 31, "total_blocks"), (3, None, "null"),
                            (3, h(form=2), "form"), (3, h(sr=4), "sr"), (3, h(sr=2), "control block"), (3, h(step_table=P, step_cap=1), "control block"),
                            (3, h(step_table=P + 4, step_cap=1), "step_table"), (3, h(step_table=P), "step_table")):
        _refused(lib, "anc_adamw8_multi", _but(ok, at, value), word)


def test_adamw8_descriptor_and_options(fake_device, tmp_path):
    from ancora_cutile_amd import AdamW, HybridOptimizer, _lib
    with pytest.raises(ValueError, match="state_bits"):
        AdamW({"p": np.zeros(64, F32)}, state_bits=16)
    with pytest.raises(ValueError, match="multiple of 64"):
        AdamW({"p": np.zeros(65, F32)}, state_bits=8)
    p = {"a": np.zeros(64 * 5, F32), "b": np.zeros(64, F32)}
    opt = AdamW(p, state_bits=8, seed=11, grad_dtype=U16, no_decay=("b",))
    opt.launch({n: _buf(x.shape, U16) for n, x in p.items()}, 7)
    (table, n, blocks, _, ctl, si), = fake_device.calls("anc_adamw8_multi")
    assert (n, blocks, ctl, si) == (2, 2, 0, 7) and not fake_device.calls("anc_adamw_multi")
    d = (_lib.AdamW8Desc * 2).from_buffer_copy(fake_device.at(table, 2 * ctypes.sizeof(_lib.AdamW8Desc)))
    s = opt.st["a"]
    assert (d[0].m, d[0].v, d[0].ms, d[0].vs, d[0].p32, d[0].p16, d[0].n) == tuple(s[k].ptr for k in ("m", "v", "ms", "vs", "p32", "p16")) + (320,)
    assert d[0].blk0 == 0 and d[1].blk0 == 1 and d[1].wd == 0.0 and d[1].seed == 1 and d[0].g_dtype == _lib.BF16
    assert s["m"].dtype == np.uint8 and s["ms"].shape == (5,) and s["vs"].ptr == s["ms"].ptr + 8
    with pytest.raises(ValueError, match="aligned"):
        opt.launch({"a": _buf((320,), U16), "b": _lib_at(_buf((128,), U16), 2)}, 7)
    opt.free()
    hybrid = HybridOptimizer({"w_norm": np.zeros(64, F32)}, adamw_kw=dict(state_bits=8))
    assert hybrid.adamw.state_bits == 8
    hybrid.free()


def _lib_at(buf, off):
    from ancora_cutile_amd import DevBuf
    return DevBuf(shape=(64,), dtype=buf.dtype, ptr=buf.ptr + off)


def test_struct_layout(tmp_path):
    """anc_adamw8_desc_t as C has it."""
    import os
    import shutil
    import subprocess
    from ancora_cutile_amd import _lib
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [f for f, _ in _lib.AdamW8Desc._fields_]
    src, exe = tmp_path / "a.c", tmp_path / "a"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "anc_optim.h"\nint main(void) { printf("%zu", sizeof(anc_adamw8_desc_t));'
                   + "".join(f'printf(" %zu", offsetof(anc_adamw8_desc_t, {f}));' for f in names) + "return 0; }")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.AdamW8Desc)] + [getattr(_lib.AdamW8Desc, f).offset for f in names]


def test_norm_arguments(fake_device):
    from ancora_cutile_amd import NormWorkspace, rms_norm, rms_norm_grad
    T, H = 10, 64
    x, g, y, r, u8, sc, rs = _buf((T, H), U16), _buf((H,), F32), _buf((T, H), U16), _buf((T,), F32), _buf((T, H), np.uint8), _buf((T, 2), np.uint8), _buf((T, H), F32)
    bad = [dict(), dict(y=y, fp8=u8, scale=sc), dict(fp8=u8), dict(y=y, scale=sc), dict(y=y, residual=rs), dict(y=y, total=rs), dict(y=y, residual=rs, total=y),
           dict(y=_buf((T - 1, H), U16)), dict(y=_buf((T, H + 8), U16)), dict(y=u8), dict(fp8=y, scale=sc), dict(fp8=u8, scale=_buf((T, 3), np.uint8)),
           dict(y=y, rstd=_buf((T - 1,), F32)), dict(y=y, rstd=_buf((T,), U16)), dict(y=y, residual=_buf((T, H - 8), F32), total=rs)]
    for kw in bad:
        with pytest.raises(ValueError):
            rms_norm(x, g, 0, **kw)
    for a in ((_buf((T * H,), U16), g), (x, _buf((H - 8,), F32)), (_buf((T, H), np.int32), g), (x, _buf((H,), np.int32))):
        with pytest.raises(ValueError):
            rms_norm(a[0], a[1], 0, y=y)
    with pytest.raises(ValueError):
        rms_norm(_buf((T, 40), U16), _buf((40,), F32), 0, fp8=_buf((T, 40), np.uint8), scale=sc)
    assert not fake_device.calls("anc_rms_norm")
    rms_norm(x, g, 3, y=y, residual=rs, total=rs, rstd=r, eps=1e-5)
    rms_norm(x, g, 3, fp8=u8, scale=sc)
    c = fake_device.calls("anc_rms_norm")
    assert c[0] == (x.ptr, 1, rs.ptr, 0, g.ptr, 0, T, H, 1e-5, y.ptr, 1, 0, rs.ptr, r.ptr, 3)
    assert c[1] == (x.ptr, 1, 0, 1, g.ptr, 0, T, H, 1e-6, u8.ptr, 2, sc.ptr, 0, 0, 3)
    ws, dg = NormWorkspace(T, H), _buf((H,), F32)
    with pytest.raises(ValueError):
        NormWorkspace(T, 12)
    ok = dict(dy=x, x=rs, gain=g, rstd=r, si=0, dx=rs, dgain=dg, workspace=ws)
    for kw in (dict(dy=_buf((T * H,), U16)), dict(x=_buf((T - 1, H), F32)), dict(dx=y), dict(carry=y), dict(dgain=_buf((H,), U16)), dict(dgain=_buf((8,), F32)),
               dict(rstd=_buf((3,), F32)), dict(gain=_buf((8,), F32)), dict(dy=_buf((T, H), np.int32))):
        with pytest.raises(ValueError):
            rms_norm_grad(**{**ok, **kw})
    assert not fake_device.calls("anc_rms_norm_grad")
    rms_norm_grad(**ok, carry=rs, accumulate=True)
    assert fake_device.calls("anc_rms_norm_grad")[0] == (x.ptr, 1, rs.ptr, 0, g.ptr, 0, r.ptr, rs.ptr, T, H, rs.ptr, dg.ptr, 1, ws.buf.ptr, ws.buf.nbytes, 0)


def test_ffn_arguments(fake_device):
    from ancora_cutile_amd import RoutePlan, ffn_down, gated_ffn, gated_ffn_dx, gated_ffn_grad
    from ancora_cutile_amd._lib import AncoraError
    T, H, I, E = 12, 64, 40, 4
    plan = RoutePlan(T, 2, E, 8)
    for p, rows, lead in ((None, T, ()), (plan, plan.capacity, (E,))):
        x, h, y, f = _buf((rows, H), U16), _buf((rows, I), U16), _buf((rows, H), U16), _buf((rows, H), F32)
        W, Wd, g, u = _buf(lead + (H, I), U16), _buf(lead + (I, H), U16), _buf((rows, I), U16), _buf((rows, I), U16)
        calls = [(gated_ffn, dict(x=x, Wg=W, Wu=W, si=0, h=h, gate=g, up=u, plan=p)), (ffn_down, dict(h=h, Wd=Wd, si=0, y=f, residual=f, plan=p)),
                 (gated_ffn_grad, dict(dy=y, gate=g, up=u, Wd=Wd, si=0, dgate=g, dup=u, h=h, plan=p)),
                 (gated_ffn_dx, dict(dgate=g, dup=u, Wg=W, Wu=W, si=0, dx=y, residual=y, plan=p))]
        if p is not None:
            for call, kw in calls:
                with pytest.raises(AncoraError, match="routed"):
                    call(**kw)
            plan.active = T
        for call, kw in calls:
            name = "anc_" + call.__name__
            before = len(fake_device.calls(name))
            for k, b in kw.items():
                if k in ("si", "plan"):
                    continue
                wrong = [_buf(b.shape[:-1] + (b.shape[-1] + 4,), b.dtype), _buf(b.shape, np.int32), _buf((b.size,), b.dtype)]
                if "W" not in k and not (p is None and b is next(iter(kw.values()))):
                    wrong.append(_buf((b.shape[0] - 1,) + b.shape[1:], b.dtype))
                for w in wrong:
                    with pytest.raises(ValueError):
                        call(**{**kw, k: w})
            assert len(fake_device.calls(name)) == before
            call(**kw)
            assert len(fake_device.calls(name)) == before + 1
        with pytest.raises(ValueError):
            ffn_down(h, Wd, 0, f, residual=y, plan=p)
    c = fake_device.calls("anc_gated_ffn")
    assert c[0][3:10] == (0, 0, 0, T, T, H, I) and c[1][5:10] == (E, plan.capacity, 2 * T, H, I) and c[1][3].value == plan.counts.ptr and c[1][4].value == plan.offsets.ptr
