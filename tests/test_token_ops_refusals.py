"""Calls of the operators indexed by token that would read or write beside their buffers, answer wrongly or train nothing are refused
before a launch."""
import numpy as np
import pytest


def _buf(shape, dtype):
    from ancora_cutile_amd import DevBuf
    return DevBuf(shape=shape, dtype=dtype)


def test_sequential_scatter_takes_the_rows_its_groups_have_room_for(fake_device):
    """The launch is one workgroup per row of dy: rows beyond the groups' room would take a neighbouring array for theirs, fewer than
    were grouped would drop ids, and a row of the result that is not there would be written."""
    from ancora_cutile_amd import DeviceIdGroups
    from ancora_cutile_amd._lib import AncoraError
    from ancora_cutile_amd.embed import IdGroups, embed_dw_scatter
    M, V, H = 30, 50, 64
    u16, f32 = np.uint16, np.float32
    out, rows = _buf((V, H), f32), _buf((M, H), f32)
    g = DeviceIdGroups(M, V)
    with pytest.raises(AncoraError, match="no ids were grouped"):
        embed_dw_scatter(g, _buf((M, H), u16), 0, out=out)
    g.group(_buf((M,), np.int32), 0, 20)
    host = IdGroups(np.arange(M))
    for groups, dy, to in ((g, _buf((M + 1, H), u16), dict(out=out)), (g, _buf((7 * M, H), u16), dict(compact=_buf((7 * M, H), f32))),
                           (g, _buf((19, H), u16), dict(out=out)), (g, _buf((M, H), u16), dict(compact=_buf((19, H), f32))),
                           (g, _buf((M, H), u16), dict(compact=_buf((M - 1, H), f32))),     # (a replayed `group` may have made more groups)
                           (g, _buf((M, H), u16), dict(out=_buf((V - 1, H), f32))), (g, _buf((M, H), u16), dict(out=_buf((V, 2 * H), f32))),
                           (g, _buf((M, H), u16), dict(compact=_buf((M, H), u16))), (g, _buf((M, H), f32), dict(out=out)),
                           (g, _buf((M, H), u16), {}), (g, _buf((M, H), u16), dict(out=out, compact=rows)),
                           (host, _buf((M + 1, H), u16), dict(out=out)), (host, _buf((5 * M, H), u16), dict(compact=_buf((5 * M, H), f32)))):
        with pytest.raises(ValueError):
            embed_dw_scatter(groups, dy, 0, **to)
    assert not fake_device.calls("anc_embed_dw_scatter")
    for groups in (g, host):
        embed_dw_scatter(groups, _buf((M, H), u16), 0, out=out)
        embed_dw_scatter(groups, _buf((M, H), u16), 0, compact=rows)
    embed_dw_scatter(g, _buf((20, H), u16), 0, compact=_buf((20, H), f32))              # as many rows as were grouped
    embed_dw_scatter(host, _buf((M - 1, H), u16), 0, out=out, V=V)
    calls = fake_device.calls("anc_embed_dw_scatter")
    assert [c[7] for c in calls] == [M, M, M, M, 20, M - 1] and calls[0][0] == g.cnt.ptr and calls[0][2] == g.gid.ptr


def test_a_row_sparse_step_is_not_captured(fake_device):
    """A launch carries the step's number, and replays would carry it again: no row it has stepped would move any more. A catch-up before
    the first step launches nothing, so that its graph would never replay a step."""
    from ancora_cutile_amd import DeviceIdGroups
    from ancora_cutile_amd._lib import AncoraError
    from ancora_cutile_amd.embed import IdGroups, RowSparseAdamW
    V, H, M = 40, 64, 30
    opt, g = RowSparseAdamW(np.zeros((V, H), np.float32)), DeviceIdGroups(M, V)
    host, rows = IdGroups(np.arange(M)), _buf((M, H), np.float32)
    g.group(_buf((M,), np.int32), 0)
    fake_device.capturing = {7}
    calls = (lambda: opt.catch_up(g, 7), lambda: opt.catch_up(np.arange(M), 7), lambda: opt.step(g.gid, M, rows, 7),
             lambda: opt.step(host.gid, M, rows, 7), lambda: opt.step(g.gid, 0, rows, 7), lambda: opt.flush(7))
    for t in (0, 1):
        before = len(fake_device.log)
        for call in calls:
            with pytest.raises(AncoraError, match="captured"):
                call()
        assert opt.t == t and {n for n, _ in fake_device.log[before:]} == {"anc_stream_is_capturing"}
        opt.catch_up(g, 0)                                       # another stream than the captured one
        opt.step(g.gid, M, rows, 0)
    opt.flush(0)
    assert opt.t == 2


P = 1 << 20          # an address that is aligned and never read


def _refused(lib, name, args, word):
    assert getattr(lib, name)(*args) == 2, (name, args)
    assert word in lib.anc_last_error().decode(), lib.anc_last_error()


def _but(args, at, value):
    return args[:at] + (value,) + args[at + 1:]


def test_indices_that_a_call_would_write_over_are_refused():
    """Ids, slots and segments are read by workgroups while others write: an output on top of them would place rows by half-written
    numbers (a routing of ids that change on the way has slots beyond its capacity)."""
    from ancora_cutile_amd import _lib
    lib = _lib.load()
    a = [P * (16 + i) for i in range(16)]                                         # far apart
    n, M, V = 3000, 4000, 500000
    ws = lib.anc_id_groups_device_workspace_bytes(M, V)
    group = (a[0], 8, n, M, V, *a[1:9], ws, 0)
    for at in range(5, 13):
        _refused(lib, "anc_id_groups_device", _but(group, 0, group[at] - 8 * n + 8), "overlap")
        if at != 11:
            _refused(lib, "anc_id_groups_device", _but(group, 0, group[at] + (4 * M if at < 11 else lib.anc_id_groups_device_workspace_bytes(n, V) // 8 * 8) - 8), "overlap")
        for other in range(5, at):
            _refused(lib, "anc_id_groups_device", _but(group, at, group[other]), "overlap")
    T, k, E = 30000, 2, 60
    A = T * k
    ws, cap = lib.anc_route_workspace_bytes(A, E), lib.anc_route_capacity(A, E, 32)
    route = (a[0], 4, A, E, 32, a[1], a[2], a[3], a[4], a[5], cap, a[6], ws, 0)
    for at, nbytes in ((5, 4 * E), (6, 4 * E + 4), (7, 4 * E), (8, 4 * A), (9, 4 * cap), (11, ws)):
        _refused(lib, "anc_route", _but(route, 0, route[at] + nbytes - 4), "overlap")
        _refused(lib, "anc_route", _but(route, 0, route[at] - 4 * A + 4), "overlap")
        for other in (5, 6, 7, 8, 9, 11):
            if other < at:
                _refused(lib, "anc_route", _but(route, at, route[other]), "overlap")
    ws = lib.anc_embed_dw_workspace_bytes(1000, 64)
    grad = (a[0], a[1], a[2], a[3], a[4], 1000, a[5], 1, 64, 1.0, a[6], 0, 500, a[7], ws, 0)
    for at in range(5):
        for value in (a[6] + 500 * 256 - 4, a[6] - 3996, a[7] + ws - 4):
            _refused(lib, "anc_embed_dw", _but(grad, at, value), "overlap")
    move = (a[0], a[1], a[2], 10, 2, 4, 16, a[3], a[4], 200, 1, 64, 0)
    for at, nbytes in ((0, 80), (1, 16), (2, 20)):
        for value in (a[4] - nbytes + 4, a[4] + 200 * 128 - 4):
            _refused(lib, "anc_dispatch", _but(move, at, value), "overlap")
    back = (a[0], a[1], 10, 2, a[2], 200, 1, a[3], 1, 64, 0)
    for value in (a[3] - 76, a[3] + 1276):
        _refused(lib, "anc_combine", _but(back, 0, value), "overlap")
    both = (a[0], a[1], a[2], a[3], 10, 2, 4, 16, a[4], 1, a[5], a[6], 200, 1, a[7], 64, 0)
    for at, nbytes in ((0, 80), (2, 16), (3, 20)):
        for value in (a[6] - nbytes + 4, a[6] + 200 * 128 - 4, a[7] - nbytes + 4, a[7] + 76):
            _refused(lib, "anc_combine_grad", _but(both, at, value), "overlap")
    weight = 4 * 64 * 128
    for g16 in (0, a[3]):
        arr = (_lib.ExpertDwProblem * 1)(_lib.ExpertDwProblem(x=a[0], dy=a[1], dW=a[2], g16=g16, K=64, N=128, accumulate=0, reserved=0))
        for at, nbytes in ((0, 16), (1, 20), (2, 16)):
            for value in (a[2] - nbytes + 4, a[2] + 4 * weight - 4) + ((g16 + 2 * weight - 4,) if g16 else ()):
                segments = _but((a[8], a[9], a[10]), at, value)
                _refused(lib, "anc_expert_dw_multi", (arr, 1, *segments, 4, 100, 0), "overlap")


def test_row_sparse_weights_are_the_tables_from_the_start(fake_device):
    """(not a refusal: the bf16 weights are made when the optimizer is, by one cast over the table)"""
    from ancora_cutile_amd.embed import RowSparseAdamW
    opt = RowSparseAdamW(np.ones((40, 64), np.float32), sr=True)
    assert [c[:5] for c in fake_device.calls("anc_cast_bf16")] == [(opt.p32.ptr, opt.p16.ptr, 40 * 64, 0, 0)]


def test_row_sparse_state_is_in_place_for_every_stream(fake_device):
    """What the constructor fills and casts on the null stream is waited for: a stream that does not wait for that one may read it at once."""
    from ancora_cutile_amd.embed import RowSparseAdamW
    RowSparseAdamW(np.ones((40, 64), np.float32))
    names = [n for n, _ in fake_device.log]
    last = max(i for i, n in enumerate(names) if n in ("anc_cast_bf16", "anc_fill_u32"))
    assert ("anc_stream_sync", (0,)) in fake_device.log[last:]
