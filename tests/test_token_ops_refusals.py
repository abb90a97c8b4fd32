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
