"""The input embedding from ids on the device: the lookup is the rounded fp32 product bit for bit, the groups are the host's, the
gradient is within the bound of fp32 summation of the sum in 64 bits.

Bound of a sum of c fp32 terms in any order: (c - 1) roundings of at most 2^-24 of the partial sums' magnitude, at most c 2^-24 times the
sum of magnitudes; the scale and the addition onto `out` round once more each."""
import ctypes

import numpy as np
import pytest

from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from oracle.embed_ref import id_groups
from util import bits_equal

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _rows(rng, shape, kind, std=1.0):
    """(host array as uploaded, its values in fp32)."""
    x = (std * rng.standard_normal(shape)).astype(np.float32)
    if kind == "f32":
        return x, x
    b = bf16_rne_bits(x).reshape(shape)
    return b, bits_to_f32(b).reshape(shape)


def _rounded(x, kind):
    return bf16_rne_bits(x).reshape(x.shape) if kind == "bf16" else x


def _groups_want(ids, V):
    """(srt of the valid ids, start, cnt, gid)."""
    at = np.nonzero((ids >= 0) & (ids < V))[0]
    if at.size == 0:
        z = np.zeros(0, np.int32)
        return z, z, z, z
    srt, start, cnt, gid = id_groups(ids[at])
    return at[srt].astype(np.int32), start, cnt, gid


@pytest.mark.parametrize("M,V,H", [(1, 1, 1), (1, 50, 64), (3, 9, 7), (64, 1000, 130), (65, 300, 1000), (257, 5000, 1024), (5, 40, 4099)])
@pytest.mark.parametrize("tbl,out,wide", [("bf16", "bf16", False), ("f32", "bf16", True), ("bf16", "f32", True), ("f32", "f32", False)])
def test_lookup_is_the_rounded_product(gpu, M, V, H, tbl, out, wide):
    from ancora_cutile_amd import DevBuf, embed_lookup
    rng = np.random.default_rng(M + H)
    ids = rng.integers(-1, V + 1, M).astype(np.int64 if wide else np.int32)      # -1 and V name no row
    if wide and M > 2:
        ids[0], ids[1] = (1 << 32) + 0, -(1 << 32)                               # ... nor does what 32 bits would wrap into one
    host, val = _rows(rng, (V, H), tbl)
    val = val.copy()
    if V > 4:
        val[2, 0], val[3, H - 1], val[4, 0] = np.inf, -np.inf, 1e-40             # infinities and denormals go through
        host = _rounded(val, tbl)
        val = bits_to_f32(host).reshape(val.shape) if tbl == "bf16" else val
    scale = 1.0 if H == 64 else 3.3
    gids, gt = DevBuf(ids), DevBuf(host)
    behind = np.full((M + 2, H), 7, np.uint16 if out == "bf16" else np.float32)
    go = DevBuf(behind)
    embed_lookup(gids, gt, 0, go, scale=scale)
    got = go.to_numpy()
    ok = (ids >= 0) & (ids < V)
    want = np.zeros((M, H), np.float32)
    want[ok] = val[ids[ok]] * np.float32(scale)
    assert bits_equal(got[:M], _rounded(want, out)) and bits_equal(got[M:], behind[M:])
    n = M // 2
    go.upload(behind)
    embed_lookup(gids, gt, 0, go, scale=scale, n=n)                              # a prefix; none at all
    assert bits_equal(go.to_numpy()[:n], _rounded(want, out)[:n]) and bits_equal(go.to_numpy()[n:], behind[n:])
    for b in (gids, gt, go):
        b.free()


def test_lookup_keeps_nan_and_takes_unaligned_rows(gpu):
    from ancora_cutile_amd import DevBuf, embed_lookup
    V, H = 6, 16
    t = np.arange(V * H + 1, dtype=np.float32)
    bits = np.zeros(V * H + 1, np.uint16)
    bits[:] = bf16_rne_bits(t)
    bits[1 + 2 * H:1 + 3 * H] = 0xFFFF                                           # NaN in every bit
    gt, gi, go = DevBuf(bits), DevBuf(np.array([2, 0, 5], np.int32)), DevBuf.zeros((3 * H + 2,), np.uint16)
    table = DevBuf(shape=(V, H), dtype=np.uint16, ptr=gt.ptr + 2)                # rows that start at an odd element
    for off in (0, 1):
        out = DevBuf(shape=(3, H), dtype=np.uint16, ptr=go.ptr + 2 * off)
        embed_lookup(gi, table, 0, out)
        got = bits_to_f32(out.to_numpy()).reshape(3, H)
        want = bits_to_f32(bits[1:]).reshape(V, H)
        assert np.all(np.isnan(got[0])) and np.array_equal(got[1:], want[[0, 5]])
    for b in (gt, gi, go):
        b.free()


def test_lookup_and_gradient_of_rows_beyond_32_bit_offsets(gpu):
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_dw, embed_lookup
    V, H = 2_200_000, 1024                                                       # 2.25e9 elements, 9 GB in fp32
    rng = np.random.default_rng(0)
    table = DevBuf.empty((V, H), np.float32)
    ids = np.array([V - 1, 0, V - 2, V - 1, 1 << 21], np.int32)
    vals = {}
    for i in np.unique(ids):
        vals[i] = rng.standard_normal(H).astype(np.float32)
        DevBuf(shape=(H,), dtype=np.float32, ptr=table.ptr + int(i) * H * 4).upload(vals[i])
    gi, out = DevBuf(ids), DevBuf.empty((ids.size, H), np.float32)
    embed_lookup(gi, table, 0, out)
    assert bits_equal(out.to_numpy(), np.stack([vals[i] for i in ids]))
    groups = DeviceIdGroups(ids.size, V)
    groups.group(gi, 0)
    embed_dw(groups, out, 0, out=table, scale=2.0)
    for i in np.unique(ids):
        got = DevBuf(shape=(H,), dtype=np.float32, ptr=table.ptr + int(i) * H * 4).to_numpy()
        n = np.count_nonzero(ids == i)
        assert np.abs(got - vals[i] * (1.0 + 2.0 * n)).max() <= 4 * U * np.abs(vals[i]).max() * (1 + 2 * n)
    for b in (table, gi, out, groups):
        b.free()


BATCHES = [(1, 1), (2, 700), (63, 4), (64, 1), (65, 511), (1000, (1 << 31) - 1), (1024, 512), (1025, 100000), (4097, 20), (8192, 151936),
           (9000, 1), (9000, 2), (9000, 262144), (9000, 262145), (1 << 20, 1000000), (3000, 1 << 30), (65536, 50257), (65537, 151936),
           (16384, 3000), (16385, 151936), (40001, 600), (70001, 1 << 20), (140000, 40)]


@pytest.mark.parametrize("M,V", BATCHES)
def test_groups_are_the_hosts(gpu, M, V):
    from ancora_cutile_amd import DevBuf, DeviceIdGroups
    rng = np.random.default_rng(M)
    groups = DeviceIdGroups(M, V)
    for dist, dtype in (("even", np.int32), ("skewed", np.int64), ("one", np.int32), ("none", np.int64), ("distinct", np.int32)):
        if dist == "even":
            ids = rng.integers(-2, V + 2, M)
        elif dist == "skewed":
            ids = (V * rng.random(M) ** 4).astype(np.int64)
        elif dist == "one":
            ids = np.full(M, V - 1)
        elif dist == "none":
            ids = np.where(np.arange(M) % 2, -1, 1 << 40)
        else:
            ids = (np.arange(M)[::-1] * 3) % (2 * V)
        ids = ids.astype(dtype)
        buf = DevBuf(ids)
        for n in {M, M // 2, 0}:
            groups.group(buf, 0, n)
            srt, start, cnt, gid = _groups_want(ids[:n], V)
            got = [a.to_numpy().reshape(-1) for a in (groups.srt, groups.start, groups.cnt, groups.gid)]
            g = gid.size
            assert groups.count.to_numpy()[0] == g, (dist, n)
            assert np.array_equal(got[0][:srt.size], srt), (dist, n)
            assert np.array_equal(np.sort(got[0][:n]), np.arange(n)), (dist, n)
            assert np.array_equal(got[1][:g], start) and np.array_equal(got[2][:g], cnt) and np.array_equal(got[3][:g], gid), (dist, n)
            assert not got[1][g:].any() and not got[2][g:].any() and np.all(got[3][g:] == -1), (dist, n)
            inner = [a.to_numpy().reshape(-1)[:n] for a in (groups._key, groups._grp)]
            assert np.array_equal(inner[0], np.concatenate([np.repeat(gid, cnt), np.full(n - srt.size, V)])), (dist, n)
            assert np.array_equal(inner[1], np.concatenate([np.repeat(np.arange(g), cnt), np.full(n - srt.size, -1)])), (dist, n)
        buf.free()
    groups.free()


def test_groups_whatever_the_sample_sees(gpu):
    """Several workgroups share the order by a sample of the positions (one of every n / 256, spread by a hash). Here the sampled
    positions hold the table's last id and all others lie below it, or the first id and above: one workgroup's share is
    nearly everything, many times what it holds at once."""
    from ancora_cutile_amd import DevBuf, DeviceIdGroups
    for n, V in ((20000, 5000), (65536, 262144), (8192, 300)):
        rng = np.random.default_rng(n)
        i = np.arange(256, dtype=np.int64)
        at = i * n // 256 + (((i * 2654435761) & 0xFFFFFFFF) >> 8) % (n // 256)
        groups = DeviceIdGroups(n, V)
        for end in (0, V - 1, -1):
            ids = rng.integers(1, V - 1, n).astype(np.int32)
            ids[at] = end
            buf = DevBuf(ids)
            groups.group(buf, 0)
            srt, start, cnt, gid = _groups_want(ids, V)
            got = [a.to_numpy().reshape(-1) for a in (groups.srt, groups.start, groups.cnt, groups.gid)]
            g = gid.size
            assert groups.count.to_numpy()[0] == g and np.array_equal(got[0][:srt.size], srt), (n, end)
            assert np.array_equal(got[1][:g], start) and np.array_equal(got[2][:g], cnt) and np.array_equal(got[3][:g], gid), (n, end)
            assert np.array_equal(groups._grp.to_numpy().reshape(-1)[:srt.size], np.repeat(np.arange(g), cnt)), (n, end)
            buf.free()
        groups.free()


def _dw_check(groups, ids, V, val, got_rows, scale, base=None):
    _, _, cnt, gid = _groups_want(ids, V)
    ref, mag = np.zeros((gid.size, val.shape[1])), np.zeros((gid.size, val.shape[1]))
    ok = (ids >= 0) & (ids < V)
    at = np.searchsorted(gid, ids[ok])
    np.add.at(ref, at, val[ok].astype(np.float64))
    np.add.at(mag, at, np.abs(val[ok]).astype(np.float64))
    ref, mag = ref * np.float64(np.float32(scale)), mag * abs(scale)
    bound = (cnt[:, None] + 2) * U * mag + 2.0 ** -140
    if base is not None:
        ref = ref + base[gid]
        bound = bound + 2 * U * (np.abs(ref) + mag)
    assert np.all(np.abs(got_rows - ref) <= bound), float((np.abs(got_rows - ref) - bound).max())


@pytest.mark.parametrize("M,V,H,kind", [(1, 1, 1, "bf16"), (5, 3, 7, "f32"), (16, 2, 64, "bf16"), (17, 40, 130, "f32"), (33, 1, 1000, "bf16"),
                                        (300, 20, 2050, "bf16"), (1000, 30, 8, "f32"), (3000, 151936, 1024, "bf16"),
                                        (16400, 5, 72, "bf16"), (33000, 3000, 40, "f32"), (70000, 7, 19, "bf16")])
def test_gradient_against_64_bits(gpu, M, V, H, kind):
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_dw
    rng = np.random.default_rng(M + H)
    groups = DeviceIdGroups(M, V)
    host, val = _rows(rng, (M, H), kind)
    gdy = DevBuf(host)
    for dist in ("skewed", "one", "padded"):
        ids = (V * rng.random(M) ** 3).astype(np.int32)
        if dist == "one":
            ids[:] = V // 2
        if dist == "padded":
            ids[rng.random(M) < 0.3] = -1
            ids[rng.random(M) < 0.4] = V - 1
        buf = DevBuf(ids)
        groups.group(buf, 0)
        behind = rng.standard_normal((M, H)).astype(np.float32)
        compact = DevBuf(behind)
        embed_dw(groups, gdy, 0, compact=compact, scale=1.5)
        got = compact.to_numpy()
        g = int(groups.count.to_numpy()[0])
        _dw_check(groups, ids, V, val, got[:g], 1.5)
        assert bits_equal(got[g:], behind[g:])
        compact.upload(behind)
        embed_dw(groups, gdy, 0, compact=compact, scale=1.5)
        assert bits_equal(compact.to_numpy(), got)                               # run to run
        if V <= 4096:
            base = rng.standard_normal((V, H)).astype(np.float32)
            out = DevBuf(base)
            embed_dw(groups, gdy, 0, out=out)
            full = out.to_numpy()
            gid = groups.gid.to_numpy().reshape(-1)[:g]
            _dw_check(groups, ids, V, val, full[gid], 1.0, base)
            rest = np.setdiff1d(np.arange(V), gid)
            assert bits_equal(full[rest], base[rest])
            out.free()
        for b in (buf, compact):
            b.free()
    gdy.free(); groups.free()


def test_gradient_of_a_prefix_of_none_and_of_non_finite_rows(gpu):
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_dw
    M, V, H = 200, 9, 32
    rng = np.random.default_rng(4)
    ids = rng.integers(0, V, M).astype(np.int32)
    host, val = _rows(rng, (M, H), "f32")
    val[ids == 3] = np.nan
    val[np.nonzero(ids == 5)[0][0], 1] = np.inf
    groups, buf, gdy = DeviceIdGroups(M, V), DevBuf(ids), DevBuf(val)
    out = DevBuf.zeros((V, H), np.float32)
    groups.group(buf, 0)
    embed_dw(groups, gdy, 0, out=out)
    got = out.to_numpy()
    assert np.all(np.isnan(got[3])) and np.isposinf(got[5, 1]) and np.count_nonzero(~np.isfinite(got)) == H + 1
    groups.group(buf, 0, 0)
    embed_dw(groups, gdy, 0, out=out)
    assert bits_equal(out.to_numpy(), got)                                       # no ids: nothing moves
    groups.group(buf, 0, 31)
    rows = DevBuf.zeros((31, H), np.float32)
    val[31:] = np.nan                                                            # rows behind the ids are not read
    gdy.upload(val)
    embed_dw(groups, gdy, 0, compact=rows)
    got = rows.to_numpy()[:int(groups.count.to_numpy()[0])]
    gid = _groups_want(ids[:31], V)[3]
    clean = np.isin(gid, (3, 5), invert=True)                                    # (ids 3 and 5 hold NaN and infinity)
    assert np.all(np.isfinite(got[clean])) and np.all(np.isnan(got[gid == 3]))
    keep = np.isin(ids[:31], (3, 5), invert=True)
    _dw_check(groups, ids[:31][keep], V, val[:31][keep], got[clean], 1.0)
    for b in (buf, gdy, out, rows, groups):
        b.free()


@pytest.mark.parametrize("M", [500, 20000])
def test_captured_and_replayed_on_new_ids(gpu, M):
    """Lookup, grouping and gradient in one graph on a created stream, replayed on other ids each time with eager work of another
    object in between: every replay is the eager result, bit for bit."""
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_dw, embed_lookup
    hip = ctypes.CDLL("libamdhip64.so")
    V, H = 3000, 136
    rng = np.random.default_rng(M)
    s = gpu.stream_create()
    table, dy = DevBuf(_rows(rng, (V, H), "bf16")[0]), DevBuf(_rows(rng, (M, H), "bf16")[0])
    ids = DevBuf(np.zeros(M, np.int32))
    mine, other = DeviceIdGroups(M, V), DeviceIdGroups(M, V)
    x = [DevBuf.zeros((M, H), np.uint16) for _ in range(2)]
    rows = [DevBuf.zeros((M, H), np.float32) for _ in range(2)]

    def go(groups, k, si):
        embed_lookup(ids, table, si, x[k], scale=2.0)
        groups.group(ids, si)
        embed_dw(groups, dy, si, compact=rows[k])

    go(mine, 0, s)                                   # (partial rows are allocated by the first call)
    gpu.stream_sync(s)
    graph, graph_exec = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(ctypes.c_void_p(s), 0) == 0
    go(mine, 0, s)
    assert hip.hipStreamEndCapture(ctypes.c_void_p(s), ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, ctypes.c_size_t(0)) == 0
    for r in range(4):
        ids.upload((V * rng.random(M) ** (1 + r)).astype(np.int32))
        for b in rows:
            b.fill_zero(0)
        go(other, 1, 0)
        gpu.stream_sync(0)
        assert hip.hipGraphLaunch(graph_exec, ctypes.c_void_p(s)) == 0
        gpu.stream_sync(s)
        assert bits_equal(x[0].to_numpy(), x[1].to_numpy()) and bits_equal(rows[0].to_numpy(), rows[1].to_numpy()), r
        assert np.array_equal(mine.gid.to_numpy(), other.gid.to_numpy())
    hip.hipGraphExecDestroy(graph_exec)
    hip.hipGraphDestroy(graph)
    for b in (table, dy, ids, mine, other, *x, *rows):
        b.free()
    gpu.api.anc_stream_destroy(s)


def test_arrays_that_hold_anything_touch_no_other_row(gpu):
    """Sorted indices, groups and ids outside the batch and the table (a batch that was never grouped, say): no row outside the
    buffers is read or written."""
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_dw
    M, V, H = 3000, 50, 72
    rng = np.random.default_rng(1)
    groups = DeviceIdGroups(M, V)
    ids, dy = DevBuf(np.zeros(M, np.int32)), DevBuf(np.ones((M, H), np.float32))
    guard = 64
    big = DevBuf(np.full((V + 2 * guard, H), 3.0, np.float32))
    out = DevBuf(shape=(V, H), dtype=np.float32, ptr=big.ptr + guard * H * 4)
    rows = DevBuf(np.full((M + 2 * guard, H), 3.0, np.float32))
    compact = DevBuf(shape=(M, H), dtype=np.float32, ptr=rows.ptr + guard * H * 4)
    groups.group(ids, 0)
    for _ in range(3):
        for a in (groups.srt, groups.start, groups.cnt, groups._key, groups._grp):
            a.upload(rng.integers(-2 ** 31, 2 ** 31 - 1, (M, 1)).astype(np.int32) >> rng.integers(0, 31, (M, 1)).astype(np.int32))
        embed_dw(groups, dy, 0, out=out)
        embed_dw(groups, dy, 0, compact=compact)
    gpu.stream_sync(0)
    for b, n in ((big, V), (rows, M)):
        host = b.to_numpy()
        assert np.all(host[:guard] == 3.0) and np.all(host[guard + n:] == 3.0)
    for b in (groups, ids, dy, big, rows):
        b.free()


def test_two_batches_at_once_on_two_streams(gpu):
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_dw
    M, V, H = 30000, 500, 256
    rng = np.random.default_rng(8)
    streams = [gpu.stream_create(), gpu.stream_create()]
    host, val = _rows(rng, (M, H), "bf16")
    dy, work = DevBuf(host), []
    for s in streams:
        ids = (V * rng.random(M) ** 3).astype(np.int32)
        work.append((s, ids, DevBuf(ids), DeviceIdGroups(M, V), DevBuf.zeros((M, H), np.float32)))
    gpu.api.anc_device_sync()
    for _ in range(3):
        for s, _, buf, groups, rows in work:
            groups.group(buf, s)
            embed_dw(groups, dy, s, compact=rows)
    gpu.api.anc_device_sync()
    for s, ids, buf, groups, rows in work:
        _dw_check(groups, ids, V, val, rows.to_numpy()[:int(groups.count.to_numpy()[0])], 1.0)
        for b in (buf, groups, rows):
            b.free()
        gpu.api.anc_stream_destroy(s)
    dy.free()


def test_device_groups_feed_the_sequential_scatter_and_the_row_sparse_step(gpu):
    """The arrays serve what the host's serve: `embed_dw_scatter` gives the same bits, and a row-sparse step over all M entries (those
    behind the last group name no row) leaves the state of a step over the host's groups."""
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_dw
    from ancora_cutile_amd.embed import IdGroups, RowSparseAdamW, embed_dw_scatter
    M, V, H = 700, 400, 128
    rng = np.random.default_rng(3)
    W0 = (0.02 * rng.standard_normal((V, H))).astype(np.float32)
    opts = [RowSparseAdamW(W0, lr=1e-2, wd=0.1) for _ in range(2)]
    dev, rows = DeviceIdGroups(M, V), [DevBuf.zeros((M, H), np.float32) for _ in range(3)]
    for step in range(3):
        ids = (V * rng.random(M) ** 3).astype(np.int32)
        host, val = _rows(rng, (M, H), "bf16", 1e-2)
        buf, dy, hostg = DevBuf(ids), DevBuf(host), IdGroups(ids)
        dev.group(buf, 0)
        embed_dw_scatter(hostg, dy, 0, compact=rows[0])
        embed_dw_scatter(dev, dy, 0, compact=rows[1])
        g = hostg.n_groups
        assert bits_equal(rows[0].to_numpy()[:g], rows[1].to_numpy()[:g])
        embed_dw(dev, dy, 0, compact=rows[2])
        _dw_check(dev, ids, V, val, rows[2].to_numpy()[:g], 1.0)
        for o in opts:
            o.catch_up(ids, 0)
        opts[0].step(hostg.gid, g, rows[0], 0)
        opts[1].step(dev.gid, dev.M, rows[1], 0)
        for b in (buf, dy, hostg):
            b.free()
    for o in opts:
        o.flush(0)
    for a, b in ((opts[0].p32, opts[1].p32), (opts[0].m, opts[1].m), (opts[0].v, opts[1].v), (opts[0].p16, opts[1].p16)):
        assert bits_equal(a.to_numpy(), b.to_numpy())
    for b in (dev, *rows, *opts):
        b.free()


@pytest.mark.parametrize("M,V,H,kind", [(63, 5, 520, "bf16"), (64, 900, 257, "f32"), (65, 12, 1003, "bf16"), (127, 40, 24, "f32"), (128, 3, 2050, "bf16"),
                                        (129, 3, 520, "bf16")])
def test_gradient_of_few_positions(gpu, M, V, H, kind):
    """Up to 128 positions one workgroup holds all of them, 4 or 8 to a wavefront, and no second kernel joins anything."""
    test_gradient_against_64_bits(gpu, M, V, H, kind)


def test_few_positions_captured_and_replayed(gpu):
    test_captured_and_replayed_on_new_ids(gpu, 100)


def test_row_sparse_training_without_the_host_seeing_an_id(gpu):
    """Group, catch up, look up, gradient, step, all from ids on the device: rows looked up and final state have the bits of a run whose ids
    are known to the host."""
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_dw, embed_lookup
    from ancora_cutile_amd.embed import RowSparseAdamW
    M, V, H = 300, 500, 64
    rng = np.random.default_rng(12)
    W0 = (0.02 * rng.standard_normal((V, H))).astype(np.float32)
    known, opt = (RowSparseAdamW(W0, lr=1e-2, wd=0.1, sr=True, seed=5) for _ in range(2))
    groups, x, rows = DeviceIdGroups(M, V), [DevBuf.zeros((M, H), np.float32) for _ in range(2)], DevBuf.zeros((M, H), np.float32)
    for step, n in enumerate((M, 1, 0, 200, M)):
        ids = np.where(rng.random(M) < 0.1, -1, V * rng.random(M) ** 2).astype(np.int64)
        host, _ = _rows(rng, (M, H), "f32", 1e-2)
        buf, dy = DevBuf(ids), DevBuf(host)
        groups.group(buf, 0, n)
        opt.catch_up(groups, 0)
        if (ids[:n] >= 0).any():
            known.catch_up(ids[:n][ids[:n] >= 0], 0)
        for o, out in ((known, x[0]), (opt, x[1])):
            embed_lookup(buf, o.p32, 0, out, n=n)
        assert bits_equal(x[0].to_numpy(), x[1].to_numpy()), step
        embed_dw(groups, dy, 0, compact=rows)
        g = int(groups.count.to_numpy()[0])
        known.step(groups.gid, g, rows, 0)
        opt.step(groups.gid, groups.M, rows, 0)
        buf.free(); dy.free()
    for o in (known, opt):
        o.flush(0)
    for a, b in ((known.p32, opt.p32), (known.m, opt.m), (known.v, opt.v), (known.p16, opt.p16), (known.last, opt.last)):
        assert bits_equal(a.to_numpy(), b.to_numpy())
    for b in (groups, rows, *x, known, opt):
        b.free()


@pytest.mark.parametrize("sr", [False, True])
def test_the_first_forward_reads_the_rounded_rows(gpu, sr):
    """Nothing was missed before the first step: a lookup of the bf16 weights then gives the initial rows, rounded to nearest, and after a
    step the rows that it did not name still are."""
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_lookup
    from ancora_cutile_amd.embed import RowSparseAdamW
    V, H, M = 300, 192, 77
    rng = np.random.default_rng(21)
    W0 = rng.standard_normal((V, H)).astype(np.float32)
    opt, groups = RowSparseAdamW(W0, lr=1e-2, wd=0.0, sr=sr, seed=3), DeviceIdGroups(M, V)
    ids = rng.integers(0, V, M).astype(np.int32)
    buf, x, rows = DevBuf(ids), DevBuf.zeros((M, H), np.uint16), DevBuf.zeros((M, H), np.float32)
    groups.group(buf, 0)
    opt.catch_up(groups, 0)
    embed_lookup(buf, opt.p16, 0, x)
    want = bf16_rne_bits(W0).reshape(V, H)
    assert bits_equal(x.to_numpy(), want[ids])
    opt.step(groups.gid, groups.M, rows, 0)
    rest = np.setdiff1d(np.arange(V), ids)
    assert bits_equal(opt.p16.to_numpy()[rest], want[rest])
    for b in (opt, groups, buf, x, rows):
        b.free()
