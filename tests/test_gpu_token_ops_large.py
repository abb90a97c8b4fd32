"""The operators indexed by token on both sides of every line between their kernels: one or four pieces a lane, rows through or past the
caches, runs of 8, 16 and 64 positions at several wavefronts a team, several launches, tiles that follow each other on an XCD, segments that
begin behind 2^31 elements.

Bounds as in the tests of the single operators: a sum of c fp32 terms is off by at most c 2^-24 of the sum of magnitudes in any order, and
every further step rounds once more; what is moved or is one rounded product has to have the bits."""
import numpy as np
import pytest

from oracle import route_ref as ref
from oracle.bf16_ref import bf16_rne_bits, bits_to_f32
from test_gpu_embed_rows import _groups_want, _rounded, _rows
from util import bits_equal

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
MIB64 = 64 << 20
SIZE = {"bf16": 2, "f32": 4}


def _at(buf, row, H, kind=np.uint16, rows=1):
    from ancora_cutile_amd import DevBuf
    return DevBuf(shape=(rows, H), dtype=kind, ptr=buf.ptr + row * H * np.dtype(kind).itemsize)


# (n, H, table, out, four pieces a lane, past the caches)
LOOKUPS = [(16131, 520, "bf16", "bf16", False, False), (16132, 520, "bf16", "bf16", True, False), (16384, 512, "bf16", "bf16", True, False),
           (16385, 517, "bf16", "bf16", True, False), (32768, 1024, "bf16", "bf16", True, False), (32769, 1024, "bf16", "bf16", True, True),
           (65537, 520, "bf16", "bf16", True, True), (65537, 517, "bf16", "bf16", True, True),
           (16131, 259, "f32", "f32", False, False), (16385, 260, "f32", "f32", True, False), (16385, 259, "f32", "f32", True, False),
           (65537, 260, "f32", "f32", True, True), (65537, 259, "f32", "f32", True, True),
           (16385, 259, "bf16", "f32", True, False), (65537, 259, "bf16", "f32", True, True), (65537, 260, "bf16", "f32", True, True),
           (16385, 259, "f32", "bf16", True, False), (131073, 260, "f32", "bf16", True, True), (131073, 259, "f32", "bf16", True, True)]


@pytest.mark.parametrize("n,H,tbl,out,four,past", LOOKUPS)
def test_lookup_is_the_rounded_product(gpu, n, H, tbl, out, four, past):
    from ancora_cutile_amd import DevBuf, embed_lookup
    vec = 8 if (tbl, out) == ("bf16", "bf16") else 4
    assert (n * -(-H // vec) >= 1 << 20) == four and (n * H * SIZE[out] > MIB64) == past
    V, rng = 3001, np.random.default_rng(n + H)
    ids = rng.integers(-1, V + 1, n).astype(np.int32)
    ids[-1], ids[0] = V - 1, 0
    host, val = _rows(rng, (V, H), tbl)
    odd = H % vec != 0                                 # rows that start at any element, where rows of this width do anyway
    gt, gi = DevBuf(np.concatenate([np.zeros(int(odd), host.dtype), host.reshape(-1)])), DevBuf(ids)
    table = DevBuf(shape=(V, H), dtype=host.dtype, ptr=gt.ptr + odd * host.itemsize)
    behind = np.full((n + 2, H), 7, np.uint16 if out == "bf16" else np.float32)
    go = DevBuf(behind)
    embed_lookup(gi, table, 0, go, scale=3.3)
    got = go.to_numpy()
    ok = (ids >= 0) & (ids < V)
    rows = _rounded(val * np.float32(3.3), out)        # (a row's product is the same wherever it goes)
    want = np.where(ok[:, None], rows[np.where(ok, ids, 0)], rows.dtype.type(0))
    assert bits_equal(got[:n], want) and bits_equal(got[n:], behind[n:])
    for b in (gt, gi, go):
        b.free()


def test_rows_that_take_several_launches(gpu):
    """2^31 pieces and more: lookup, dispatch and combine go on with a second launch."""
    from ancora_cutile_amd import DevBuf, RoutePlan, combine, embed_lookup
    from ancora_cutile_amd.dispatch import dispatch
    H, n = 1 << 20, 16390                              # 131072 pieces a row: 16383 rows a launch; 34 GB
    marks = (0, 16382, 16383, 16384, n - 1)
    value = lambda i: np.full((1, H), 0x3F80 + i, np.uint16)                        # noqa: E731
    table = DevBuf(np.concatenate([value(i) for i in range(4)]))
    ids = np.full(n, -1, np.int32)
    ids[list(marks)] = (1, 2, 3, 1, 2)
    gi, out, xs = DevBuf(ids), DevBuf.empty((n, H), np.uint16), DevBuf.empty((n, H), np.uint16)
    embed_lookup(gi, table, 0, out)
    for t in marks:
        assert np.all(_at(out, t, H).to_numpy() == 0x3F80 + ids[t]), t
    assert not _at(out, 16381, H).to_numpy().any() and not _at(out, n - 2, H).to_numpy().any()
    # every token to its own place from behind: the last expert gets the first tokens
    experts = ((n - 1 - np.arange(n)) * 4 // n).astype(np.int32).reshape(n, 1)
    plan, ge = RoutePlan(n, 1, 4), DevBuf(experts)
    plan.route(ge, 0)
    slot = ref.route(experts, 4, 1)[2].reshape(-1)
    dispatch(plan, out, 0, xs)
    for t in marks:
        assert np.all(_at(xs, slot[t], H).to_numpy() == 0x3F80 + ids[t]), t
        _at(out, t, H).upload(value(9))
    combine(plan, xs, None, 0, out)
    for t in marks:
        assert np.all(_at(out, t, H).to_numpy() == 0x3F80 + ids[t]), t
    assert not _at(out, n - 2, H).to_numpy().any()
    for b in (table, gi, out, xs, plan, ge):
        b.free()


# (M, V, H, type of dy, positions of a run, past the caches)
GRADIENTS = [(8192, 300, 4095, "bf16", 8, False), (8192, 300, 4097, "bf16", 8, True), (8193, 300, 4099, "bf16", 16, True),
             (32768, 700, 1023, "bf16", 16, False), (32700, 5000, 516, "f32", 16, True), (32769, 700, 1024, "bf16", 64, True),
             (33000, 700, 1025, "bf16", 64, True), (33000, 64, 508, "f32", 64, False), (33000, 64, 509, "f32", 64, True),
             (40001, 151936, 1024, "bf16", 64, True)]


@pytest.mark.parametrize("M,V,H,kind,run,past", GRADIENTS)
def test_gradient_against_64_bits(gpu, M, V, H, kind, run, past):
    from ancora_cutile_amd import DevBuf, DeviceIdGroups, embed_dw
    assert (M * H * SIZE[kind] > MIB64) == past and (8 if M <= 8192 else 16 if M <= 32768 else 64) == run
    rng = np.random.default_rng(M + H)
    host, val = _rows(rng, (M, H), kind)
    ids = (V * rng.random(M) ** 2).astype(np.int32)
    ids[rng.random(M) < 0.05] = -1
    ids[rng.random(M) < 0.3] = V - 1                   # a third of the batch on one id
    groups, buf, dy = DeviceIdGroups(M, V), DevBuf(ids), DevBuf(host)
    groups.group(buf, 0)
    srt, start, cnt, gid = _groups_want(ids, V)
    sums = np.add.reduceat(val[srt].astype(np.float64), start, axis=0)
    mag = np.add.reduceat(np.abs(val[srt]).astype(np.float64), start, axis=0)
    g = gid.size
    scale = 1.5
    behind = np.float32(rng.standard_normal((1, H)))
    compact = DevBuf(np.broadcast_to(behind, (M, H)))
    embed_dw(groups, dy, 0, compact=compact, scale=scale)
    got = compact.to_numpy()
    assert int(groups.count.to_numpy()[0]) == g
    assert np.all(np.abs(got[:g] - scale * sums) <= (cnt[:, None] + 2) * U * scale * mag)
    assert np.array_equal(got[g:], np.broadcast_to(behind, (M - g, H)))
    base = np.float32(rng.standard_normal((1, H)))
    out = DevBuf(np.broadcast_to(base, (V, H)))
    embed_dw(groups, dy, 0, out=out)
    full = out.to_numpy()
    want = sums + base
    assert np.all(np.abs(full[gid] - want) <= (cnt[:, None] + 2) * U * mag + 2 * U * (np.abs(want) + mag))
    rest = np.setdiff1d(np.arange(V), gid)
    assert np.array_equal(full[rest], np.broadcast_to(base, (rest.size, H)))
    for b in (groups, buf, dy, compact, out):
        b.free()


# (T, k, H, type of dy, type of ys, past the caches)
COMBINES = [(8100, 8, 513, "bf16", "bf16", False), (8200, 8, 513, "bf16", "bf16", True), (8200, 8, 520, "bf16", "bf16", True),
            (8200, 8, 513, "f32", "bf16", True), (8200, 8, 516, "f32", "bf16", True), (4200, 8, 501, "bf16", "f32", True),
            (4200, 8, 501, "f32", "f32", True), (11000, 3, 512, "f32", "f32", True)]


@pytest.mark.parametrize("T,k,H,dy_kind,kind,past", COMBINES)
def test_gradients_of_combine(gpu, T, k, H, dy_kind, kind, past):
    from ancora_cutile_amd import DevBuf, RoutePlan, combine_grad
    assert (T * k * H * SIZE[kind] > MIB64) == past
    rng, E = np.random.default_rng(T + H), 24
    experts = rng.integers(0, E, (T, k))
    experts[rng.random(T) < 0.05] = -1
    plan, ge = RoutePlan(T, k, E, 16), DevBuf(experts.astype(np.int32))
    plan.route(ge, 0)
    _, offsets, slot, src = ref.route(experts, E, 16)
    S, end = plan.capacity, int(offsets[-1])
    dy, dv = _rows(rng, (T, H), dy_kind)
    ys, yv = _rows(rng, (S, H), kind)
    w = rng.random((T, k)).astype(np.float32)
    gdy, gys, gw = DevBuf(dy), DevBuf(ys), DevBuf(w)
    dys, dw = DevBuf(np.full((S, H), 7, ys.dtype)), DevBuf(np.full((T, k), 9.0, np.float32))
    combine_grad(plan, gdy, gys, gw, 0, dys, dw)
    got, got_dw = dys.to_numpy(), dw.to_numpy()
    assert np.all(got[end:] == 7) and not got[np.nonzero(src < 0)[0]].any()
    for j in range(k):
        at = slot[:, j] >= 0
        s = slot[at, j]
        assert bits_equal(got[s], _rounded(w[at, j, None] * dv[at], kind)), j
        prod = dv[at].astype(np.float64) * yv[s]
        assert np.all(np.abs(got_dw[at, j] - prod.sum(1)) <= (H + 1) * U * np.abs(prod).sum(1)), j
        assert not got_dw[~at, j].any()
    for b in (plan, ge, gdy, gys, gw, dys, dw):
        b.free()


# rows of each expert, and how many 256x256 (128x256) tiles follow each other on one XCD
@pytest.mark.parametrize("E,K,N,rows,tiles", [(16, 1032, 1032, 280, 256), (8, 1032, 1032, 290, 256), (16, 1032, 520, 100, 128), (4, 1288, 1032, 300, 256)])
def test_experts_gradients_of_a_layer(gpu, E, K, N, rows, tiles):
    """Three weights at once over ragged segments, one of them empty, in the order that evens out the XCDs."""
    from ancora_cutile_amd import DevBuf, RoutePlan, expert_dW
    rng = np.random.default_rng(E + K)
    counts = rng.multinomial(E * rows, rng.dirichlet(np.full(E, 6.0)))
    counts[E // 2] = 0
    counts[E // 2 - 1] += E * rows - counts.sum()
    experts = rng.permutation(np.repeat(np.arange(E), counts)).astype(np.int32).reshape(-1, 1)
    plan, ge = RoutePlan(experts.size, 1, E, 16), DevBuf(experts)
    plan.route(ge, 0)
    c, o, _, _ = ref.route(experts, E, 16)
    S = plan.capacity
    wide = 3 * -(-K // 256) * -(-N // 256) * E
    assert (256 if wide >= 256 and S >= 256 * E else 128) == tiles
    x, a, b = (_rows(rng, (S, n), "bf16") for n in (K, N, N))
    gx, ga, gb = (DevBuf(t[0]) for t in (x, a, b))
    outs = [DevBuf(np.full((E, K, N), np.nan, np.float32)) for _ in range(2)]
    onto = rng.standard_normal((E, 1, N)).astype(np.float32)
    outs.append(DevBuf(np.broadcast_to(onto, (E, K, N))))
    g16 = DevBuf.zeros((E, K, N), np.uint16)
    expert_dW(plan, [dict(x=gx, dy=ga, dW=outs[0], g16=g16), dict(x=gx, dy=gb, dW=outs[1]), dict(x=gx, dy=gb, dW=outs[2], accumulate=True)], 0)
    got = [w.to_numpy() for w in outs]
    for i, (dv, base) in enumerate(((a[1], 0.0), (b[1], 0.0), (b[1], onto))):
        want, mag = ref.expert_dw(c, o, x[1], dv), ref.expert_dw(c, o, np.abs(x[1]), np.abs(dv))
        bound = c[:, None, None] * 2.0 ** -23 * mag
        want = want + base
        if i == 2:
            bound = bound + U * (np.abs(want) + bound)
        assert np.all(np.abs(got[i] - want) <= bound), i
    assert not got[0][c == 0].any() and np.array_equal(got[2][c == 0], np.broadcast_to(onto, (E, K, N))[c == 0])
    assert bits_equal(g16.to_numpy(), bf16_rne_bits(got[0]).reshape(got[0].shape))
    for t in (plan, ge, gx, ga, gb, g16, *outs):
        t.free()


def test_a_segment_that_begins_behind_2_to_the_31_elements(gpu):
    """Expert 1's segment, and the filling before it, lie behind 2^31 elements of expert 0's: rows there and back, their gradients
    and the weights' by 64-bit offsets."""
    from ancora_cutile_amd import DevBuf, RoutePlan, combine, combine_grad, expert_dW
    from ancora_cutile_amd.dispatch import dispatch
    T, H, first = 34000, 65536, 33000
    experts = (np.arange(T) >= first).astype(np.int32).reshape(T, 1)
    plan, ge = RoutePlan(T, 1, 2, 256), DevBuf(experts)
    plan.route(ge, 0)
    S, start = plan.capacity, -(-first // 256) * 256
    assert start * H > 1 << 31 and plan.offsets.to_numpy()[1] == start
    x, xs, y, dys = (DevBuf.empty((n, H), np.uint16) for n in (T, S, T, S))
    for b in (x, y):
        b.fill_zero(0)
    marks = {0: 1, first - 1: 2, first: 3, T - 1: 4}                                 # token: value, in all its elements
    bits = lambda v: bf16_rne_bits(np.full(H, v, np.float32)).reshape(1, H)          # noqa: E731
    for t, v in marks.items():
        _at(x, t, H).upload(bits(v))
    place = {t: t if t < first else start + t - first for t in marks}
    fill = _at(xs, first, H, rows=start - first)
    junk = np.full(fill.shape, 0x4040, np.uint16)
    fill.upload(junk)
    _at(dys, first, H, rows=start - first).upload(junk)
    dispatch(plan, x, 0, xs)
    assert not fill.to_numpy().any()
    w, dw = DevBuf(np.full((T, 1), 0.5, np.float32)), DevBuf.zeros((T, 1), np.float32)
    combine(plan, xs, w, 0, y)
    combine_grad(plan, x, xs, w, 0, dys, dw)
    assert not _at(dys, first, H, rows=start - first).to_numpy().any()
    got = dw.to_numpy()
    for t, v in marks.items():
        assert np.array_equal(_at(xs, place[t], H).to_numpy(), bits(v)), t
        assert np.array_equal(_at(y, t, H).to_numpy(), bits(0.5 * v)), t
        assert np.array_equal(_at(dys, place[t], H).to_numpy(), bits(0.5 * v)), t
        assert got[t, 0] == H * v * v, t                                             # whole numbers below 2^24
    assert np.count_nonzero(got) == len(marks)
    # the weights' gradient, contracted with a small gradient that is zero except at the marks (and NaN where no token is)
    small = np.zeros((S, 8), np.uint16)
    small[first:start] = small[start + T - first:] = 0x7FFF
    for t, v in marks.items():
        small[place[t]] = bf16_rne_bits(np.full(8, 1.0 + v, np.float32))
    dy, dW = DevBuf(small), DevBuf.empty((2, H, 8), np.float32)
    expert_dW(plan, [dict(x=xs, dy=dy, dW=dW)], 0)
    for e, want in ((0, 1 * 2 + 2 * 3), (1, 3 * 4 + 4 * 5)):
        assert np.all(dW.to_numpy()[e] == want), e
    for b in (plan, ge, x, xs, y, dys, w, dw, dy, dW):
        b.free()
