"""What the operators indexed by token refuse, at the C boundary and in the host layer, without a GPU: no launch is reached."""
import numpy as np
import pytest

P = 1 << 20          # an address that is aligned and never read


@pytest.fixture(scope="module")
def lib():
    from ancora_cutile_amd import _lib
    return _lib.load()


def _refused(lib, name, args, word):
    assert getattr(lib, name)(*args) == 2, (name, args)
    assert word in lib.anc_last_error().decode(), lib.anc_last_error()


def _but(args, at, value):
    return args[:at] + (value,) + args[at + 1:]


def test_lookup_refusals(lib):
    ok = (P, 4, 10, P, 1, 100, 64, 1.0, P, 1, 0)
    for at, value, word in ((0, 0, "null"), (0, P + 2, "misaligned"), (1, 2, "bytes"), (2, -1, "n="), (2, 1 << 31, "n="), (3, 0, "null"),
                            (3, P + 1, "misaligned"), (4, 2, "types"), (5, 0, "V="), (6, 0, "H="), (6, (1 << 20) + 1, "H="), (8, 0, "null"),
                            (8, P + 1, "misaligned"), (9, -1, "types")):
        _refused(lib, "anc_embed_lookup", _but(ok, at, value), word)
    _refused(lib, "anc_embed_lookup", _but(_but(ok, 0, P + 4), 1, 8), "misaligned")
    assert lib.anc_embed_lookup(*_but(_but(ok, 2, 0), 0, 0)) == 0                # no ids: nothing to do


def test_group_refusals(lib):
    ws = lib.anc_id_groups_device_workspace_bytes(100000, 5000)
    assert ws > 0 and lib.anc_id_groups_device_workspace_bytes(100, 5000) > 0
    for M, V in ((0, 10), ((1 << 20) + 1, 10), (10, 0), (10, 1 << 31)):
        assert lib.anc_id_groups_device_workspace_bytes(M, V) == -1
    ok = (P, 4, 90000, 100000, 5000, P, P, P, P, P, P, P, P, ws, 0)
    for at, value, word in ((0, 0, "null"), (0, P + 1, "misaligned"), (1, 1, "bytes"), (2, -1, "n="), (2, 100001, "n="), (3, 1 << 21, "M="),
                            (4, 0, "V="), (4, 1 << 31, "V="), (13, 100, "workspace holds")) + \
            tuple((i, 0, "null") for i in range(5, 13)) + tuple((i, P + 2, "misaligned") for i in range(5, 13)) + ((12, P + 8, "misaligned"),):
        _refused(lib, "anc_id_groups_device", _but(ok, at, value), word)


def test_gradient_refusals(lib):
    ws = lib.anc_embed_dw_workspace_bytes(1000, 64)
    assert ws == 32 * 2 * 64 * 4
    # one buffer serves every batch up to its size: chunks are shorter for smaller ones
    assert lib.anc_embed_dw_workspace_bytes(9000, 8) == lib.anc_embed_dw_workspace_bytes(8192, 8)
    for M, H in ((0, 64), ((1 << 20) + 1, 64), (10, 0), (10, (1 << 20) + 1)):
        assert lib.anc_embed_dw_workspace_bytes(M, H) == -1
    ok = (P, P, P, P, P, 1000, P, 1, 64, 1.0, P, 0, 500, P, ws, 0)
    for at, value, word in ((5, -1, "n="), (5, (1 << 20) + 1, "n="), (6, 0, "null"), (6, P + 1, "misaligned"), (7, 7, "type"), (8, 0, "H="),
                            (10, 0, "one of"), (10, P + 2, "misaligned"), (11, P, "one of"), (12, 0, "V="), (12, 1 << 31, "V="), (13, 0, "null"), (13, P + 8, "misaligned"),
                            (14, ws - 1, "workspace holds")) + tuple((i, 0, "null") for i in range(5)):
        _refused(lib, "anc_embed_dw", _but(ok, at, value), word)


def test_route_refusals(lib):
    assert lib.anc_route_capacity(100, 8, 16) == 100 + 8 * 15 and lib.anc_route_capacity(3, 8, 16) == 3 + 3 * 15
    for a in ((0, 8, 1), ((1 << 22) + 1, 8, 1), (10, 0, 1), (10, 513, 1), (10, 8, 0), (10, 8, 3), (10, 8, 512)):
        assert lib.anc_route_capacity(*a) == -1
    A, E = 50000, 60
    ws, cap = lib.anc_route_workspace_bytes(A, E), lib.anc_route_capacity(A, E, 32)
    ok = (P, 4, A, E, 32, P, P, P, P, P, cap, P, ws, 0)
    for at, value, word in ((0, 0, "null"), (0, P + 2, "misaligned"), (1, 3, "bytes"), (2, -1, "assignments"), (3, 0, "experts"), (3, 600, "experts"),
                            (4, 24, "align"), (10, cap - 1, "needed"), (10, 1 << 31, "needed"), (12, ws - 1, "workspace holds")) + \
            tuple((i, 0, "null") for i in (5, 6, 7, 8, 9, 11)) + tuple((i, P + 1, "misaligned") for i in (5, 6, 7, 8, 9, 11)):
        _refused(lib, "anc_route", _but(ok, at, value), word)


def test_row_mover_refusals(lib):
    ok = (P, P, P, 10, 2, 4, 16, P, P, 200, 1, 64, 0)
    for at, value, word in ((0, 0, "slots"), (0, P + 2, "slots"), (1, 0, "segments"), (2, P + 1, "segments"), (3, -1, "tokens"), (4, 0, "choices"),
                            (4, 513, "choices"), (5, 0, "segments"), (5, 513, "segments"), (6, 0, "segments"), (7, 0, "null"), (8, 0, "null"),
                            (8, P + 1, "misaligned"), (9, 0, "room"), (9, 1 << 31, "room"), (10, 5, "type"), (11, 0, "width")):
        _refused(lib, "anc_dispatch", _but(ok, at, value), word)
    ok = (P, P, 10, 2, P, 200, 1, P, 0, 64, 0)
    for at, value, word in ((0, 0, "slots"), (1, P + 2, "misaligned"), (2, -1, "tokens"), (3, 0, "choices"), (4, 0, "null"), (5, 0, "room"), (6, 9, "types"), (7, 0, "null"),
                            (7, P + 2, "misaligned"), (8, 9, "types"), (9, 0, "width")):
        _refused(lib, "anc_combine", _but(ok, at, value), word)
    ok = (P, P, P, P, 10, 2, 4, 16, P, 0, P, P, 200, 1, P, 64, 0)
    for at, value, word in ((0, 0, "slots"), (1, 0, "null"), (2, 0, "segments"), (3, 0, "segments"), (4, -1, "tokens"), (8, 0, "null"), (8, P + 2, "misaligned"),
                            (9, 3, "types"), (10, 0, "null"), (11, P + 1, "misaligned"), (12, 0, "room"), (13, 3, "types"), (14, 0, "null"), (14, P + 2, "misaligned")):
        _refused(lib, "anc_combine_grad", _but(ok, at, value), word)


def _buf(shape, dtype):
    from ancora_cutile_amd import DevBuf
    return DevBuf(shape=shape, dtype=dtype)


def test_embedding_calls_that_do_not_fit_launch_nothing(fake_device):
    from ancora_cutile_amd import DeviceIdGroups, embed_dw, embed_lookup
    from ancora_cutile_amd._lib import AncoraError
    V, H, M = 50, 16, 30
    ids, table, out = _buf((M,), np.int32), _buf((V, H), np.uint16), _buf((M, H), np.float32)
    embed_lookup(ids, table, 0, out)
    assert len(fake_device.calls("anc_embed_lookup")) == 1
    for bad in (lambda: embed_lookup(_buf((M,), np.float32), table, 0, out), lambda: embed_lookup(ids, _buf((V, H), np.int32), 0, out),
                lambda: embed_lookup(ids, _buf((V * H,), np.uint16), 0, out), lambda: embed_lookup(ids, table, 0, _buf((M - 1, H), np.uint16)),
                lambda: embed_lookup(ids, table, 0, _buf((M, H + 1), np.uint16)), lambda: embed_lookup(ids, table, 0, out, n=M + 1),
                lambda: embed_lookup(ids, table, 0, out, n=-1), lambda: embed_lookup(ids, table, 0, _buf((M, H), np.int32))):
        with pytest.raises(ValueError):
            bad()
    assert len(fake_device.calls("anc_embed_lookup")) == 1
    for M_, V_ in ((0, 5), ((1 << 20) + 1, 5), (5, 0), (5, 1 << 31)):
        with pytest.raises(ValueError):
            DeviceIdGroups(M_, V_)
    g = DeviceIdGroups(M, V)
    dy, rows, dE = _buf((M, H), np.uint16), _buf((M, H), np.float32), _buf((V, H), np.float32)
    with pytest.raises(AncoraError):
        embed_dw(g, dy, 0, out=dE)                                    # nothing grouped yet
    for bad in (lambda: g.group(_buf((M + 1,), np.int32), 0), lambda: g.group(_buf((M,), np.uint32), 0), lambda: g.group(ids, 0, M + 1),
                lambda: g.group(ids, 0, -1)):
        with pytest.raises(ValueError):
            bad()
    assert not fake_device.calls("anc_id_groups_device")
    g.group(ids, 0)
    for bad in (lambda: embed_dw(g, dy, 0), lambda: embed_dw(g, dy, 0, out=dE, compact=rows), lambda: embed_dw(g, dy, 0, out=rows),
                lambda: embed_dw(g, _buf((M - 1, H), np.uint16), 0, out=dE), lambda: embed_dw(g, _buf((M, H + 1), np.uint16), 0, out=dE),
                lambda: embed_dw(g, dy, 0, compact=_buf((M - 1, H), np.float32)), lambda: embed_dw(g, dy, 0, compact=_buf((M, H), np.uint16)),
                lambda: embed_dw(g, _buf((M, H), np.int32), 0, out=dE)):
        with pytest.raises(ValueError):
            bad()
    assert not fake_device.calls("anc_embed_dw")
    # partial rows: one buffer for a width, kept while a wider one joins it (a captured graph may hold its address)
    embed_dw(g, dy, 0, out=dE)
    first = fake_device.calls("anc_embed_dw")[-1][13]
    wide = _buf((M, 4 * H), np.uint16)
    embed_dw(g, wide, 0, compact=_buf((M, 4 * H), np.float32))
    assert fake_device.calls("anc_embed_dw")[-1][13] != first and first in fake_device.blocks
    embed_dw(g, dy, 0, out=dE)
    assert fake_device.calls("anc_embed_dw")[-1][13] == first
    # a width that would allocate inside a capture is refused before anything is launched
    fake_device.capturing.add(7)
    before = len(fake_device.calls("anc_embed_dw"))
    with pytest.raises(AncoraError, match="before the stream is captured"):
        embed_dw(g, _buf((M, 9 * H), np.uint16), 7, compact=_buf((M, 9 * H), np.float32))
    assert len(fake_device.calls("anc_embed_dw")) == before
    embed_dw(g, dy, 7, out=dE)
    g.free()
    g.free()
    assert first not in fake_device.blocks
    with pytest.raises(AncoraError):
        g.group(ids, 0)
    with pytest.raises(AncoraError):
        embed_dw(g, dy, 0, out=dE)


def test_routing_calls_that_do_not_fit_launch_nothing(fake_device):
    from ancora_cutile_amd import RoutePlan, combine, combine_grad, dispatch_grad
    from ancora_cutile_amd._lib import AncoraError
    from ancora_cutile_amd.dispatch import dispatch
    T, k, E, H = 20, 2, 4, 24
    for a in ((0, k, E), (T, 0, E), (T, 513, E), (T, k, 0), (T, k, 513), (T, k, E, 0), (T, k, E, 3), (T, k, E, 512), (1 << 22, 2, E)):
        with pytest.raises(ValueError):
            RoutePlan(*a)
    p = RoutePlan(T, k, E, 8)
    S = p.capacity
    x, xs, w = _buf((T, H), np.uint16), _buf((S, H), np.uint16), _buf((T, k), np.float32)
    ids = _buf((T, k), np.int64)
    with pytest.raises(AncoraError):
        dispatch(p, x, 0, xs)
    for bad in (lambda: p.route(_buf((T * k,), np.int32), 0), lambda: p.route(_buf((T, k + 1), np.int32), 0), lambda: p.route(_buf((T, k), np.float32), 0),
                lambda: p.route(_buf((T + 1, k), np.int32), 0), lambda: p.route(ids, 0, T + 1), lambda: p.route(ids, 0, -1)):
        with pytest.raises(ValueError):
            bad()
    assert not fake_device.calls("anc_route")
    p.route(ids, 0)
    f = lambda *sh: _buf(sh, np.float32)                                            # noqa: E731
    for bad in (lambda: dispatch(p, x, 0, f(S, H)), lambda: dispatch(p, x, 0, _buf((S - 1, H), np.uint16)), lambda: dispatch(p, _buf((T - 1, H), np.uint16), 0, xs),
                lambda: dispatch(p, x, 0, _buf((S, H + 1), np.uint16)), lambda: dispatch(p, _buf((T, H), np.int32), 0, _buf((S, H), np.int32)),
                lambda: combine(p, _buf((S - 1, H), np.uint16), w, 0, x), lambda: combine(p, xs, f(T, k + 1), 0, x), lambda: combine(p, xs, f(T - 1, k), 0, x),
                lambda: combine(p, xs, _buf((T, k), np.uint16), 0, x), lambda: combine(p, xs, w, 0, f(T - 1, H)), lambda: dispatch_grad(p, xs, 0, f(T, H + 1)),
                lambda: combine_grad(p, x, xs, w, 0, f(S, H), f(T, k)), lambda: combine_grad(p, x, xs, w, 0, xs, f(T, k + 1)),
                lambda: combine_grad(p, x, xs, w, 0, _buf((S - 1, H), np.uint16), f(T, k)), lambda: combine_grad(p, f(T - 1, H), xs, w, 0, xs, f(T, k))):
        with pytest.raises(ValueError):
            bad()
    assert not any(fake_device.calls(n) for n in ("anc_dispatch", "anc_combine", "anc_combine_grad"))
    dispatch(p, x, 0, xs)
    combine(p, xs, w, 0, f(T, H))
    dispatch_grad(p, xs, 0, x)
    combine_grad(p, x, xs, w, 0, _buf((S, H), np.uint16), f(T, k))
    assert [len(fake_device.calls(n)) for n in ("anc_dispatch", "anc_combine", "anc_combine_grad")] == [1, 2, 1]
    p.free()
    p.free()
    for bad in (lambda: p.route(ids, 0), lambda: dispatch(p, x, 0, xs)):
        with pytest.raises(AncoraError):
            bad()


def test_expert_gradient_refusals(lib):
    import ctypes
    from ancora_cutile_amd._lib import ExpertDwProblem
    fields = dict(x=P, dy=P, dW=P, g16=0, K=64, N=128, accumulate=0, reserved=0)

    def call(n=1, counts=P, offsets=P, order=P, experts=4, capacity=100, **kw):
        arr = (ExpertDwProblem * 9)(*[ExpertDwProblem(**{**fields, **kw}) for _ in range(9)])
        return lib.anc_expert_dw_multi(arr, n, counts, offsets, order, experts, capacity, 0)

    for kw, word in ((dict(n=0), "problems"), (dict(n=9), "problems"), (dict(counts=0), "segments"), (dict(offsets=P + 2), "segments"), (dict(order=0), "segments"),
                     (dict(experts=0), "segments"), (dict(capacity=0), "room"), (dict(experts=513), "segments"), (dict(K=12), "K % 8"), (dict(N=0), "K % 8"),
                     (dict(N=(1 << 17) + 8), "K % 8"), (dict(x=0), "null"), (dict(dy=P + 8), "misaligned"), (dict(dW=P + 4), "misaligned"),
                     (dict(g16=P + 4), "misaligned")):
        assert call(**kw) == 2 and word in lib.anc_last_error().decode(), (kw, lib.anc_last_error())
    assert lib.anc_expert_dw_multi(ctypes.POINTER(ExpertDwProblem)(), 1, P, P, P, 4, 100, 0) == 2


def test_expert_gradient_calls_that_do_not_fit_launch_nothing(fake_device):
    from ancora_cutile_amd import RoutePlan, expert_dW
    from ancora_cutile_amd._lib import AncoraError
    E, K, N = 3, 16, 24
    p = RoutePlan(10, 2, E, 4)
    S = p.capacity
    good = dict(x=_buf((S, K), np.uint16), dy=_buf((S, N), np.uint16), dW=_buf((E, K, N), np.float32))
    with pytest.raises(AncoraError):
        expert_dW(p, [good], 0)
    p.route(_buf((10, 2), np.int32), 0)
    for bad in (dict(x=_buf((S - 1, K), np.uint16)), dict(x=_buf((S, K), np.float32)), dict(dy=_buf((S * N,), np.uint16)),
                dict(dW=_buf((E, K, N), np.uint16)), dict(dW=_buf((E, K, N + 8), np.float32)), dict(dW=_buf((E, N, K), np.float32)),
                dict(g16=_buf((E, K, N), np.float32)), dict(x=_buf((S, 12), np.uint16), dW=_buf((E, 12, N), np.float32))):
        with pytest.raises(ValueError):
            expert_dW(p, [good, {**good, **bad}], 0)
    assert not fake_device.calls("anc_expert_dw_multi")
    expert_dW(p, [dict(good, dW=_buf((E * K, N), np.float32))] * 11, 0)
    assert [a[1] for a in fake_device.calls("anc_expert_dw_multi")] == [8, 3]
    expert_dW(p, [], 0)
    assert len(fake_device.calls("anc_expert_dw_multi")) == 2


def test_outputs_that_overlap_are_refused(lib):
    from ancora_cutile_amd._lib import ExpertDwProblem
    a = [P * (16 + i) for i in range(12)]                                          # far apart
    look = (a[0], 4, 10, a[1], 1, 100, 64, 1.0, a[2], 1, 0)
    for out in (a[1], a[1] + 100 * 128 - 2, a[1] - 10 * 128 + 2, a[0], a[0] + 36):
        _refused(lib, "anc_embed_lookup", _but(look, 8, out), "overlaps")
    ws = lib.anc_embed_dw_workspace_bytes(1000, 64)
    grad = (a[0], a[1], a[2], a[3], a[4], 1000, a[5], 1, 64, 1.0, a[6], 0, 500, a[7], ws, 0)
    for at, value in ((10, a[5]), (10, a[5] + 1000 * 128 - 4), (10, a[7] + ws - 4), (13, a[5]), (13, a[6] + 500 * 256 - 16)):
        _refused(lib, "anc_embed_dw", _but(grad, at, value), "overlap")
    move = (a[0], a[1], a[2], 10, 2, 4, 16, a[3], a[4], 200, 1, 64, 0)
    for x in (a[4], a[4] + 200 * 128 - 2, a[4] - 10 * 128 + 2):
        _refused(lib, "anc_dispatch", _but(move, 7, x), "overlap")
    back = (a[0], a[1], 10, 2, a[2], 200, 1, a[3], 1, 64, 0)
    for y in (a[2], a[2] + 200 * 128 - 2, a[1] - 2, a[1] + 78):
        _refused(lib, "anc_combine", _but(back, 7, y), "overlaps")
    both = (a[0], a[1], a[2], a[3], 10, 2, 4, 16, a[4], 1, a[5], a[6], 200, 1, a[7], 64, 0)
    for at, value in ((11, a[5]), (11, a[4] + 1278), (11, a[1] + 78), (14, a[1]), (14, a[5] + 4), (14, a[4]), (14, a[6])):
        _refused(lib, "anc_combine_grad", _but(both, at, value), "overlaps")
    for name, args in (("anc_dispatch", move), ("anc_combine", back), ("anc_combine_grad", both)):
        at = 2 if name == "anc_combine" else 3 if name == "anc_dispatch" else 4
        _refused(lib, name, _but(_but(args, at, (1 << 21) + 1), at + 1, 2), "tokens")      # more than can be routed

    def call(*problems):
        fields = dict(x=a[0], dy=a[1], dW=a[2], g16=0, K=64, N=128, accumulate=0, reserved=0)
        arr = (ExpertDwProblem * len(problems))(*[ExpertDwProblem(**{**fields, **p}) for p in problems])
        return lib.anc_expert_dw_multi(arr, len(problems), a[8], a[9], a[10], 4, 100, 0)

    weight = 4 * 64 * 128 * 4
    for ps in ((dict(dW=a[0]),), (dict(dW=a[1] + 100 * 256 - 16),), (dict(g16=a[2] + weight - 8),), (dict(g16=a[0]),), (dict(g16=a[1]),), ({}, {}),
               ({}, dict(dW=a[2] + weight - 16)), (dict(g16=a[3]), dict(dW=a[3])), (dict(g16=a[3]), dict(dW=a[4], g16=a[3])), ({}, dict(dW=a[3], x=a[2])),
               (dict(x=a[4]), dict(dW=a[4])), (dict(dy=a[4]), dict(dW=a[3], g16=a[4]))):
        assert call(*ps) == 2 and "overlaps" in lib.anc_last_error().decode(), (ps, lib.anc_last_error())


def test_catch_up_from_groups_on_the_device(fake_device):
    from ancora_cutile_amd import DeviceIdGroups
    from ancora_cutile_amd._lib import AncoraError
    from ancora_cutile_amd.embed import RowSparseAdamW
    opt = RowSparseAdamW(np.zeros((40, 64), np.float32))
    g, other = DeviceIdGroups(30, 40), DeviceIdGroups(30, 41)
    with pytest.raises(AncoraError, match="no ids were grouped"):
        opt.catch_up(g, 0)
    g.group(_buf((30,), np.int32), 0, 20)
    other.group(_buf((30,), np.int32), 0)
    with pytest.raises(ValueError):
        opt.catch_up(other, 0)
    opt.catch_up(g, 0)                                                # no step yet: nothing was missed
    assert not fake_device.calls("anc_adamw_rows")
    opt.t = 3
    opt.catch_up(g, 0)
    (call,) = fake_device.calls("anc_adamw_rows")
    assert call[0] == g.gid.ptr and call[1] == 20 and call[2] == 0
    g.group(_buf((30,), np.int32), 0, 0)
    opt.catch_up(g, 0)
    assert len(fake_device.calls("anc_adamw_rows")) == 1
