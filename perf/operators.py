"""Performance cases of the operators that are indexed by token: the input embedding's lookup and gradient, tokens sorted by
expert and back, and the experts' weight gradients.

A case is a dict of plain values; `kind` selects the operator:

    lookup      embed_lookup: rows of the table times a scale
    embed_grad  DeviceIdGroups.group + embed_dw: the batch's ids grouped on the device, then the table's gradient
    dispatch    RoutePlan.route + dispatch: tokens sorted by expert; with `back` also dispatch_grad of the sorted rows' gradient
    combine     combine: the experts' rows back to their tokens, weighted and summed
    combine_grad  combine_grad: gradients of the experts' rows and of the weights
    expert_dw   expert_dW: the weight gradients of the experts' three projections over the sorted tokens

With `own` false the same results come from elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"


def listed():
    return [
        # One decoding step of a few sequences: launch latency is all there is.
        dict(name="lookup_decode", kind="lookup", M=5, V=151936, H=1024, tbl="bf16", out="bf16", ids64=False, scale=1.0, skip=0.0),
        # A training batch of the 152 K vocabulary, scaled by the square root of the width.
        dict(name="lookup_8192", kind="lookup", M=8192, V=151936, H=1024, tbl="bf16", out="bf16", ids64=True, scale=32.0,
             skip=0.02),
        # A large packed batch from fp32 master rows into an fp32 residual stream; a width that is no power of two.
        dict(name="lookup_65536_f32", kind="lookup", M=65536, V=50257, H=760, tbl="f32", out="f32", ids64=False, scale=1.0,
             skip=0.0),
        # A short and ragged micro-batch of a small model, gradient added onto the dense table's.
        dict(name="embed_grad_77", kind="embed_grad", M=77, V=8192, H=512, dy="bf16", dense=True, pad=0.0, skip=0.05, scale=1.0),
        # A training batch of the 152 K vocabulary: one summed row per distinct id, for the row-sparse optimizer.
        dict(name="embed_grad_8192", kind="embed_grad", M=8192, V=151936, H=1024, dy="bf16", dense=False, pad=0.0, skip=0.0,
             scale=32.0),
        # A large padded batch: a third of the positions hold one id.
        dict(name="embed_grad_65536_pad", kind="embed_grad", M=65536, V=50257, H=1000, dy="bf16", dense=False, pad=0.33,
             skip=0.0, scale=1.0),
        # One decoding step of a few sequences through a mixture-of-experts layer.
        dict(name="dispatch_decode", kind="dispatch", T=4, k=2, E=16, H=1024, type="bf16", align=1, mask=0.0, back=False),
        # A training batch, each expert's segment filled up to whole tiles, there and back.
        dict(name="dispatch_8192", kind="dispatch", T=8192, k=2, E=16, H=1024, type="bf16", align=128, mask=0.0, back=True),
        # The way back of the same layer, into an fp32 residual stream.
        dict(name="combine_8192", kind="combine", T=8192, k=2, E=16, H=1024, type="bf16", out="f32", align=128, mask=0.1),
        # Many small experts per token: the largest of the row movers.
        dict(name="combine_grad_16384_k8", kind="combine_grad", T=16384, k=8, E=128, H=640, type="bf16", out="bf16", align=16,
             mask=0.05),
        # The weight gradients of one mixture-of-experts layer at a training batch, skewed as a young router leaves it.
        dict(name="expert_dw_16x1024", kind="expert_dw", T=8192, k=2, E=16, H=1024, Ie=1024, align=1, mask=0.0, g16=True),
        # A small model's last micro-batch: ragged segments of a few tokens, experts that none reached.
        dict(name="expert_dw_small", kind="expert_dw", T=301, k=2, E=8, H=640, Ie=392, align=16, mask=0.2, g16=False),
    ]


# ---------------------------------------------------------------- drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly multiples of 8, now and then an odd width."""
    h = _log(rng, lo, hi)
    return h if rng.random() < 0.25 else max(8, h // 8 * 8)


def _type(rng):
    return "bf16" if rng.random() < 0.7 else "f32"


def draw(rng):
    kind = rng.choice(("lookup", "embed_grad", "embed_grad", "dispatch", "combine", "combine_grad", "expert_dw"))
    if kind == "lookup":
        H = _width(rng, 64, 2048)
        return dict(kind=kind, M=_log(rng, 1, min(65536, 40000000 // H)), V=_log(rng, 1000, 151936), H=H, tbl=_type(rng),
                    out=_type(rng), ids64=rng.random() < 0.5, scale=rng.choice((1.0, round(math.sqrt(H), 3))),
                    skip=rng.choice((0.0, 0.05)))
    if kind == "embed_grad":
        H = _width(rng, 64, 2048)
        V = _log(rng, 1000, 151936)
        return dict(kind=kind, M=_log(rng, 1, min(65536, 40000000 // H)), V=V, H=H, dy=_type(rng),
                    dense=V * H <= 1 << 24 and rng.random() < 0.7, pad=rng.choice((0.0, 0.0, 0.2, 0.9)),
                    skip=rng.choice((0.0, 0.05)), scale=rng.choice((1.0, round(math.sqrt(H), 3))))
    E = _log(rng, 2, 160)
    if kind == "expert_dw":
        H, Ie = 8 * _log(rng, 8, 192), 8 * _log(rng, 8, 192)
        k = rng.randint(1, min(8, E))
        most = min(8192, int(1.0e11 / (6.0 * H * Ie * k)), int(1.5e8 / (k * (H + Ie))))
        E = max(k, min(E, int(6.0e7 / (H * Ie)) + 1))
        return dict(kind=kind, T=_log(rng, 1, max(1, most)), k=k, E=E, H=H, Ie=Ie, align=rng.choice((1, 16, 128)),
                    mask=rng.choice((0.0, 0.1)), g16=rng.random() < 0.5)
    H = _width(rng, 64, 2048)
    k = rng.randint(1, min(8, E))
    c = dict(kind=kind, T=_log(rng, 1, max(1, min(16384, 28000000 // (k * H)))), k=k, E=E, H=H, type=_type(rng),
             align=rng.choice((1, 16, 128)), mask=rng.choice((0.0, 0.0, 0.1)))
    if kind == "dispatch":
        c["back"] = rng.random() < 0.5
    else:
        c["out"] = _type(rng)
    return c


# ---------------------------------------------------------------- inputs
_T = {"bf16": torch.bfloat16, "f32": torch.float32}


def _gen(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    return gen


def _normal(gen, shape, std, kind):
    return (std * torch.randn(shape, generator=gen, device=DEV)).to(_T[kind])


def _capacity(c):
    """Slots that hold every assignment and every segment's padding, whatever the routing."""
    A = c["T"] * c["k"]
    return A + (min(c["E"], A) if c["align"] > 1 else 0) * (c["align"] - 1)


def _token_ids(c, gen):
    """Word frequencies falling with the id; a share of one frequent id, a share that names no row."""
    M, V = c["M"], c["V"]
    ids = (V * torch.rand(M, generator=gen, device=DEV) ** 3).long().clamp(max=V - 1)
    ids = (ids * 7919 + 13) % V                       # frequent words lie anywhere in the table
    u = torch.rand(M, generator=gen, device=DEV)
    ids = torch.where(u < c.get("pad", 0.0), torch.full_like(ids, V // 2), ids)
    return torch.where(u > 1.0 - c["skip"], torch.full_like(ids, -1), ids)


def _routing(c, gen):
    """(expert ids (T, k) int32 with -1 for masked tokens, weights (T, k) fp32): softmax over random logits with a
    preference per expert, the k largest."""
    T, k, E = c["T"], c["k"], c["E"]
    logits = torch.randn((T, E), generator=gen, device=DEV) + torch.linspace(0.7, -0.7, E, device=DEV)
    val, ids = torch.topk(logits, k, dim=1)
    w = torch.exp(val - val[:, :1])
    w = w / w.sum(1, keepdim=True)
    masked = torch.rand(T, generator=gen, device=DEV) < c["mask"]
    ids = torch.where(masked[:, None], torch.full_like(ids, -1), ids)
    return ids.to(torch.int32).contiguous(), w.contiguous()


def _inputs(c, seed):
    """The tensors that a user's program has in hand before the call, from the seed alone."""
    gen, kind = _gen(seed), c["kind"]
    if kind == "lookup":
        ids = _token_ids(c, gen)
        return dict(ids=ids if c["ids64"] else ids.to(torch.int32), table=_normal(gen, (c["V"], c["H"]), 0.02, c["tbl"]))
    if kind == "embed_grad":
        return dict(ids=_token_ids(c, gen).to(torch.int32), dy=_normal(gen, (c["M"], c["H"]), 1e-3, c["dy"]))
    experts, w = _routing(c, gen)
    S, T, H = _capacity(c), c["T"], c["H"]
    d = dict(experts=experts, w=w)
    if kind == "dispatch":
        d["x"] = _normal(gen, (T, H), 1.0, c["type"])
        if c["back"]:
            d["dxs"] = _normal(gen, (S, H), 1e-3, c["type"])
    elif kind == "combine":
        d["ys"] = _normal(gen, (S, H), 1.0, c["type"])
    elif kind == "combine_grad":
        d["ys"] = _normal(gen, (S, H), 1.0, c["type"])
        d["dy"] = _normal(gen, (T, H), 1e-3, c["out"])
    else:
        for n, width, std in (("x", H, 1.0), ("h", c["Ie"], 1.0), ("dg", c["Ie"], 1e-3), ("du", c["Ie"], 1e-3), ("dy", H, 1e-3)):
            d[n] = _normal(gen, (S, width), std, "bf16")
    return d


# ---------------------------------------------------------------- the plain form
def _plain_route(experts, E, align, S):
    """counts, offsets, slot of every assignment (-1: masked), assignment of every slot (-1: padding)."""
    T, k = experts.shape
    flat = experts.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, torch.full_like(flat, E))
    counts = (key[:, None] == torch.arange(E, device=DEV)).sum(0)
    padded = (counts + align - 1) // align * align
    ends, starts = torch.cumsum(padded, 0), torch.cumsum(counts, 0) - counts
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    sorted_key, order = torch.sort(key, stable=True)
    e = sorted_key.clamp(max=E - 1)
    at = offsets[e] + torch.arange(T * k, device=DEV) - starts[e]
    at = torch.where(sorted_key < E, at, torch.full_like(at, -1))
    slot = torch.empty_like(flat)
    slot[order] = at
    src = torch.full((S + 1,), -1, device=DEV, dtype=torch.long)
    src[torch.where(at >= 0, at, torch.full_like(at, S))] = order       # (masked ones all write behind the end)
    return (counts.to(torch.int32), offsets.to(torch.int32), slot.to(torch.int32).view(T, k), src[:S].to(torch.int32))


def _plain_weighted(rows, slot, w, out):
    g = rows[slot.clamp(min=0).long()].float()
    if w is not None:
        g = g * w[:, :, None]
    return torch.where((slot >= 0)[:, :, None], g, torch.zeros_like(g)).sum(1).to(out)


def _plain(c, d):
    kind = c["kind"]
    if kind == "lookup":
        ids = d["ids"].long()
        ok = (ids >= 0) & (ids < c["V"])
        rows = d["table"][torch.where(ok, ids, torch.zeros_like(ids))].float() * c["scale"]
        return torch.where(ok[:, None], rows, torch.zeros_like(rows)).to(_T[c["out"]])
    if kind == "embed_grad":
        M, V, H, ids = c["M"], c["V"], c["H"], d["ids"].long()
        key, order = torch.sort(torch.where((ids >= 0) & (ids < V), ids, torch.full_like(ids, V)), stable=True)
        head = torch.ones_like(key)
        head[1:] = (key[1:] != key[:-1]).long()
        group = torch.cumsum(head, 0) - 1
        n = (head * (key < V)).sum()
        gid = torch.full((M,), -1, device=DEV, dtype=torch.long)
        gid[group] = torch.where(key < V, key, torch.full_like(key, -1))
        dy = d["dy"][order].float() * (key < V)[:, None]
        if c["dense"]:
            d["dE"].zero_()
            d["dE"].index_add_(0, key.clamp(max=V - 1), dy, alpha=c["scale"])
            return dict(n=n.to(torch.int32), gid=gid.to(torch.int32), dE=d["dE"])
        rows = torch.zeros((M, H), device=DEV).index_add_(0, group, dy)
        return dict(n=n.to(torch.int32), gid=gid.to(torch.int32), rows=rows * c["scale"])
    S = _capacity(c)
    if kind == "dispatch":
        counts, offsets, slot, src = _plain_route(d["experts"], c["E"], c["align"], S)
        xs = d["x"][src.clamp(min=0).long() // c["k"]]
        xs = torch.where((src >= 0)[:, None], xs, torch.zeros_like(xs))
        got = dict(counts=counts, offsets=offsets, slot=slot, src=src, xs=xs)
        if c["back"]:
            got["dx"] = _plain_weighted(d["dxs"], slot, None, _T[c["type"]])
        return got
    slot, src = d["slot"], d["src"]
    if kind == "combine":
        return _plain_weighted(d["ys"], slot, d["w"], _T[c["out"]])
    if kind == "combine_grad":
        dy, at = d["dy"].float(), src.clamp(min=0).long()
        dys = dy[at // c["k"]] * d["w"].reshape(-1)[at][:, None]
        dys = torch.where((src >= 0)[:, None], dys, torch.zeros_like(dys)).to(_T[c["type"]])
        dw = (d["ys"][slot.clamp(min=0).long()].float() * dy[:, None]).sum(-1)
        return dict(dys=dys, dw=torch.where(slot >= 0, dw, torch.zeros_like(dw)))
    out = {}
    for n, a, b in (("gate", "x", "dg"), ("up", "x", "du"), ("down", "h", "dy")):
        W = torch.stack([d[a][s:s + m].float().t() @ d[b][s:s + m].float() for s, m in d["segments"]])
        out[n] = W
        if c["g16"]:
            out[n + "16"] = W.to(torch.bfloat16)
    return out


# ---------------------------------------------------------------- the framework's calls
def _buf(t):
    """The library's view of a torch tensor (bf16 as bit patterns); the tensor stays the owner."""
    from ancora_cutile_amd import DevBuf
    kinds = {torch.float32: np.float32, torch.bfloat16: np.uint16, torch.int32: np.int32, torch.int64: np.int64}
    return DevBuf(shape=tuple(t.shape), dtype=kinds[t.dtype], ptr=t.data_ptr())


class _Kept:
    """A plan or groups, freed when the state and every tensor that shows one of its arrays are gone."""

    def __init__(self, owner):
        self.owner = owner

    def __del__(self):
        torch.cuda.synchronize()
        self.owner.free()


class _Shown:
    def __init__(self, buf, kept):
        self.kept = kept            # (a tensor holds what it was made from)
        self.__cuda_array_interface__ = {"shape": buf.shape, "typestr": buf.dtype.str, "data": (buf.ptr, False), "version": 2}


def _tensor(buf, kept, shape):
    return torch.as_tensor(_Shown(buf, kept), device=DEV).view(shape)


class State:
    def __init__(self, case, data):
        self.case, self.data, self.go, self.out, self.kept = case, data, None, None, None


def _ready(c, d, state):
    """Buffers, handles and plans of the framework's calls; `state.go` is one pass."""
    from ancora_cutile_amd import embed, dispatch, grads
    kind, si = c["kind"], torch.cuda.current_stream().cuda_stream
    b = {n: _buf(t) for n, t in d.items() if torch.is_tensor(t)}
    if kind == "lookup":
        out = torch.empty((c["M"], c["H"]), device=DEV, dtype=_T[c["out"]])
        o = _buf(out)
        state.go = lambda: embed.embed_lookup(b["ids"], b["table"], si, o, scale=c["scale"])
        state.out = out
        return
    if kind == "embed_grad":
        groups = embed.DeviceIdGroups(c["M"], c["V"])
        kept = state.kept = _Kept(groups)
        state.out = dict(n=_tensor(groups.count, kept, ()), gid=_tensor(groups.gid, kept, (c["M"],)))
        if c["dense"]:
            state.out["dE"] = d["dE"]

            def go():
                b["dE"].fill_zero(si)
                groups.group(b["ids"], si)
                embed.embed_dw(groups, b["dy"], si, out=b["dE"], scale=c["scale"])
        else:
            state.out["rows"] = torch.zeros((c["M"], c["H"]), device=DEV)
            rows = _buf(state.out["rows"])

            def go():
                groups.group(b["ids"], si)
                embed.embed_dw(groups, b["dy"], si, compact=rows, scale=c["scale"])
        state.go = go
        return
    S, T, k, E, H = _capacity(c), c["T"], c["k"], c["E"], c["H"]
    plan = dispatch.RoutePlan(T, k, E, align=c["align"])
    kept = state.kept = _Kept(plan)
    assert plan.capacity == S
    if kind == "dispatch":
        xs = torch.zeros((S, H), device=DEV, dtype=_T[c["type"]])
        bxs = _buf(xs)
        state.out = dict(counts=_tensor(plan.counts, kept, (E,)), offsets=_tensor(plan.offsets, kept, (E + 1,)),
                         slot=_tensor(plan.slot, kept, (T, k)), src=_tensor(plan.src, kept, (S,)), xs=xs)
        if c["back"]:
            state.out["dx"] = torch.empty((T, H), device=DEV, dtype=_T[c["type"]])
            bdx = _buf(state.out["dx"])

        def go():
            plan.route(b["experts"], si)
            dispatch.dispatch(plan, b["x"], si, bxs)
            if c["back"]:
                dispatch.dispatch_grad(plan, b["dxs"], si, bdx)
        state.go = go
        return
    plan.route(b["experts"], si)
    if kind == "combine":
        state.out = torch.empty((T, H), device=DEV, dtype=_T[c["out"]])
        y = _buf(state.out)
        state.go = lambda: dispatch.combine(plan, b["ys"], b["w"], si, y)
    elif kind == "combine_grad":
        state.out = dict(dys=torch.zeros((S, H), device=DEV, dtype=_T[c["type"]]), dw=torch.empty((T, k), device=DEV))
        dys, dw = _buf(state.out["dys"]), _buf(state.out["dw"])
        state.go = lambda: dispatch.combine_grad(plan, b["dy"], b["ys"], b["w"], si, dys, dw)
    else:
        Ie, problems = c["Ie"], []
        state.out = {}
        for n, x, dy, K, N in (("gate", "x", "dg", H, Ie), ("up", "x", "du", H, Ie), ("down", "h", "dy", Ie, H)):
            state.out[n] = torch.empty((E, K, N), device=DEV)
            p = dict(x=b[x], dy=b[dy], dW=_buf(state.out[n]))
            if c["g16"]:
                state.out[n + "16"] = torch.empty((E, K, N), device=DEV, dtype=torch.bfloat16)
                p["g16"] = _buf(state.out[n + "16"])
            problems.append(p)
        state.go = lambda: grads.expert_dW(plan, problems, si)


def prepare(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "embed_grad" and c["dense"]:
        d["dE"] = torch.zeros((c["V"], c["H"]), device=DEV)
    state = State(c, d)
    if own:
        _ready(c, d, state)
    elif c["kind"] in ("combine", "combine_grad", "expert_dw"):
        counts, offsets, d["slot"], d["src"] = _plain_route(d["experts"], c["E"], c["align"], _capacity(c))
        if c["kind"] == "expert_dw":
            d["segments"] = list(zip(offsets[:-1].tolist(), counts.tolist()))
    return state


def run(state):
    if not own:
        return _plain(state.case, state.data)
    state.go()
    return state.out


# ---------------------------------------------------------------- in 64 bits, on the host's view of the definition
def _exact_route(c, experts):
    """The routing by counting, one assignment after the other, on the host."""
    T, k, E, align, S = c["T"], c["k"], c["E"], c["align"], _capacity(c)
    flat = experts.cpu().numpy().reshape(-1)
    per = [np.flatnonzero(flat == e) for e in range(E)]
    counts = np.array([p.size for p in per], np.int32)
    offsets = np.zeros(E + 1, np.int32)
    slot, src = np.full(T * k, -1, np.int32), np.full(S, -1, np.int32)
    for e, p in enumerate(per):
        offsets[e + 1] = offsets[e] + -(-p.size // align) * align
        slot[p] = offsets[e] + np.arange(p.size)
        src[slot[p]] = p
    return counts, offsets, slot.reshape(T, k), src


def exact(case, seed):
    c, d, kind = case, _inputs(case, seed), case["kind"]
    f64 = torch.float64
    if kind == "lookup":
        out = torch.zeros((c["M"], c["H"]), device=DEV, dtype=f64)
        at = torch.nonzero((d["ids"] >= 0) & (d["ids"] < c["V"])).reshape(-1)
        out[at] = d["table"].index_select(0, d["ids"][at].long()).to(f64) * c["scale"]
        return out
    if kind == "embed_grad":
        ids = d["ids"].cpu().numpy()
        at = np.flatnonzero((ids >= 0) & (ids < c["V"]))
        gid, inverse = np.unique(ids[at], return_inverse=True)
        dy = d["dy"][torch.from_numpy(at).to(DEV)].to(f64)
        rows = torch.zeros((c["M"], c["H"]), device=DEV, dtype=f64)
        rows.index_add_(0, torch.from_numpy(inverse.reshape(-1)).to(DEV), dy)
        rows *= c["scale"]
        padded = np.full(c["M"], -1, np.int32)
        padded[:gid.size] = gid
        out = dict(n=torch.tensor(gid.size, dtype=torch.int32), gid=padded)
        if c["dense"]:
            out["dE"] = torch.zeros((c["V"], c["H"]), device=DEV, dtype=f64)
            out["dE"][torch.from_numpy(gid.astype(np.int64)).to(DEV)] = rows[:gid.size]
        else:
            out["rows"] = rows
        return out
    counts, offsets, slot, src = _exact_route(c, d["experts"])
    T, k, H, S = c["T"], c["k"], c["H"], _capacity(c)
    a = np.flatnonzero(slot.reshape(-1) >= 0)                       # assignments that have a slot
    sl = torch.from_numpy(slot.reshape(-1)[a].astype(np.int64)).to(DEV)
    tok, a = torch.from_numpy(a // k).to(DEV), torch.from_numpy(a).to(DEV)
    if kind == "dispatch":
        xs = torch.zeros((S, H), device=DEV, dtype=f64)
        xs[sl] = d["x"][tok].to(f64)
        out = dict(counts=counts, offsets=offsets, slot=slot, src=src, xs=xs)
        if c["back"]:
            out["dx"] = torch.zeros((T, H), device=DEV, dtype=f64).index_add_(0, tok, d["dxs"][sl].to(f64))
        return out
    w = d["w"].reshape(-1)[a].to(f64)
    if kind == "combine":
        return torch.zeros((T, H), device=DEV, dtype=f64).index_add_(0, tok, d["ys"][sl].to(f64) * w[:, None])
    if kind == "combine_grad":
        dy, dys = d["dy"][tok].to(f64), torch.zeros((S, H), device=DEV, dtype=f64)
        dys[sl] = dy * w[:, None]
        dw = torch.zeros(T * k, device=DEV, dtype=f64)
        dw[a] = (dy * d["ys"][sl].to(f64)).sum(1)
        return dict(dys=dys, dw=dw.view(T, k))
    if 6.0 * T * k * H * c["Ie"] > 2.0e11:
        return None
    out = {}
    for n, x, dy in (("gate", "x", "dg"), ("up", "x", "du"), ("down", "h", "dy")):
        W = torch.zeros((c["E"], d[x].shape[1], d[dy].shape[1]), device=DEV, dtype=f64)
        for e in range(c["E"]):
            rows = slice(int(offsets[e]), int(offsets[e]) + int(counts[e]))
            W[e] = torch.matmul(d[x][rows].to(f64).t().contiguous(), d[dy][rows].to(f64))
        out[n] = W
        if c["g16"]:
            out[n + "16"] = W
    return out


# ---------------------------------------------------------------- work
_SIZE = {"bf16": 2.0, "f32": 4.0}


def _distinct(c):
    """Expected number of distinct ids of a batch."""
    edge = np.linspace(0.0, 1.0, 4097) ** (1.0 / 3.0)
    p, per = np.diff(edge), c["V"] / 4096.0
    return float(np.sum(per * -np.expm1(-c["M"] * (1.0 - c.get("pad", 0.0) - c["skip"]) * p / per)))


def work(case):
    c, kind = case, case["kind"]
    if kind == "lookup":
        n, M = _distinct(c), c["M"]
        return {"bytes": M * (8.0 if c["ids64"] else 4.0) + c["H"] * (n * _SIZE[c["tbl"]] + M * _SIZE[c["out"]]),
                "flops": float(M * c["H"])}
    if kind == "embed_grad":
        n, M, H = _distinct(c), c["M"], c["H"]
        out = 4.0 * c["V"] * H if c["dense"] else 4.0 * n * H
        return {"bytes": 8.0 * M + M * (1.0 - c["skip"]) * H * _SIZE[c["dy"]] + out, "flops": float(M * H)}
    A, T, H, E = c["T"] * c["k"] * (1.0 - c["mask"]), c["T"], c["H"], c["E"]
    pad = min(E, A) * (c["align"] - 1) / 2.0
    if kind == "dispatch":
        s = _SIZE[c["type"]]
        by = 12.0 * T * c["k"] + 8.0 * E + H * s * (T + A + pad)
        if c["back"]:
            by += H * s * (T + A)
        return {"bytes": by, "flops": A * H if c["back"] else 0.0}
    if kind == "combine":
        return {"bytes": 8.0 * T * c["k"] + H * (A * _SIZE[c["type"]] + T * _SIZE[c["out"]]), "flops": 2.0 * A * H}
    if kind == "combine_grad":
        return {"bytes": 12.0 * T * c["k"] + H * ((2.0 * A + pad) * _SIZE[c["type"]] + T * _SIZE[c["out"]]),
                "flops": 3.0 * A * H}
    Ie = c["Ie"]
    return {"bytes": 2.0 * A * (2.0 * H + 3.0 * Ie) + 3.0 * E * H * Ie * (6.0 if c["g16"] else 4.0), "flops": 6.0 * A * H * Ie}
