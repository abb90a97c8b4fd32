"""Performance cases of the operators of a layer's feed-forward half and its update: the norm in front of it, the gated feed-forward
block, dense and by expert, forwards and backwards, and AdamW with states in 8 bits.

A case is a dict of plain values; `kind` selects the operator:

    norm        rms_norm: the residual's addition, the norm, rows of 32, 16 or 8 bits (MXFP8)
    norm_grad   rms_norm_grad: gradients of the rows and of the gain
    ffn         gated_ffn + ffn_down: h = silu(x Wg) * (x Wu), y = h Wd + residual; over all rows, or by expert (E > 0)
    ffn_grad    gated_ffn_grad + gated_ffn_dx: from dy to the pre-activations' gradients, h and dx
    adamw8      AdamW(state_bits=8): one step over several tensors

With `own` false the same results come from elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # One decoding step of a few sequences: launch latency is all there is.
        dict(name="norm_decode", kind="norm", T=6, H=1024, x="bf16", stream="bf16", add=True, out="bf16", train=False),
        # A training batch in front of an 8-bit product: the residual's addition, the sum kept for the backward pass.
        dict(name="norm_8192_mx8", kind="norm", T=8192, H=1024, x="bf16", stream="bf16", add=True, out="mx8", train=True),
        # The queries' heads of the same batch, each a row of its own.
        dict(name="norm_heads_131072", kind="norm", T=131072, H=128, x="bf16", stream="bf16", add=False, out="bf16", train=True),
        # The backward pass of a training batch, with the gradient that comes along the residual stream.
        dict(name="norm_grad_8192", kind="norm_grad", T=8192, H=1024, dy="bf16", stream="bf16", carry=True),
        # A short, ragged batch of a wider model with a residual stream in 32 bits.
        dict(name="norm_grad_1237_f32", kind="norm_grad", T=1237, H=2056, dy="bf16", stream="f32", carry=True),
        # One decoding step of a few sequences through a dense layer: its weights' bytes.
        dict(name="ffn_decode", kind="ffn", T=5, H=1024, I=2816, E=0, k=1, align=1, mask=0.0, add=True, train=False),
        # A training batch through a dense layer, pre-activations kept.
        dict(name="ffn_8192", kind="ffn", T=8192, H=1024, I=2816, E=0, k=1, align=1, mask=0.0, add=True, train=True),
        # The same batch through a mixture-of-experts layer, segments as uneven as a young router leaves them.
        dict(name="ffn_moe_8192", kind="ffn", T=8192, H=1024, I=1024, E=16, k=2, align=16, mask=0.05, add=False, train=True),
        # Backwards through the dense layer.
        dict(name="ffn_grad_8192", kind="ffn_grad", T=8192, H=1024, I=2816, E=0, k=1, align=1, mask=0.0, add=True),
        # Backwards through a small model's experts: ragged segments, odd widths.
        dict(name="ffn_grad_moe_1500", kind="ffn_grad", T=1500, H=648, I=392, E=8, k=2, align=1, mask=0.1, add=False),
        # The tensors of a small layer that Muon leaves to AdamW: gains and a router.
        dict(name="adamw8_small", kind="adamw8", sizes="1024 1024 128 128 16384 64", grad="f32", sr=False, t=3, wd=0.01),
        # An embedding table and a final gain, bf16 gradients, stochastic weights.
        dict(name="adamw8_embed", kind="adamw8", sizes="51511296 1024", grad="bf16", sr=True, t=200, wd=0.01),
    ]


# ---------------------------------------------------------------- drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _type(rng):
    return "bf16" if rng.random() < 0.7 else "f32"


def draw(rng):
    kind = rng.choice(("norm", "norm", "norm_grad", "ffn", "ffn", "ffn_grad", "ffn_grad", "adamw8"))
    if kind in ("norm", "norm_grad"):
        H = 8 * _log(rng, 4, 1024)
        if kind == "norm_grad":
            return dict(kind=kind, T=_log(rng, 1, max(1, min(65536, 8000000 // H))), H=H, dy=_type(rng), stream=_type(rng),
                        carry=rng.random() < 0.7)
        out = rng.choice(("bf16", "f32", "mx8"))
        H = max(32, H // 32 * 32) if out == "mx8" else H
        x, stream = rng.choice((("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")))
        return dict(kind=kind, T=_log(rng, 1, max(1, min(131072, 8000000 // H))), H=H, x=x, stream=stream,
                    add=rng.random() < 0.7, out=out, train=rng.random() < 0.5)
    if kind == "adamw8":
        n = rng.randint(1, 8)
        return dict(kind=kind, sizes=" ".join(str(64 * _log(rng, 1, 60000)) for _ in range(n)), grad=_type(rng), sr=rng.random() < 0.5,
                    t=_log(rng, 1, 2000), wd=rng.choice((0.0, 0.01, 0.1)))
    H, I = 8 * _log(rng, 8, 320), 8 * _log(rng, 8, 512)
    E = 0 if rng.random() < 0.4 else _log(rng, 2, 128)
    k = rng.randint(1, min(8, E)) if E else 1
    E = max(k, min(E, int(6.0e7 / (H * I)) + 1)) if E else 0
    most = min(8192, int(1.0e11 / (6.0 * H * I * k)), int(4.0e7 / (k * (H + 3 * I))))
    c = dict(kind=kind, T=_log(rng, 1, max(1, most)), H=H, I=I, E=E, k=k, align=rng.choice((1, 16, 128)) if E else 1,
             mask=rng.choice((0.0, 0.1)) if E else 0.0, add=not E and rng.random() < 0.7)
    if kind == "ffn":
        c["train"] = rng.random() < 0.5
    return c


# ---------------------------------------------------------------- inputs
_T = {"bf16": torch.bfloat16, "f32": torch.float32}
LR, B1, B2, AEPS, SEED = 3e-4, 0.9, 0.95, 1e-8, 7


def _gen(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    return gen


def _normal(gen, shape, std, kind):
    return (std * torch.randn(shape, generator=gen, device=DEV)).to(_T[kind])


def _sizes(c):
    return [int(n) for n in c["sizes"].split()]


def _capacity(c):
    """Slots that hold every assignment and every segment's filling, whatever the routing."""
    A = c["T"] * c["k"]
    return A + (min(c["E"], A) if c["align"] > 1 else 0) * (c["align"] - 1)


def _routing(c, gen):
    """Expert of every choice (T, k) int32, -1 for masked tokens: the k largest of random logits with a preference per expert."""
    T, k, E = c["T"], c["k"], c["E"]
    logits = torch.randn((T, E), generator=gen, device=DEV) + torch.linspace(0.7, -0.7, E, device=DEV)
    ids = torch.topk(logits, k, dim=1)[1]
    masked = torch.rand(T, generator=gen, device=DEV) < c["mask"]
    return torch.where(masked[:, None], torch.full_like(ids, -1), ids).to(torch.int32).contiguous()


def _segments(c, experts):
    """First row and number of rows of every expert, as lists on the host."""
    if not c["E"]:
        return [(0, c["T"])]
    counts = (experts.reshape(-1, 1).long() == torch.arange(c["E"], device=DEV)).sum(0).tolist()
    at, out = 0, []
    for n in counts:
        out.append((at, n))
        at += -(-n // c["align"]) * c["align"]
    return out


def _inputs(c, seed):
    """The tensors that a user's program has in hand before the call, from the seed alone."""
    gen, kind = _gen(seed), c["kind"]
    if kind in ("norm", "norm_grad"):
        T, H = c["T"], c["H"]
        scale = torch.exp(0.5 * torch.randn((T, 1), generator=gen, device=DEV))            # rows differ in size
        d = dict(gain=1.0 + 0.1 * torch.randn(H, generator=gen, device=DEV))
        if kind == "norm":
            d["x"] = (scale * torch.randn((T, H), generator=gen, device=DEV)).to(_T[c["x"]])
            if c["add"]:
                d["residual"] = _normal(gen, (T, H), 2.0, c["stream"])
            return d
        d["x"] = (scale * torch.randn((T, H), generator=gen, device=DEV)).to(_T[c["stream"]])
        d["rstd"] = torch.rsqrt(d["x"].double().square().mean(1) + EPS).float()
        d["dy"] = _normal(gen, (T, H), 1e-2, c["dy"])
        if c["carry"]:
            d["carry"] = _normal(gen, (T, H), 1e-2, c["stream"])
        return d
    if kind == "adamw8":
        d = dict(g=[], p32=[], m=[], ms=[], v=[], vs=[])
        for n in _sizes(c):
            d["g"].append(_normal(gen, (n,), 1e-3, c["grad"]))
            d["p32"].append(0.02 * torch.randn(n, generator=gen, device=DEV))
            # moments as earlier steps leave them: 8-bit codes whose blocks' largest lie where the scales put them
            m = 0.3 * torch.randn(n, generator=gen, device=DEV)
            v = (m * (0.5 + torch.rand(n, generator=gen, device=DEV))).square()
            e = torch.randint(-13, -9, (n // 64,), generator=gen, device=DEV)
            d["m"].append((m * 128).clamp(-255, 255).to(torch.float8_e4m3fn))
            d["v"].append((v * 16384 + 1e-4).clamp(max=32000).to(torch.float8_e5m2))
            d["ms"].append((e + 127 - 7).to(torch.uint8))
            d["vs"].append((2 * e + 127 - 14).to(torch.uint8))
        return d
    H, I, n = c["H"], c["I"], max(1, c["E"])
    experts = _routing(c, gen) if c["E"] else None
    S = _capacity(c) if c["E"] else c["T"]
    d = dict(experts=experts, segments=_segments(c, experts))
    for name, shape in (("Wg", (n, H, I)), ("Wu", (n, H, I)), ("Wd", (n, I, H))):
        d[name] = _normal(gen, shape, shape[1] ** -0.5, "bf16")
    if kind == "ffn":
        d["x"] = _normal(gen, (S, H), 1.0, "bf16")
    else:
        d["gate"], d["up"] = _normal(gen, (S, I), 1.0, "bf16"), _normal(gen, (S, I), 1.0, "bf16")
        d["dy"] = _normal(gen, (S, H), 1e-2, "bf16")
    if c["add"]:
        d["residual"] = _normal(gen, (S, H), 1.0 if kind == "ffn" else 1e-2, "bf16")
    return d


# ---------------------------------------------------------------- the plain form
def _plain_mx8(y):
    """(codes, scales) of rows in blocks of 32: the largest magnitude of a block lands in [128, 256)."""
    b = y.view(y.shape[0], -1, 32)
    ea = (b.abs().amax(2).contiguous().view(torch.int32) >> 23) & 255
    byte = (ea - 7).clamp(min=0)
    up = ((254 - byte) << 23).view(torch.float32)
    return (b * up[:, :, None]).to(torch.float8_e4m3fn).view(y.shape), byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _plain_norm(c, d):
    s = d["x"].float()
    if c["add"]:
        s = s + d["residual"].float()
    r = 1.0 / torch.sqrt((s * s).sum(1) / c["H"] + EPS)
    y = s * r[:, None] * d["gain"]
    out = dict(zip(("fp8", "scale"), _plain_mx8(y))) if c["out"] == "mx8" else dict(y=y.to(_T[c["out"]]))
    if c["add"]:
        out["total"] = s.to(_T[c["stream"]])
    if c["train"]:
        out["rstd"] = r
    return out


def _plain_norm_grad(c, d):
    s, dy, r = d["x"].float(), d["dy"].float(), d["rstd"][:, None]
    a, xhat = dy * d["gain"], s * r
    dx = r * (a - xhat * ((a * xhat).sum(1, keepdim=True) / c["H"]))
    if c["carry"]:
        dx = dx + d["carry"].float()
    return dict(dx=dx.to(_T[c["stream"]]), dgain=(dy * xhat).sum(0))


def _by_expert(c, d, rows, width, f):
    """f(expert, slice) of every segment, in the rows of a result that is zero elsewhere."""
    if not c["E"]:
        return f(0, slice(0, rows))
    out = torch.zeros((rows, width), device=DEV)
    at = torch.cat([torch.arange(s, s + n, device=DEV) for s, n in d["segments"]])
    out[at] = torch.cat([f(e, slice(s, s + n)) for e, (s, n) in enumerate(d["segments"])])
    return out


def _plain_ffn(c, d):
    x, H, I = d["x"], c["H"], c["I"]
    g = _by_expert(c, d, x.shape[0], I, lambda e, s: x[s].float() @ d["Wg"][e].float())
    u = _by_expert(c, d, x.shape[0], I, lambda e, s: x[s].float() @ d["Wu"][e].float())
    h = g / (1.0 + torch.exp(-g)) * u
    y = _by_expert(c, d, x.shape[0], H, lambda e, s: h[s] @ d["Wd"][e].float())
    if c["add"]:
        y = y + d["residual"].float()
    out = dict(h=h.to(torch.bfloat16), y=y.to(torch.bfloat16))
    if c["train"]:
        out["gate"], out["up"] = g.to(torch.bfloat16), u.to(torch.bfloat16)
    return out


def _plain_ffn_grad(c, d):
    dy, H, I = d["dy"], c["H"], c["I"]
    dh = _by_expert(c, d, dy.shape[0], I, lambda e, s: dy[s].float() @ d["Wd"][e].float().t())
    g, u = d["gate"].float(), d["up"].float()
    if c["E"]:                                        # rows outside the segments are nobody's
        mine = torch.zeros(dy.shape[0], device=DEV)
        mine[torch.cat([torch.arange(s, s + n, device=DEV) for s, n in d["segments"]])] = 1.0
        g = g * mine[:, None]
    sig = 1.0 / (1.0 + torch.exp(-g))
    dg, du, h = dh * u * sig * (1.0 + g * (1.0 - sig)), dh * g * sig, g * sig * u
    dx = _by_expert(c, d, dy.shape[0], H, lambda e, s: dg[s] @ d["Wg"][e].float().t() + du[s] @ d["Wu"][e].float().t())
    if c["add"]:
        dx = dx + d["residual"].float()
    b = torch.bfloat16
    return dict(dgate=dg.to(b), dup=du.to(b), h=h.to(b), dx=dx.to(b))


def _hash(n, seed):
    """32 bits for every element of a tensor, from its place in rows of 64 and the seed."""
    i, low = torch.arange(n, device=DEV), 0xFFFFFFFF
    h = (((i >> 6) * 73856093 & low) ^ ((i & 63) * 19349663 & low) ^ seed) * 0x9E3779B1 & low
    h = h ^ (h >> 16)
    h = h * 0x85EBCA6B & low
    return h ^ (h >> 13)


def _plain_store8(x, dither, bits, low, code0, top):
    """x (non-negative, in blocks of 64) as 8-bit floats of `bits` mantissa bits: the block's power of two, then the code, rounded up
    where the dropped bits and 16 bits of dither carry. low: the least normal number, code0: what an exponent
    field of 0 stands for in 32 bits."""
    ea = (x.view(-1, 64).amax(1).contiguous().view(torch.int32) >> 23) & 255
    byte = (ea - top).clamp(min=1)
    y = (x.view(-1, 64) * ((254 - byte) << 23).view(torch.float32)[:, None]).view(-1)
    small = y < low
    y = torch.where(small, y + low, y).view(torch.int32)
    drop = 23 - bits
    code = ((y + (dither << (drop - 16)).to(torch.int32)) >> drop) - (code0 << bits)
    return torch.where(small, code - (1 << bits), code), byte.to(torch.uint8)


def _plain_adamw8(c, d):
    f, t, out = np.float32, c["t"] + d["done"], []
    d["done"] += 1
    b1, b2, o1, o2, lr, eps = (float(f(v)) for v in (B1, B2, 1 - B1, 1 - B2, LR, AEPS))
    bc1, bc2, wd = float(f(1 - B1 ** t)), float(f(1 - B2 ** t)), float(f(c["wd"]))
    for i, n in enumerate(_sizes(c)):
        g, seed = d["g"][i].float(), (SEED + 1000003 * t + i) & 0xFFFFFFFF
        up = lambda s: (s.to(torch.int32) << 23).view(torch.float32)[:, None]  # noqa: E731
        m = (d["m"][i].float().view(-1, 64) * up(d["ms"][i])).view(-1) * b1 + g * o1
        v = (d["v"][i].float().view(-1, 64) * up(d["vs"][i])).view(-1) * b2 + g * o2 * g
        p = d["p32"][i]
        p = p - (m / bc1 / (torch.sqrt(v / bc2) + eps) + p * wd) * lr
        h = _hash(n, seed ^ 0x3C6EF372)
        mc, ms = _plain_store8(m.abs(), h & 0xFFFF, 3, 2.0 ** -6, 120, 7)
        vc, vs = _plain_store8(v, h >> 16, 2, 2.0 ** -14, 112, 14)
        mc = mc | (torch.signbit(m).to(torch.int32) << 7)
        vc = torch.where(v > 0, vc.clamp(min=1), vc)
        bits = p.view(torch.int32)
        if c["sr"]:
            bits = bits + (_hash(n, seed) & 0xFFFF).to(torch.int32)
        else:
            bits = bits + 0x7FFF + ((bits >> 16) & 1)
        d["p32"][i] = p
        d["m"][i], d["ms"][i] = mc.to(torch.uint8).view(torch.float8_e4m3fn), ms
        d["v"][i], d["vs"][i] = vc.to(torch.uint8).view(torch.float8_e5m2), vs
        out.append(dict(p32=p, p16=(bits >> 16).to(torch.int16).view(torch.bfloat16), m=d["m"][i], v=d["v"][i],
                        ms=ms.view(torch.float8_e8m0fnu), vs=vs.view(torch.float8_e8m0fnu)))
    return out


_PLAIN = dict(norm=_plain_norm, norm_grad=_plain_norm_grad, ffn=_plain_ffn, ffn_grad=_plain_ffn_grad, adamw8=_plain_adamw8)


# ---------------------------------------------------------------- the framework's calls
_KINDS = {torch.float32: np.float32, torch.bfloat16: np.uint16, torch.int32: np.int32, torch.uint8: np.uint8}


def _buf(t):
    """The library's view of a torch tensor (bf16 as bit patterns); the tensor stays the owner."""
    from ancora_cutile_amd import DevBuf
    return DevBuf(shape=tuple(t.shape), dtype=_KINDS[t.dtype], ptr=t.data_ptr())


class _Kept:
    """A plan, workspace or optimizer, freed when the state and every tensor that shows one of its arrays are gone."""

    def __init__(self, owner):
        self.owner = owner

    def __del__(self):
        torch.cuda.synchronize()
        self.owner.free()


class _Shown:
    def __init__(self, buf, typestr, kept):
        self.kept = kept            # (a tensor holds what it was made from)
        self.__cuda_array_interface__ = {"shape": (buf.size,), "typestr": typestr, "data": (buf.ptr, False), "version": 2}


class State:
    def __init__(self, case, data):
        self.case, self.data, self.go, self.out, self.kept = case, data, None, None, None


def _ready_norm(c, d, state, si):
    from ancora_cutile_amd import norm
    T, H, out, b = c["T"], c["H"], {}, {}
    if c["out"] == "mx8":
        out["fp8"] = torch.empty((T, H), device=DEV, dtype=torch.uint8)
        out["scale"] = torch.empty((T, H // 32), device=DEV, dtype=torch.uint8)
    else:
        out["y"] = torch.empty((T, H), device=DEV, dtype=_T[c["out"]])
    if c["add"]:
        out["total"], b["residual"] = torch.empty((T, H), device=DEV, dtype=_T[c["stream"]]), _buf(d["residual"])
    if c["train"]:
        out["rstd"] = torch.empty(T, device=DEV)
    b.update({n: _buf(t) for n, t in out.items()})
    x, gain = _buf(d["x"]), _buf(d["gain"])
    state.go = lambda: norm.rms_norm(x, gain, si, eps=EPS, **b)
    if c["out"] == "mx8":
        out["fp8"], out["scale"] = out["fp8"].view(torch.float8_e4m3fn), out["scale"].view(torch.float8_e8m0fnu)
    state.out = out


def _ready_norm_grad(c, d, state, si):
    from ancora_cutile_amd import norm
    T, H = c["T"], c["H"]
    state.out = dict(dx=torch.empty((T, H), device=DEV, dtype=_T[c["stream"]]), dgain=torch.empty(H, device=DEV))
    b = {n: _buf(t) for n, t in {**d, **state.out}.items()}
    ws = norm.NormWorkspace(T, H)
    state.kept = _Kept(ws)
    state.go = lambda: norm.rms_norm_grad(b["dy"], b["x"], b["gain"], b["rstd"], si, b["dx"], b["dgain"], ws,
                                          carry=b.get("carry"))


def _ready_ffn(c, d, state, si):
    from ancora_cutile_amd import dispatch, ffn
    plan, H, I = None, c["H"], c["I"]
    S = c["T"]
    if c["E"]:
        plan = dispatch.RoutePlan(c["T"], c["k"], c["E"], align=c["align"])
        state.kept = _Kept(plan)
        plan.route(_buf(d["experts"]), si)
        S = plan.capacity
        assert S == _capacity(c)
    b = {n: _buf(t) for n, t in d.items() if torch.is_tensor(t)}
    new = lambda width: torch.zeros((S, width), device=DEV, dtype=torch.bfloat16)  # noqa: E731
    if c["kind"] == "ffn":
        state.out = dict(h=new(I), y=new(H))
        if c["train"]:
            state.out.update(gate=new(I), up=new(I))
        b.update({n: _buf(t) for n, t in state.out.items()})

        def go():
            ffn.gated_ffn(b["x"], b["Wg"], b["Wu"], si, b["h"], gate=b.get("gate"), up=b.get("up"), plan=plan)
            ffn.ffn_down(b["h"], b["Wd"], si, b["y"], residual=b.get("residual"), plan=plan)
    else:
        state.out = dict(dgate=new(I), dup=new(I), h=new(I), dx=new(H))
        b.update({n: _buf(t) for n, t in state.out.items()})

        def go():
            ffn.gated_ffn_grad(b["dy"], b["gate"], b["up"], b["Wd"], si, b["dgate"], b["dup"], h=b["h"], plan=plan)
            ffn.gated_ffn_dx(b["dgate"], b["dup"], b["Wg"], b["Wu"], si, b["dx"], residual=b.get("residual"), plan=plan)
    state.go = go


def _ready_adamw8(c, d, state, si):
    from ancora_cutile_amd import AdamW, _lib
    opt = AdamW({str(i): np.zeros(n, np.float32) for i, n in enumerate(_sizes(c))}, lr=LR, betas=(B1, B2), eps=AEPS, wd=c["wd"],
                sr=c["sr"], seed=SEED, grad_dtype=_KINDS[_T[c["grad"]]], state_bits=8)
    opt.t = c["t"] - 1
    kept = state.kept = _Kept(opt)
    kinds = dict(p32=("<f4", torch.float32), p16=("<i2", torch.bfloat16), m=("|u1", torch.float8_e4m3fn), v=("|u1", torch.float8_e5m2),
                 ms=("|u1", torch.float8_e8m0fnu), vs=("|u1", torch.float8_e8m0fnu))
    state.out = []
    for i, n in enumerate(_sizes(c)):
        st = opt.st[str(i)]
        for name in ("p32", "m", "ms", "v", "vs"):
            _lib.api.anc_memcpy_d2d(st[name].ptr, d[name][i].data_ptr(), st[name].nbytes, si)
        state.out.append({name: torch.as_tensor(_Shown(st[name], s, kept), device=DEV).view(t) for name, (s, t) in kinds.items()})
    grads = {str(i): _buf(g) for i, g in enumerate(d["g"])}
    state.go = lambda: opt.launch(grads, si)


def prepare(case, seed):
    c, d = case, _inputs(case, seed)
    state = State(c, d)
    if own:
        si = torch.cuda.current_stream().cuda_stream
        dict(norm=_ready_norm, norm_grad=_ready_norm_grad, ffn=_ready_ffn, ffn_grad=_ready_ffn, adamw8=_ready_adamw8)[c["kind"]](
            c, d, state, si)
    else:
        d["done"] = 0
    return state


def run(state):
    if not own:
        return _PLAIN[state.case["kind"]](state.case, state.data)
    state.go()
    return state.out


# ---------------------------------------------------------------- in 64 bits
def _grid(x, mantissa, least):
    """Spacing of 8-bit floats around x > 0: `mantissa` bits, subnormal below 2^least."""
    e = torch.floor(torch.log2(x.clamp(min=1e-300)))
    e = torch.where(torch.exp2(e) > x, e - 1, e)
    return torch.exp2(e.clamp(min=least) - mantissa)


def _scale_byte(amax, top, least):
    e = torch.floor(torch.log2(amax.clamp(min=1e-300)))
    return (e + 127 - top).clamp(min=least)


def _exact_adamw8(c, d):
    t, out = c["t"], []
    bc1, bc2 = 1 - B1 ** t, 1 - B2 ** t
    for i, n in enumerate(_sizes(c)):
        g, seed = d["g"][i].double(), (SEED + 1000003 * t + i) & 0xFFFFFFFF
        wide = lambda code, s: (code.double().view(-1, 64) * torch.exp2(s.double() - 127)[:, None]).view(-1)  # noqa: E731
        m = B1 * wide(d["m"][i], d["ms"][i]) + (1 - B1) * g
        v = B2 * wide(d["v"][i], d["vs"][i]) + (1 - B2) * g * g
        p = d["p32"][i].double()
        p = p - LR * ((m / bc1) / (torch.sqrt(v / bc2) + AEPS) + c["wd"] * p)
        row, col = torch.arange(n, device=DEV) // 64, torch.arange(n, device=DEV) % 64
        two32 = 1 << 32

        def mixed(s):
            a = ((row * 73856093) % two32).bitwise_xor((col * 19349663) % two32).bitwise_xor(torch.full_like(row, s))
            a = (a * 2654435761) % two32
            a = (a ^ (a // 65536)) * 2246822507 % two32
            return a ^ (a // 8192)
        h = mixed(seed ^ 0x3C6EF372)
        ms, vs = (_scale_byte(x.abs().view(-1, 64).amax(1), top, 1) for x, top in ((m, 7), (v, 14)))
        a = m.abs() * torch.exp2(127 - ms).repeat_interleave(64)
        b = v * torch.exp2(127 - vs).repeat_interleave(64)
        sa, sb = _grid(a, 3, -6), _grid(b, 2, -14)
        qa = torch.floor(a / sa + (h % 65536) / 65536.0) * sa
        qb = torch.floor(b / sb + (h // 65536) / 65536.0) * sb
        qb = torch.where(b > 0, qb.clamp(min=2.0 ** -16), qb)
        p16 = p
        if c["sr"]:
            step = _grid(p.abs(), 7, -126)
            p16 = torch.sign(p) * torch.floor(p.abs() / step + (mixed(seed) % 65536) / 65536.0) * step
        out.append(dict(p32=p, p16=p16, m=torch.sign(m) * qa, v=qb, ms=torch.exp2(ms - 127), vs=torch.exp2(vs - 127)))
    return out


def exact(case, seed):
    c, d, kind = case, _inputs(case, seed), case["kind"]
    if kind == "norm":
        s = d["x"].double() + (d["residual"].double() if c["add"] else 0.0)
        r = (s.pow(2).mean(1) + EPS).pow(-0.5)
        y, out = s * r[:, None] * d["gain"].double(), {}
        if c["out"] == "mx8":
            b = y.view(c["T"], -1, 32)
            byte = _scale_byte(b.abs().amax(2), 7, 0)
            b = b * torch.exp2(127 - byte)[:, :, None]
            step = _grid(b.abs(), 3, -6)
            out["fp8"], out["scale"] = (torch.round(b / step) * step).view(y.shape), torch.exp2(byte - 127)
        else:
            out["y"] = y
        if c["add"]:
            out["total"] = s
        if c["train"]:
            out["rstd"] = r
        return out
    if kind == "norm_grad":
        s, dy, r = d["x"].double(), d["dy"].double(), d["rstd"].double()
        w = dy * d["gain"].double()
        dx = w * r[:, None] - s * (r.pow(3) * (w * s).mean(1))[:, None]
        if c["carry"]:
            dx = dx + d["carry"].double()
        return dict(dx=dx, dgain=torch.mv((dy * s).t().contiguous(), r))
    if kind == "adamw8":
        return _exact_adamw8(c, d)
    if 6.0 * c["T"] * c["k"] * c["H"] * c["I"] > 2.0e11:
        return None
    rows = d["x" if kind == "ffn" else "dy"].shape[0]
    wide = lambda w: torch.zeros((rows, w), device=DEV, dtype=torch.float64)  # noqa: E731
    Wg, Wu, Wd = (d[n].double() for n in ("Wg", "Wu", "Wd"))
    names = ("gate", "up", "h") if kind == "ffn" else ("dgate", "dup", "h")
    out = {n: wide(c["I"]) for n in names}
    y = wide(c["H"])
    for e, (s, n) in enumerate(d["segments"]):
        at = slice(s, s + n)
        if kind == "ffn":
            x = d["x"][at].double()
            g, u = torch.mm(x, Wg[e]), torch.mm(x, Wu[e])
            h = g * torch.sigmoid(g) * u
            y[at] = torch.mm(h, Wd[e])
            a, b = g, u
        else:
            g, u, dh = d["gate"][at].double(), d["up"][at].double(), torch.mm(d["dy"][at].double(), Wd[e].t())
            sg = torch.sigmoid(g)
            h = u * (g * sg)
            a, b = dh * u * (sg + g * sg * (1 - sg)), dh * (g * sg)
            y[at] = torch.mm(a, Wg[e].t()) + torch.mm(b, Wu[e].t())
        for name, val in zip(names, (a, b, h)):
            out[name][at] = val
    if c["add"]:
        y = y + d["residual"].double()
    if kind == "ffn" and not c["train"]:
        del out["gate"], out["up"]
    out["y" if kind == "ffn" else "dx"] = y
    return out


# ---------------------------------------------------------------- work
_SIZE = {"bf16": 2.0, "f32": 4.0, "mx8": 1.0 + 1.0 / 32.0}


def work(case):
    c, kind = case, case["kind"]
    if kind == "norm":
        n = float(c["T"] * c["H"])
        by = n * (_SIZE[c["x"]] + _SIZE[c["out"]] + (2.0 * _SIZE[c["stream"]] if c["add"] else 0.0))
        return {"bytes": by + 4.0 * c["H"] + (4.0 * c["T"] if c["train"] else 0.0), "flops": 5.0 * n}
    if kind == "norm_grad":
        n, s = float(c["T"] * c["H"]), _SIZE[c["stream"]]
        return {"bytes": n * (_SIZE[c["dy"]] + (3.0 if c["carry"] else 2.0) * s) + 8.0 * c["H"] + 4.0 * c["T"], "flops": 10.0 * n}
    if kind == "adamw8":
        n = float(sum(_sizes(c)))
        return {"bytes": n * (_SIZE[c["grad"]] + 14.0 + 4.0 / 64.0), "flops": 30.0 * n}
    A, H, I, E = c["T"] * c["k"] * (1.0 - c["mask"]), c["H"], c["I"], c["E"]
    used = E * -math.expm1(-A / E) if E else 1.0              # experts that some token reaches
    by = used * 6.0 * H * I + A * H * (6.0 if c["add"] else 4.0)
    # h is written and read again by the product that follows it, as are the pre-activations' gradients
    by += A * I * ((4.0 + (4.0 if c["train"] else 0.0)) if kind == "ffn" else 14.0)
    return {"bytes": by, "flops": 6.0 * A * H * I}
