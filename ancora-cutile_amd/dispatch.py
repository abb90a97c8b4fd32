"""Tokens sorted by expert and back, for the layers whose expert tensors `ExpertOptimizer` steps.

    plan = RoutePlan(tokens, top_k, experts, align=128)
    plan.route(expert_ids, si)                       # (T, k) expert of every choice, -1: none (a masked token)
    dispatch(plan, x, si, xs)                        # xs: one segment of rows per expert
    ...                                              # the experts' products, ys
    combine(plan, ys, weights, si, y)                # y[t] = sum over j of weights[t, j] * ys[slot[t, j]]

and backwards `combine_grad` (rows and weights), `grads.expert_dW` (the experts' weights, over the ragged segments) and
`dispatch_grad`. Everything is decided on the device: no copy to the host, and each call may be captured into a graph. Outputs
that overlap an input are refused.
"""
import numpy as np

from . import _lib
from ._lib import api
from .devbuf import DevBuf
from .embed import _TYPES, _ids, _rows_of, _type


class RoutePlan:
    """Where every (token, choice) of a batch goes: room for `tokens` tokens of `top_k` choices among `experts`.

    counts (E,) int32     tokens of each expert
    offsets (E + 1,)      first slot of each expert's segment, filled up to a multiple of `align` (a power of two up to 256)
    order (E,)            the experts by falling number of tokens (as they are numbered beyond 256 experts)
    slot (tokens, k)      slot of token t's choice j, -1: none
    src (capacity,)       the assignment t * k + j of a slot, -1: filling, or behind the last segment
    capacity              slots (rows of xs, ys) that hold every routing of `tokens` tokens

    The order inside a segment is the tokens' own. The arrays are one set of buffers: calls on different streams (or
    replays of graphs) that use one plan are put in order by the caller; work that overlaps takes a plan each."""

    def __init__(self, tokens, top_k, experts, align=1):
        _lib.init()
        self.tokens, self.k, self.E, self.align = int(tokens), int(top_k), int(experts), int(align)
        if self.tokens <= 0 or not 0 < self.k <= 512:
            raise ValueError(f"RoutePlan: {tokens} tokens of {top_k} choices")
        A = self.tokens * self.k
        self.capacity = api.anc_route_capacity(A, self.E, self.align)
        if self.capacity < 0:
            raise ValueError("RoutePlan: " + _lib.load().anc_last_error().decode())
        nbytes = api.anc_route_workspace_bytes(A, self.E)
        sizes = (self.E, self.E + 1, self.E, A, self.capacity)
        self._block = DevBuf.empty((sum(sizes),), np.int32)
        self._ws = DevBuf.empty((nbytes,), np.uint8)
        at = [self._block.ptr + 4 * sum(sizes[:i]) for i in range(5)]
        shapes = ((self.E,), (self.E + 1,), (self.E,), (self.tokens, self.k), (self.capacity,))
        bufs = [DevBuf(shape=sh, dtype=np.int32, ptr=p) for sh, p in zip(shapes, at)]
        self.counts, self.offsets, self.order, self.slot, self.src = bufs
        # (as the library takes them: converting a number of every call's arguments was a tenth of a small call)
        self._at = (*(_lib.u64(p) for p in at), _lib.i64(self.capacity), _lib.u64(self._ws.ptr), _lib.i64(nbytes))
        self.active = None                     # tokens of the last `route`

    def _used(self, who):
        if self._block is None:
            raise _lib.AncoraError("RoutePlan: freed")
        if self.active is None and who:
            raise _lib.AncoraError(f"{who}: no tokens were routed yet")

    def route(self, expert_ids, si, tokens=None):
        """Sort the choices of the first `tokens` tokens (default: all of expert_ids). expert_ids: (T, k) int32 or int64
        DevBuf, T at most the plan's tokens. Later calls work on that many tokens. Asynchronous on `si`."""
        self._used(None)
        nbytes, have = _ids(expert_ids, "RoutePlan.route")
        if len(expert_ids.shape) != 2 or expert_ids.shape[1] != self.k:
            raise ValueError(f"RoutePlan.route: expert ids are {expert_ids.shape}, (T, {self.k}) expected")
        n = expert_ids.shape[0] if tokens is None else int(tokens)
        if not 0 <= n <= min(expert_ids.shape[0], self.tokens):
            raise ValueError(f"RoutePlan.route: {n} of {expert_ids.shape[0]} tokens, room for {self.tokens}")
        api.anc_route(expert_ids.ptr, nbytes, n * self.k, self.E, self.align, *self._at, int(si))
        self.active = n

    def free(self):
        if self._block is not None:
            self._block.free()
            self._ws.free()
            self._block = None


def dispatch(plan, x, si, xs):
    """xs[slot[t, j]] = x[t]: x (T, H) into the experts' segments of xs (capacity, H), both float32 or both bf16 bits. The rows
    that fill up a segment become zero; rows behind the last segment are left as they were."""
    plan._used("dispatch")
    H = x.shape[-1]
    _rows_of(x, plan.active, H, "dispatch", "x")
    _rows_of(xs, plan.capacity, H, "dispatch", "xs")
    if x.dtype != xs.dtype:
        raise ValueError(f"dispatch: x is {x.dtype}, xs {xs.dtype}")
    counts, offsets, _, slot = plan._at[:4]
    api.anc_dispatch(slot, counts, offsets, plan.active, plan.k, plan.E, plan.align, x.ptr, xs.ptr, plan._at[5],
                     _type(x, "dispatch"), H, int(si))


def _weights(plan, w, who):
    if _TYPES.get(w.dtype) != _lib.F32 or len(w.shape) != 2 or w.shape[1] != plan.k or w.shape[0] < plan.active:
        raise ValueError(f"{who}: weights are {w.shape} {w.dtype}, ({plan.active}, {plan.k}) float32 expected")
    return w.ptr


def combine(plan, ys, weights, si, y):
    """y[t] = sum over j of weights[t, j] * ys[slot[t, j]]: ys (capacity, H), weights (T, k) fp32 (None: all one), y (T, H); rows
    float32 or bf16 bits, each of its own type. Sums are fp32 in the order of j. A choice without a slot adds nothing, a
    token without any gives a zero row."""
    plan._used("combine")
    H = y.shape[-1]
    _rows_of(ys, plan.capacity, H, "combine", "ys")
    _rows_of(y, plan.active, H, "combine", "y")
    w = 0 if weights is None else _weights(plan, weights, "combine")
    api.anc_combine(plan._at[3], w, plan.active, plan.k, ys.ptr, plan._at[5], _type(ys, "combine"), y.ptr,
                    _type(y, "combine"), H, int(si))


def dispatch_grad(plan, dxs, si, dx):
    """Gradient of `dispatch`: dx[t] = sum over j of dxs[slot[t, j]]."""
    combine(plan, dxs, None, si, dx)


def combine_grad(plan, dy, ys, weights, si, dys, dweights):
    """Gradients of `combine` for dy (T, H): dys[slot[t, j]] = weights[t, j] * dy[t] in dys (capacity, H), of the type of ys, with
    the rows that fill up a segment zero; dweights[t, j] = <dy[t], ys[slot[t, j]]> fp32, 0 for a choice without a slot."""
    plan._used("combine_grad")
    H = dy.shape[-1]
    _rows_of(dy, plan.active, H, "combine_grad", "dy")
    _rows_of(ys, plan.capacity, H, "combine_grad", "ys")
    _rows_of(dys, plan.capacity, H, "combine_grad", "dys")
    if ys.dtype != dys.dtype:
        raise ValueError(f"combine_grad: ys is {ys.dtype}, dys {dys.dtype}")
    counts, offsets, _, slot = plan._at[:4]
    api.anc_combine_grad(slot, _weights(plan, weights, "combine_grad"), counts, offsets, plan.active, plan.k, plan.E, plan.align, dy.ptr,
                         _type(dy, "combine_grad"), ys.ptr, dys.ptr, plan._at[5], _type(ys, "combine_grad"),
                         _weights(plan, dweights, "combine_grad"), H, int(si))
