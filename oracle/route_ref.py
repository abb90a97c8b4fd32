"""Tokens by expert, there and back, restated in numpy in 64 bits from the definitions. Test infrastructure only.

Pinned by tests/test_oracle_route.py: the routing through its defining properties (every assignment to a valid expert has one
slot of that expert's segment, in its own order), the row movers through the identity of inner products between a linear map and its
gradient, and the weights' gradient against differences."""
import numpy as np


def route(experts, E, align):
    """experts (T, k). (counts, offsets, slot (T, k), src (offsets[E],))."""
    experts = np.asarray(experts)
    flat = experts.reshape(-1)
    counts = np.array([np.count_nonzero(flat == e) for e in range(E)], np.int64)
    offsets = np.zeros(E + 1, np.int64)
    offsets[1:] = np.cumsum(-(-counts // align) * align)
    slot = np.full(flat.size, -1, np.int64)
    src = np.full(int(offsets[-1]), -1, np.int64)
    for e in range(E):
        at = np.nonzero(flat == e)[0]
        slot[at] = offsets[e] + np.arange(at.size)
        src[slot[at]] = at
    return counts, offsets, slot.reshape(experts.shape), src


def dispatch(slot, x, xs):
    """xs (S, H) with x's rows in their slots."""
    xs = np.array(xs, np.float64)
    for j in range(slot.shape[1]):
        at = slot[:, j] >= 0
        xs[slot[at, j]] = x[at]
    return xs


def combine(slot, ys, w=None):
    """y (T, H)."""
    y = np.zeros((slot.shape[0], ys.shape[1]))
    for j in range(slot.shape[1]):
        at = slot[:, j] >= 0
        y[at] += np.asarray(ys, np.float64)[slot[at, j]] * (1.0 if w is None else np.asarray(w, np.float64)[at, j, None])
    return y


def combine_grad(slot, dy, ys, w):
    """(dys as a function of the slot: (S, H) with zeros elsewhere, dw (T, k))."""
    dy, ys, w = (np.asarray(a, np.float64) for a in (dy, ys, w))
    dys, dw = np.zeros_like(ys), np.zeros(w.shape)
    for j in range(slot.shape[1]):
        at = slot[:, j] >= 0
        dys[slot[at, j]] = w[at, j, None] * dy[at]
        dw[at, j] = np.sum(dy[at] * ys[slot[at, j]], axis=1)
    return dys, dw


def expert_dw(counts, offsets, x, dy):
    """(E, K, N)."""
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    return np.stack([x[o:o + c].T @ dy[o:o + c] for o, c in zip(offsets[:-1], counts)])
