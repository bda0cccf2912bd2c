"""Token rows to expert-major order and back, in float64.

dispatch: the (token, choice) slots with an id in [0, E) in stable expert
order; combine: out[t] = sum_j w[t, j] * row of slot (t, j); the gradients of
both and of the renormalised top-k softmax weights."""
from __future__ import annotations

import numpy as np


def order(ids: np.ndarray, E: int):
    """(sorted_slots, slot_rows, counts) of ids [T, k]; dropped slots have row -1,
    rows past the last kept one the sentinel T * k."""
    flat = ids.reshape(-1)
    n = flat.size
    by_expert = [np.flatnonzero(flat == e) for e in range(E)]
    kept = np.concatenate(by_expert).astype(np.int64)
    slots = np.full(n, n, np.int32)
    slots[:kept.size] = kept
    rows = np.full(n, -1, np.int32)
    rows[kept] = np.arange(kept.size, dtype=np.int32)
    return slots, rows, np.array([b.size for b in by_expert], np.int32)


def dispatch(x: np.ndarray, ids: np.ndarray, E: int) -> np.ndarray:
    slots, _, counts = order(ids, E)
    out = np.zeros((ids.size, x.shape[1]), np.float64)
    kept = int(counts.sum())
    out[:kept] = x[slots[:kept] // ids.shape[1]]
    return out


def slot_values(rows: np.ndarray, slot_rows: np.ndarray, T: int, k: int) -> np.ndarray:
    """[T, k, H]: each slot's row, 0 where it was dropped."""
    v = np.where((slot_rows >= 0)[:, None], rows[np.maximum(slot_rows, 0)].astype(np.float64), 0.0)
    return v.reshape(T, k, rows.shape[1])


def combine(rows: np.ndarray, slot_rows: np.ndarray, w: np.ndarray) -> np.ndarray:
    return (slot_values(rows, slot_rows, *w.shape) * w[:, :, None].astype(np.float64)).sum(axis=1)


def combine_grad(rows: np.ndarray, slot_rows: np.ndarray, w: np.ndarray, d_out: np.ndarray):
    """(d_rows, d_weights) of combine."""
    T, k = w.shape
    d_out = d_out.astype(np.float64)
    d_w = (slot_values(rows, slot_rows, T, k) * d_out[:, None, :]).sum(axis=2)
    d_rows = np.zeros(rows.shape, np.float64)
    s = np.flatnonzero(slot_rows >= 0)
    d_rows[slot_rows[s]] = w.reshape(-1)[s][:, None].astype(np.float64) * d_out[s // k]
    return d_rows, d_w


def route_weights(logits: np.ndarray, ids: np.ndarray) -> np.ndarray:
    """Renormalised softmax weights of the chosen experts."""
    z = np.exp(logits.astype(np.float64) - logits.max(axis=1, keepdims=True))
    p = z / z.sum(axis=1, keepdims=True)
    c = np.take_along_axis(p, ids.astype(np.int64), axis=1)
    return c / c.sum(axis=1, keepdims=True)


def route_grad(ids: np.ndarray, w: np.ndarray, d_w: np.ndarray, E: int) -> np.ndarray:
    w, d_w = w.astype(np.float64), d_w.astype(np.float64)
    g = w * (d_w - (w * d_w).sum(axis=1, keepdims=True))
    out = np.zeros((ids.shape[0], E), np.float64)
    t, j = np.nonzero((ids >= 0) & (ids < E))
    np.add.at(out, (t, ids[t, j]), g[t, j])
    return out
