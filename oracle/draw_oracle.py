"""Draws of indices from scores restated from their definition (include/pointslam_hip.h, psl_draw_indices) with numpy in
extended precision: sort, cut, running sums, search.  Test infrastructure only."""
import numpy as np


def kept_weights(s, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """Weights (longdouble [V]) of one row after the cuts; zeros where an entry cannot be drawn."""
    s = np.asarray(s, dtype=np.float64)
    out = np.zeros(s.shape, dtype=np.longdouble)
    ok = ~np.isnan(s) & (s != -np.inf)
    if mask is not None:
        ok &= np.asarray(mask).astype(bool)
    order = np.flatnonzero(ok)
    if order.size == 0:
        return out
    order = order[np.argsort(-s[order], kind="stable")]          # score descending, index ascending
    M = s[order[0]]
    if not temperature > 0 or top_p <= 0:
        order = order[:1]
        temperature = 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(s[order] == M, 1.0, 0.0 if M == np.inf else np.exp((s[order] - M).astype(np.longdouble) / temperature))
    w = w.astype(np.longdouble)
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    if top_p < 1:
        cum = np.cumsum(w)
        # the product is an fp64 number by definition: of 700 equal entries 0.8 keeps 560, though the fp64 number 0.8 lies
        # 4e-17 above 4/5 and the exact product 3e-14 above 560
        # (summed from the smallest: 15 000 entries of 4e-18 behind 138 of 1 are lost one by one, together they are 6e-14)
        total = np.cumsum(w[::-1])[-1]
        n = min(int(np.searchsorted(cum, np.longdouble(np.float64(top_p) * np.float64(total)), side="left")) + 1, w.size)
        order, w = order[:n], w[:n]
    keep = w >= min(max(min_p, 0.0), 1.0)
    out[order[keep]] = w[keep]
    return out


def draws(s, u, **cut):
    """(indices int64 [n], probabilities float64 [n]) of one row."""
    w = kept_weights(s, **cut)
    u = np.asarray(u, dtype=np.float64)
    u = np.clip(np.where(np.isnan(u), 0.0, u), 0.0, 1.0 - 2.0 ** -24)
    if not (w > 0).any():
        return np.full(u.shape, -1, np.int64), np.zeros(u.shape)
    cum = np.cumsum(w)
    idx = np.searchsorted(cum, u.astype(np.longdouble) * cum[-1], side="right")
    idx = np.minimum(idx, np.flatnonzero(w > 0)[-1])
    return idx, (w[idx] / cum[-1]).astype(np.float64)
