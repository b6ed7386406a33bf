"""Layers in 8-bit integers, dense and of experts, restated in 64 bits (numpy, on the CPU): what include/dcq.h says of
dcq_quantize_i8, dcq_rms_norm_i8, dcq_mul_mat_i8, dcq_moe_route, dcq_moe_gate_up_i8 and dcq_moe_down_i8."""
import numpy as np


def to_steps(p):
    """Rows of 64-bit values -> (int8 steps, largest magnitude): the nearest of 255 steps, halves to even; 0 and NaN for a
    row with a NaN or an infinity."""
    p = np.asarray(p, np.float64)
    top = np.abs(p).max(1)
    bad = ~np.isfinite(p).all(1)
    with np.errstate(all="ignore"):
        inv = np.where(top > 0, 127.0 / top, 0.0)
        q = np.rint(p * inv[:, None])
    q[bad] = 0
    return q.astype(np.int8), np.where(bad, np.nan, top)


def quantize(x):
    """(q, s) of rows x."""
    q, top = to_steps(np.asarray(x, np.float64))
    return q, (top / 127.0).astype(np.float32)


def rms_norm(x, w, eps, r=None):
    """(h, q, s in 64 bits, y in 64 bits)."""
    h = np.asarray(x, np.float32)
    if r is not None:
        with np.errstate(all="ignore"):
            h = h + np.asarray(r, np.float32)
    h64 = h.astype(np.float64)
    with np.errstate(all="ignore"):
        p = h64 * np.asarray(w, np.float64)
        root = np.sqrt((h64 ** 2).mean(1) + np.float64(np.float32(eps)))
        q, top = to_steps(p)
        s = np.where(top == 0, 0.0, top / (127.0 * root))
        return h, q, s, p / root[:, None]


def sums(w, x):
    """Exact sums [M, N] of int8 rows x [M, K] and w [N, K]."""
    return np.asarray(x, np.float64) @ np.asarray(w, np.float64).T  # below 2^53: exact


def mul_mat(w, ws, x, xs):
    return sums(w, x) * np.asarray(ws, np.float64) * np.asarray(xs, np.float64)[:, None]


def route(logits, k, scoring="softmax", bias=None, n_group=1, topk_group=1, group_best=1, renorm=True, scale=1.0):
    """(ids, weights in 64 bits), one token after the other."""
    x = np.asarray(logits, np.float64)
    m, e = x.shape
    ids, weights = np.full((m, k), -1, np.int32), np.zeros((m, k))
    for i in range(m):
        row = x[i]
        if np.isnan(row).any() or (row == np.inf).any():
            continue
        open_ = row > -np.inf
        if bias is not None:
            open_ &= np.isfinite(bias)
        if scoring == "softmax":
            if not (row > -np.inf).any():
                continue
            score = np.exp(row - row.max())
            score /= score.sum()
        else:
            with np.errstate(over="ignore"):
                score = 1.0 / (1.0 + np.exp(-row))
        choice = np.where(open_, score + (0.0 if bias is None else np.where(np.isfinite(bias), bias, 0).astype(np.float64)), -np.inf)
        if n_group > 1:
            parts = choice.reshape(n_group, -1)
            worth = []
            for g in range(n_group):
                best = [c for c in sorted(parts[g], reverse=True)[:group_best] if c > -np.inf]
                worth.append(sum(best) if best else -np.inf)
            kept = sorted(range(n_group), key=lambda g: (-worth[g], g))[:topk_group]
            for g in range(n_group):
                if g not in kept:
                    parts[g] = -np.inf
            choice = parts.reshape(-1)
        got = [j for j in sorted(range(e), key=lambda j: (-choice[j], j)) if choice[j] > -np.inf][:k]
        total = sum(score[j] for j in got)
        for j, ex in enumerate(got):
            ids[i, j] = ex
            weights[i, j] = scale * score[ex]
            if renorm:
                weights[i, j] = weights[i, j] / total if total > 0 else 0.0
    return ids, weights


def gate_up(ids, n_expert, wg, wgs, wu, wus, x, xs):
    """(h, gate, up) in 64 bits, a row per slot; zeros for slots of no expert."""
    m, k = ids.shape
    gate, up = np.zeros((m * k, wg.shape[1])), np.zeros((m * k, wg.shape[1]))
    for slot, e in enumerate(ids.reshape(-1)):
        if 0 <= e < n_expert:
            t = slice(slot // k, slot // k + 1)
            gate[slot] = mul_mat(wg[e], wgs[e], x[t], xs[t])[0]
            up[slot] = mul_mat(wu[e], wus[e], x[t], xs[t])[0]
    with np.errstate(over="ignore"):
        return gate / (1.0 + np.exp(-gate)) * up, gate, up


def down(ids, n_expert, w, ws, h, hs, weights, r=None):
    """(y, the sum of the terms' magnitudes) in 64 bits."""
    m, k = ids.shape
    y, size = np.zeros((m, w.shape[1])), np.zeros((m, w.shape[1]))
    for slot, e in enumerate(ids.reshape(-1)):
        if 0 <= e < n_expert:
            t = slice(slot, slot + 1)
            part = np.float64(weights.reshape(-1)[slot]) * mul_mat(w[e], ws[e], h[t], hs[t])[0]
            y[slot // k] += part
            size[slot // k] += np.abs(part)
    if r is not None:
        y, size = y + r, size + np.abs(r)
    return y, size
