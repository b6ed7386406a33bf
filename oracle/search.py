"""Plain restatement, in numpy with 64-bit arithmetic, of the search operators over the paged KV cache:
attention of drafted trees, accepted paths, forks, compaction and the selection of beams.

TEST INFRASTRUCTURE ONLY: imported by tests/ alone. One row, sequence or page at a time, from the
definitions; slot bytes come from oracle/kv.py.
"""
import numpy as np

from . import kv as KV

BLOCK = KV.KV_BLOCK


def tree_attention(q, k_hist, v_hist, k_cur, v_cur, seen, scale):
    """One sequence. q [n, H, D], k_hist / v_hist [P, G, D], k_cur / v_cur [n, G, D], seen [n, n] bool.
    Returns (out [n, H, D], A [n, H, D], B [n, H]) with A = sum_t p_t |v_t| and B = the largest
    scale sum_d |q_d k_td| of the keys seen; zeros for a row that sees nothing."""
    q, k_hist, v_hist, k_cur, v_cur = (np.asarray(x, np.float64) for x in (q, k_hist, v_hist, k_cur, v_cur))
    n, heads, d = q.shape
    past, groups = k_hist.shape[:2]
    out, a, b = np.zeros((n, heads, d)), np.zeros((n, heads, d)), np.zeros((n, heads))
    for i in range(n):
        idx = np.flatnonzero(seen[i])
        for h in range(heads):
            g = h // (heads // groups)
            k = np.concatenate([k_hist[:, g], k_cur[idx, g]])
            v = np.concatenate([v_hist[:, g], v_cur[idx, g]])
            if len(k) == 0:
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                s = (k @ q[i, h]) * scale
                b[i, h] = (np.abs(k) @ np.abs(q[i, h])).max() * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[i, h], a[i, h] = w @ v, w @ np.abs(v)
    return out, a, b


def mask_words(seen):
    """[n, n] bool -> int64 [n, ceil(n / 64)], bit i of row j = seen[j, i]."""
    n = seen.shape[0]
    words = np.zeros((n, (n + 63) // 64), np.uint64)
    for j in range(n):
        for i in np.flatnonzero(seen[j]):
            words[j, i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return words.view(np.int64)


def write_path(ct, arena, n_blocks, n_layer, tables, past, path, n_path, cur):
    """cur [n_layer, S, N, elems] into arena (uint8, in place)."""
    n_tokens = cur.shape[2]
    sb = KV.slot_bytes(ct, cur.shape[3])
    for s in range(len(past)):
        for j in range(n_path[s]):
            pos, tok = past[s] + j, path[s][j]
            if not 0 <= tok < n_tokens or pos < 0 or pos // BLOCK >= len(tables[s]):
                continue
            blk = tables[s][pos // BLOCK]
            if not 0 <= blk < n_blocks:
                continue
            for layer in range(n_layer):
                at = KV.slot_offset(blk, layer, n_layer, pos % BLOCK, sb)
                arena[at:at + sb] = KV.encode_row(ct, cur[layer, s, tok])


def _held(table, length, n_blocks):
    """Valid pages among the first ceil(length / 16) entries."""
    return [p for p in table[:-(-length // BLOCK)] if 0 <= p < n_blocks]


def fork(tables, lengths, parents, refs):
    """(tables, lengths, refs, missing, pairs): the children, and the copies (from, to) of whole pages."""
    width, refs = len(tables[0]), list(refs)
    n_blocks = len(refs)
    lengths = [min(max(n, 0), width * BLOCK) for n in lengths]
    for t, n in zip(tables, lengths):
        for p in _held(t, n, n_blocks):
            refs[p] -= 1
    outside = list(refs)  # holders beyond this call
    new, lens = [], []
    for p in parents:
        ok = 0 <= p < len(tables)
        lens.append(lengths[p] if ok else 0)
        new.append(list(tables[p][:-(-lens[-1] // BLOCK)]) if ok else [])
    for t, n in zip(new, lens):
        for p in _held(t, n, n_blocks):
            refs[p] += 1
    full = set()
    for t, n in zip(new, lens):
        full |= {p for p in t[:n // BLOCK] if 0 <= p < n_blocks}
    held = {p for t, n in zip(new, lens) for p in _held(t, n, n_blocks)}
    free, kept, pairs, missing = [p for p in range(n_blocks) if refs[p] <= 0 and p not in held], set(), [], 0
    for t, n in zip(new, lens):
        if n % BLOCK == 0 or not 0 <= t[-1] < n_blocks:
            continue
        last = t[-1]
        if outside[last] == 0 and last not in full and last not in kept:
            kept.add(last)
            continue
        refs[last] -= 1
        if free:
            t[-1] = free.pop(0)
            refs[t[-1]] = 1
            pairs.append((last, t[-1]))
        else:
            t[-1] = -1
            missing += 1
    return [t + [-1] * (width - len(t)) for t in new], lens, refs, missing, pairs


def compact(tables, lengths, refs):
    """(tables, refs, n_live, pairs)."""
    tables, refs = [list(t) for t in tables], list(refs)
    live = sum(r > 0 for r in refs)
    movers = [p for p in range(live, len(refs)) if refs[p] > 0]
    pairs = list(zip(movers, [p for p in range(live) if refs[p] <= 0]))
    goes = dict(pairs)
    for src, dst in pairs:
        refs[dst], refs[src] = refs[src], 0
    for t, n in zip(tables, lengths):
        for i in range(min(max(-(-n // BLOCK), 0), len(t))):
            t[i] = goes.get(t[i], t[i])
    return tables, refs, live, pairs


def beam_select(x, beam, n_out):
    """x [B * W, V] -> (scores float64, parents, tokens) [B, n_out]."""
    x = np.asarray(x, np.float64)
    b, w = beam.shape
    scores, parents, tokens = np.full((b, n_out), -np.inf), np.full((b, n_out), -1), np.full((b, n_out), -1)
    for i in range(b):
        found = []
        for j in range(w):
            row = x[i * w + j]
            if np.isnan(row).any() or (row == np.inf).any() or (row == -np.inf).all() or not np.isfinite(beam[i, j]):
                continue
            top = row.max()
            lp = float(beam[i, j]) + ((row - top) - np.log(np.exp(row - top).sum()))
            best = np.argsort(-lp, kind="stable")[:n_out]
            found += [(-lp[t], j, int(t)) for t in best if lp[t] > -np.inf]
        for r, (s, j, t) in enumerate(sorted(found)[:n_out]):
            scores[i, r], parents[i, r], tokens[i, r] = -s, i * w + j, t
    return scores, parents, tokens
