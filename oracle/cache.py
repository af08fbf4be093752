"""64-bit plain forms of the cache operators: attention of drafted tokens, attention weights, eviction.

Rows are float64 arrays [B, N, H, D]; lengths a list of rows per sequence.  Rows a query does not see are never
read into its sums, so what they hold has no influence.
"""
import numpy as np


def dense_rows(pages, table, keys):
    """K and V [B, keys, H, D] of pages [blocks, block, 2, H, D] through a table (negative entries from the end)."""
    block = pages.shape[1]
    n = np.arange(keys)
    rows = pages[table[:, n // block], n % block]
    return rows[:, :, 0], rows[:, :, 1]


def tree_attention(q, k, v, lengths, draft_k, draft_v, mask, scale):
    """(out [B, T, Hq, D], lse [B, Hq, T], terms): terms [B, T, Hq, D] = sum of weight times |v|, and per row the
    largest |score|, the largest sum of |q k| products and the sum of exp(score - largest)."""
    B, T, Hq, D = q.shape
    G = Hq // draft_k.shape[2]
    out, terms = np.zeros_like(q), np.zeros_like(q)
    lse, top, mass = np.full((B, Hq, T), -np.inf), np.zeros((B, Hq, T)), np.zeros((B, Hq, T))
    total = np.ones((B, Hq, T))
    for b in range(B):
        for h in range(Hq):
            keys, values = k[b, :lengths[b], h // G], v[b, :lengths[b], h // G]
            for t in range(T):
                sees = np.arange(T) <= t if mask is None else (mask if mask.ndim == 2 else mask[b])[t]
                ks = np.concatenate([keys, draft_k[b, sees, h // G]])
                vs = np.concatenate([values, draft_v[b, sees, h // G]])
                if not len(ks):
                    continue
                s = ks @ q[b, t, h] * scale
                m = s.max()
                p = np.exp(s - m)
                total[b, h, t] = p.sum()
                lse[b, h, t] = m + np.log(p.sum())
                p /= p.sum()
                out[b, t, h], terms[b, t, h] = p @ vs, p @ np.abs(vs)
                top[b, h, t], mass[b, h, t] = np.abs(s).max(), (np.abs(ks) @ np.abs(q[b, t, h])).max() * scale
    return out, lse, terms, top, mass, total


def attention_weights(q, lse, k, lengths, scale, causal=True, previous=None):
    """(weights [B, H, N], added: what the queries add, top and mass as above over the call)."""
    B, L, Hq, D = q.shape
    N, H = k.shape[1:3]
    G = Hq // H
    added = np.zeros((B, H, N))
    top = mass = 0.0
    for b in range(B):
        for h in range(Hq):
            for row in range(L):
                seen = min(lengths[b], lengths[b] - L + row + 1 if causal else lengths[b])
                if seen <= 0 or lse[b, h, row] == -np.inf:
                    continue
                keys = k[b, :seen, h // G]
                s = keys @ q[b, row, h] * scale
                added[b, h // G, :seen] += np.exp(s - lse[b, h, row])
                top = max(top, np.abs(s).max(), abs(lse[b, h, row]))
                mass = max(mass, (np.abs(keys) @ np.abs(q[b, row, h])).max() * scale)
    return (0 if previous is None else previous) + added, added, top, mass


def select_rows(weights, keep, lengths, sink, recent):
    """(rows [B, H, keep] with -1 past the count, counts [B])."""
    B, H, N = weights.shape
    rows, counts = np.full((B, H, keep), -1, np.int32), np.zeros(B, np.int32)
    for b in range(B):
        n = max(0, min(lengths[b], N))
        counts[b] = min(n, keep)
        for h in range(H):
            if n <= keep:
                rows[b, h, :n] = np.arange(n)
                continue
            middle = [(-np.inf if np.isnan(w) else float(w), np.isnan(w), i)
                      for i, w in enumerate(weights[b, h, :n]) if sink <= i < n - recent]
            middle.sort(key=lambda x: (-x[0], x[1], x[2]))           # NaN after -inf, then by index
            chosen = [i for _, _, i in middle[:keep - sink - recent]]
            rows[b, h] = sorted(list(range(sink)) + chosen + list(range(n - recent, n)))
    return rows, counts


def compact_rows(rows, counts, x, keep):
    """x [B, N, H, ...] -> [B, keep, H, ...], zero from counts on."""
    B, N, H = x.shape[:3]
    out = np.zeros((B, keep) + x.shape[2:], x.dtype)
    for b in range(B):
        for h in range(H):
            index = rows[b, h if rows.shape[1] > 1 else 0, :counts[b]]
            out[b, :counts[b], h] = x[b, index, h]
    return out
