"""CPU restatement, in numpy and 64 bits, of the attention weights of cached
tokens, of the choice of the tokens that stay and of their moving."""

from __future__ import annotations

import numpy as np

from oracle import fp8_oracle as O

D = 128


def rows_of(cache, scales, table, n, block):
    """The first n rows [n, H, 128] of a sequence's pages in 64 bits, zeros in
    invalid blocks, and which of them exist."""
    nb = cache.shape[0]
    t = np.arange(n)
    blk = np.asarray(table, np.int64)[t // block] if n else np.zeros(0, np.int64)
    ok = (blk >= 0) & (blk < nb)
    at = np.where(ok, blk, 0)
    x = O.e4m3fn_decode(cache[at, t % block]).astype(np.float64)
    x = x * scales[at, t % block].astype(np.float64)[..., None]
    return x * ok[:, None, None], ok


def probabilities(q, k, ok, scale, sees):
    """softmax weights [Lq, Hq, keys] of queries [Lq, Hq, 128]; query i sees the
    existing keys before sees[i]."""
    q = np.asarray(q, np.float64)
    lq, hq, _ = q.shape
    n, hk, _ = k.shape
    group = hq // hk
    s = np.einsum("qhgd,khd->qhgk", q.reshape(lq, hk, group, D), k) * scale
    seen = ok[None] & (np.arange(n)[None] < np.asarray(sees)[:, None])
    s = np.where(seen[:, None, None], s, -np.inf)
    top = s.max(-1, keepdims=True, initial=-np.inf)
    p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdims=True)
    return (p / np.where(total == 0, 1.0, total)).reshape(lq, hq, n)


def record(weights, sums, ok, table, start, keep):
    """weights [NB, H, BS]: entry = keep(position) * entry + sums[h, position]."""
    block = weights.shape[2]
    for t in range(max(start, 0), sums.shape[1]):
        if ok[t]:
            at = (table[t // block], slice(None), t % block)
            weights[at] = (weights[at] if keep(t) else 0.0) + sums[:, t]


def by_kv_head(p, hk):
    """The sums over queries and the q heads of each kv head: [hk, keys]."""
    lq, hq, n = p.shape
    return p.reshape(lq, hk, hq // hk, n).sum((0, 2))


def select(weights, length, table, budget, recent, start):
    """kept [H, budget] of one sequence, and its new length."""
    nb, heads, block = weights.shape
    length = max(0, min(length, len(table) * block))
    n = min(length, budget)
    kept = np.full((heads, budget), -1, np.int32)
    first = min(start, n)
    last = min(recent, n - first)
    for h in range(heads):
        fixed = set(range(length)) if n == length else (
            set(range(first)) | set(range(length - last, length)))
        rest = [t for t in range(length) if t not in fixed]

        def weight(t):
            blk = table[t // block]
            x = weights[blk, h, t % block] if 0 <= blk < nb else np.nan
            return -np.inf if np.isnan(x) else float(x)

        lightest = {t for t in rest if not 0 <= table[t // block] < nb
                    or np.isnan(weights[table[t // block], h, t % block])}
        rest.sort(key=lambda t: (t in lightest, -weight(t), t))
        kept[h, :n] = sorted(fixed | set(rest[:n - len(fixed)]))
    return kept, n


def evict(arrays, kept, n, table, block):
    """Rows of arrays [NB, BS, H, ...] of one sequence, moved in place."""
    nb = arrays[0].shape[0]
    old = [a.copy() for a in arrays]
    for h in range(kept.shape[0]):
        for i in range(n):
            t = kept[h, i]
            a, b = table[t // block], table[i // block]
            if 0 <= a < nb and 0 <= b < nb:
                for x, o in zip(arrays, old):
                    x[b, i % block, h] = o[a, t % block, h]
