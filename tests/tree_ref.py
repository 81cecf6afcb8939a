"""Trees of drafted tokens in plain numpy, 64 bits: what their rows see, attention
over it, which drafts stay, and the move of their positions (see
citlali_hip_draft_tree and the calls after it)."""
from __future__ import annotations

import numpy as np


def tree(rng, n, wide=3):
    """Parents of a tree of n rows, level after level."""
    parents, at = [-1], 0
    for i in range(1, n):
        at = min(i - 1, at + int(rng.random() < 1 / wide))
        parents.append(at)
    return parents[:n]


def masks_of(parents):
    """[n][n] what each row sees, and the rows' depths (-1: no way to the top)."""
    n = len(parents)
    see, depth = np.zeros((n, n), bool), np.full(n, -1)
    for i, p in enumerate(parents):
        if p != -1 and not (0 <= p < i and depth[p] >= 0):
            continue
        if p >= 0:
            see[i] = see[p]
        see[i, i] = True
        depth[i] = see[i].sum() - 1
    return see, depth


def pack(see, words):
    """Rows of bits as uint64 words."""
    out = np.zeros((len(see), words), np.uint64)
    for i, row in enumerate(see):
        for j in np.flatnonzero(row):
            out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out


def attention(cache, q, query_start, lens, table, sees, max_context=None, max_query=None):
    """kv4_ref.attention with sees[s][i][j]: row i of sequence s sees row j."""
    tokens, heads, hd = q.shape
    kv, page = cache.kv, cache.page
    g = heads // kv
    out = np.full(q.shape, np.nan)
    spread, reach = np.zeros(q.shape), np.zeros((tokens, heads, 1))
    for s, length in enumerate(lens):
        r0, r1 = int(query_start[s]), int(query_start[s + 1])
        n = r1 - r0
        length = max(0, int(length))
        p = np.arange(length if max_context is None else min(length, max_context))
        pages = np.asarray(table[s])[p // page] if len(p) else np.zeros(0, int)
        here = (pages >= 0) & (pages < cache.num_pages)
        at = np.where(here, pages, 0)
        k = cache.k[at, :, p % page].astype(np.float64)
        v = cache.v[at, :, p % page].astype(np.float64)
        node = p - (length - n)
        for i in range(n if max_query is None else min(n, max_query)):
            seen = here & ((node < 0) | sees[s][i][np.clip(node, 0, max(0, n - 1))])
            for h in range(heads):
                kk, vv = k[seen, h // g], v[seen, h // g]
                if not len(kk):
                    out[r0 + i, h] = 0
                    continue
                qq = q[r0 + i, h].astype(np.float64)
                x = kk @ qq / np.sqrt(hd)
                w = np.exp(x - x.max())
                w /= w.sum()
                out[r0 + i, h] = w @ vv
                spread[r0 + i, h] = w @ np.abs(vv)
                reach[r0 + i, h] = (np.abs(kk) @ np.abs(qq)).max() / np.sqrt(hd)
    return out, spread, reach


def distribution(x, heat):
    """A row's probabilities; None where it has none."""
    x = np.asarray(x).astype(np.float64)
    if np.isnan(x).any() or not np.isfinite(x.max()):
        return None
    if not heat > 0:
        p = np.zeros(len(x))
        p[np.argmax(x)] = 1                    # numpy's: the first of equal ones
        return p
    e = np.exp((x - x.max()) / np.float64(np.float32(heat)))
    return e / e.sum()


def unit(u):
    """Random numbers as the calls take them: nearest in [0, 1), NaN as 0."""
    u = np.float32(u)
    return float(min(u, np.float32(1 - 2 ** -24))) if u >= 0 else 0.0


def draw(p, u):
    """The first id whose running sum exceeds u of the total."""
    run = np.cumsum(p)
    return int(np.searchsorted(run, unit(u) * run[-1], side="right"))


def verify(logits, draft, tokens, parents, heat, uniforms, max_query):
    """(path, next token, probabilities) of one sequence's rows."""
    n = min(len(logits), max_query)
    probs = np.zeros(n)
    if n == 0:
        return [], -1, probs
    vocab = logits.shape[1]
    p = [distribution(x, heat) for x in logits[:n]]
    q = [distribution(x, heat) for x in draft[:n]] if draft is not None else None
    parents = list(range(-1, n - 1)) if parents is None else list(parents[:n])
    real = lambda i: 0 <= parents[i] < i and 0 <= tokens[i] < vocab and p[parents[i]] is not None  # noqa: E731
    for i in range(n):
        if real(i):
            probs[i] = p[parents[i]][tokens[i]]
    current, path = 0, [0]
    rest = None if p[0] is None else p[0].copy()
    left = 1.0
    for i in range(1, n):
        if not 0 <= parents[i] < i or parents[i] != current or rest is None:
            continue
        x = int(tokens[i])
        inside = 0 <= x < vocab
        mine = rest[x] if inside else 0.0
        if draft is None:
            taken = unit(uniforms[i]) * left < mine
        else:
            row = q[current]
            taken = row is not None and unit(uniforms[i]) * (row[x] if inside else 0.0) < mine
        if taken:
            current, left = i, 1.0
            path.append(i)
            rest = None if p[i] is None else p[i].copy()
        elif draft is None:
            left -= mine
            if inside:
                rest[x] = 0
        elif q[current] is not None:
            rest = np.maximum(rest - q[current], 0)
    if rest is None:
        return path, -1, probs
    if not rest.sum() > 0:
        rest = p[current]
    return path, draw(rest, uniforms[0]), probs


def keep(read, write, first, kept, count):
    """Positions first + kept[j] to first + j, all read before any is written.
    read(position) gives a token's bytes or None, write(position, bytes) takes them."""
    moves = [(first + j, read(first + k)) for j, k in enumerate(kept[:count]) if k > j]
    for to, what in moves:
        if what is not None:
            write(to, what)
