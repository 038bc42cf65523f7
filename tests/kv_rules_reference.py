"""Positions on several axes, masks and rules on scores, copies and compaction of the paged cache in 64 bits, for the
tests: numpy only, written from the formulas. The cache's bytes and values are those of kv_reference."""
import numpy as np

from kv_reference import F16


def turn_at(x, at, axis, table, rope_dim, halves, norm=None, eps=1e-6):
    """Norm and rotation of rows [tokens][heads][dim], pair i by the position at[axis[i]][token], f64."""
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
    y, half = x.copy(), rope_dim // 2
    for i in range(half):
        a, b = (i, half + i) if halves else (2 * i, 2 * i + 1)
        p = at[axis[i]].astype(np.int64)
        there = p < table.shape[0]
        c, s = (np.where(there, table[np.minimum(p, table.shape[0] - 1), j, i].astype(np.float64), np.nan)[:, None] for j in range(2))
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def random_tree(rng, n, back=0.4):
    """The parent of each of n drafts, -1 for the first."""
    return [-1] + [max(0, i - 1 - int(rng.exponential(1 / back))) for i in range(1, n)]


def tree_mask(parents):
    """[n][n]: which drafts a draft sees, its ancestors and itself."""
    m = np.zeros((len(parents), len(parents)), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def tree_words(masks, words):
    """The masks of several sequences [n][n] as rows of u32 words, one after the other."""
    rows = []
    for m in masks:
        for r in m:
            bits = np.zeros(32 * words, np.uint64)
            bits[:len(r)] = r
            rows.append((bits.reshape(words, 32) << np.arange(32, dtype=np.uint64)).sum(1).astype(np.uint32))
    return np.array(rows, np.uint32).reshape(-1, words)


def attend_rules(values, b, q, q_heads, scale, window=0, cap=0.0, slopes=None, ranges=None, masks=None):
    """softmax of the scores under the rules, times v, of every new token of the batch b, f64.

    ranges [tokens][2], masks: a tree's [n][n] of each sequence. A token that sees nothing gives zeros."""
    pages, _, heads, _, dim = values.shape
    out, group = np.zeros(q.shape), q_heads // heads
    for s, length in enumerate(b.lens):
        n = b.new[s]
        if n == 0 or length == 0:
            continue
        first, t = length - n, np.arange(length)
        place = first + np.arange(n)
        page = b.table[s][t // b.page]
        pos, key = place, t
        if masks is not None:
            m = np.asarray(masks[s], bool)
            pos = first + m.sum(1) - 1
            seen = np.ones((n, length), bool)
            key = t.copy()
            for j in range(n):
                if first + j >= 0:
                    seen[:, first + j] = m[:, j]
                    key[first + j] = pos[j]
        elif ranges is not None:
            r = ranges[b.starts[s]:b.starts[s] + n].astype(np.int64)
            seen = (t >= r[:, :1]) & (t < r[:, 1:])
        else:
            seen = t <= pos[:, None]
        if window:
            seen = seen & (key > pos[:, None] - window)
        seen = seen & (place >= 0)[:, None] & (page < pages)
        used = seen.any(0)
        if not used.any():
            continue
        some = seen.any(1)
        p, slot = page[used].astype(np.int64), (t % b.page)[used]
        far = np.abs(pos[:, None] - key[used]).astype(np.float64)
        for h in range(q_heads):
            k, v = values[p, 0, h // group, slot], values[p, 1, h // group, slot]
            x = q[b.starts[s]:b.starts[s] + n, h].astype(np.float64) @ k.T * scale
            if cap:
                x = cap * np.tanh(x / cap)
            if slopes is not None:
                x = x - np.float64(slopes[h]) * far
            x = np.where(seen[:, used], x, -np.inf)[some]
            w = np.exp(x - x.max(1, keepdims=True))
            out[np.arange(b.starts[s], b.starts[s] + n)[some], h] = w @ v / w.sum(1, keepdims=True)
    return out


def row_bytes(t, data, pages, heads, dim, page):
    """The cache's rows as bytes, [pages][2][heads][page][bytes]: int8 rows with their scales."""
    if t == F16:
        return data.reshape(pages, 2, heads, page, 2 * dim).copy()
    d = data.reshape(pages, 2, heads, page * (dim + 4))
    return np.concatenate([d[..., :page * dim].reshape(pages, 2, heads, page, dim), d[..., page * dim:].reshape(pages, 2, heads, page, 4)], -1)
