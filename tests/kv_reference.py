"""The paged cache, its attention and its append in 64 bits, for the tests: numpy only, written from the formulas."""
import numpy as np

NO_PAGE = 0xFFFFFFFF
F16, I8 = 1, 24


def page_bytes(t, heads, dim, page):
    return 2 * heads * page * (2 * dim if t == F16 else dim + 4)


def encode(t, rows):
    """Pages of f32 rows [pages][2][heads][page][dim] as the cache's bytes, and the values they stand for (f64)."""
    pages = rows.shape[0]
    if t == F16:
        h = rows.astype(np.float16)
        return h.view(np.uint8).reshape(pages, -1), h.astype(np.float64)
    top = np.abs(rows).max(-1)
    scale = (top / np.float32(127)).astype(np.float32)
    q = np.clip(np.rint(rows * np.where(top > 0, 127 / np.where(top > 0, top, 1), 0)[..., None]), -127, 127).astype(np.int8)
    parts = [q.reshape(*q.shape[:3], -1).view(np.uint8), scale.view(np.uint8).reshape(*scale.shape[:3], -1)]
    return np.concatenate(parts, -1).reshape(pages, -1), q * scale[..., None].astype(np.float64)


def decode(t, data, pages, heads, dim, page):
    """The cache's bytes as values (f64): [pages][2][heads][page][dim]."""
    if t == F16:
        return data.view(np.float16).reshape(pages, 2, heads, page, dim).astype(np.float64)
    d = data.reshape(pages, 2, heads, page * (dim + 4))
    q = d[..., :page * dim].copy().view(np.int8).reshape(pages, 2, heads, page, dim)
    scale = d[..., page * dim:].copy().view(np.float32)
    with np.errstate(invalid="ignore"):
        return q * scale[..., None].astype(np.float64)


def attend(values, table, starts, lens, q, q_heads, scale, window, page):
    """softmax(scale q . k) v of every new token, f64; `values` as of decode, q [tokens][q_heads][dim]."""
    pages, _, heads, _, dim = values.shape
    out = np.zeros(q.shape)
    group = q_heads // heads
    for s, length in enumerate(lens):
        new = slice(starts[s], starts[s + 1])
        pos = int(length) - int(starts[s + 1] - starts[s]) + np.arange(starts[s + 1] - starts[s])
        at = np.arange(int(length))
        p = table[s][at // page] if len(at) else np.zeros(0, np.uint32)
        at, p = at[p < pages], p[p < pages].astype(np.int64)
        seen = at[None] <= pos[:, None]
        if window:
            seen &= at[None] > pos[:, None] - window
        some = seen.any(1)
        if not some.any():
            continue
        # what is not seen may be any bits
        used = seen.any(0)
        at, p, seen = at[used], p[used], seen[:, used]
        for h in range(q_heads):
            k, v = values[p, 0, h // group, at % page], values[p, 1, h // group, at % page]
            x = np.where(seen, q[new, h].astype(np.float64) @ k.T * scale, -np.inf)[some]
            w = np.exp(x - x.max(1, keepdims=True))
            out[np.arange(starts[s], starts[s + 1])[some], h] = w @ v / w.sum(1, keepdims=True)
    return out


def turn(x, pos, table, rope_dim, halves, norm=None, eps=1e-6):
    """Norm and rotation of rows [tokens][heads][dim] at positions pos, f64."""
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
    if not rope_dim:
        return x
    c, s = (table.astype(np.float64)[pos][:, i, None, :] for i in range(2))
    a = slice(0, rope_dim // 2) if halves else slice(0, rope_dim, 2)
    b = slice(rope_dim // 2, rope_dim) if halves else slice(1, rope_dim, 2)
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


class Batch:
    """Sequences with their new tokens, and pages in a shuffled order."""

    def __init__(self, rng, new, lens, page, spare=2, table_pages=None):
        self.new, self.lens, self.page = list(new), list(lens), page
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
        self.tokens = int(self.starts[-1])
        need = [-(-n // page) for n in lens]
        self.table_pages = table_pages or max(1, max(need))
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(lens), self.table_pages), NO_PAGE, np.uint32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.spare = order[at:]

    def positions(self):
        return np.concatenate([np.arange(n) + length - n for n, length in zip(self.new, self.lens)]).astype(np.int64)

    def seq(self):
        return np.repeat(np.arange(len(self.new)), self.new)

    def upload(self, eff, ctx, max_new=None, max_len=None):
        b = [ctx.upload(x.astype(np.uint32)) for x in (self.table, self.starts, np.array(self.lens))]
        return eff.KvBatch(*b, seqs=len(self.new), tokens=self.tokens, table_pages=self.table_pages,
                           max_new=max_new or max(1, max(self.new)), max_len=max_len or max(1, max(self.lens)))
