"""numpy restatement, in 64 bits, of the language-model operators (test oracle; see oracle/__init__).

Inputs are float64 arrays (of values that the tested type holds); results stay in float64.  The page operations
work on lists, one sequence at a time.
"""
from __future__ import annotations

import numpy as np


# ------------------------------------------------------------ norms of queries and keys, rotation
def rope_pairs(rotary, interleaved):
    i = np.arange(rotary // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)


def rotate(y, cos, sin, rotary, interleaved, back=False):
    """cos, sin: [tokens, rotary / 2], y [tokens, heads, dim]."""
    a, b = rope_pairs(rotary, interleaved)
    c, s = cos[:, None], sin[:, None] * (-1 if back else 1)
    z = y.copy()
    z[..., a] = y[..., a] * c - y[..., b] * s
    z[..., b] = y[..., b] * c + y[..., a] * s
    return z


def norm_rope(x, w, cos, sin, rotary, interleaved, eps):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return rotate(x * r * w, cos, sin, rotary, interleaved)


def norm_rope_backward(dz, x, w, cos, sin, rotary, interleaved, eps):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    dy = rotate(dz, cos, sin, rotary, interleaved, back=True)
    xh = x * r
    g = dy * w
    return r * (g - xh * (g * xh).mean(-1, keepdims=True)), (dy * xh).sum((0, 1))


# ------------------------------------------------------------ attention over a paged cache
def keys_of(pages, prefix, row, n):
    """The first n keys (or values) of a sequence: [n, heads, dim]."""
    page_size = pages.shape[1]
    got = [pages[prefix[j // page_size] if j // page_size < len(prefix) else row[j // page_size], j % page_size]
           for j in range(n)]
    return np.array(got).reshape(n, *pages.shape[2:])


def shared_prefix_attention(q, k_pages, v_pages, prefix, table, lens, scale):
    """(out, lse, bound): bound[...] = softmax @ |v|, what the error of out is measured by."""
    B, Q, hq, d = q.shape
    group = hq // k_pages.shape[2]
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full((B, Q, hq), -np.inf)
    for b in range(B):
        n = max(int(lens[b]), 0)
        k, v = keys_of(k_pages, prefix, table[b], n), keys_of(v_pages, prefix, table[b], n)
        for t in range(Q):
            m = n - Q + 1 + t
            if m <= 0:
                continue
            for h in range(hq):
                s = scale * (k[:m, h // group] @ q[b, t, h])
                top = s.max()
                p = np.exp(s - top)
                lse[b, t, h] = top + np.log(p.sum())
                p /= p.sum()
                out[b, t, h] = p @ v[:m, h // group]
                mag[b, t, h] = p @ np.abs(v[:m, h // group])
    return out, lse, mag


# ------------------------------------------------------------ the paged cache
class Cache:
    """The state of a paged cache on lists, and its operations."""

    def __init__(self, pool, table, lens, refs):
        self.pool = pool.copy()  # [planes, pages, page_size, ...]
        self.page = pool.shape[2]
        self.width = table.shape[1]
        self.table = table.copy()
        self.lens = lens.copy()
        self.refs = refs.copy()

    def _free(self):
        return [p for p in range(len(self.refs)) if self.refs[p] == 0]

    def _valid(self, slots, i):
        return 0 <= slots[i] < len(self.lens) and slots[i] not in slots[:i]

    def reserve(self, seqs, tokens):
        free, asked, granted = self._free(), 0, []
        for i, c in enumerate(seqs):
            ok = self._valid(list(seqs), i) and self.lens[c] + tokens <= self.width * self.page
            need = 0
            if ok:
                held = -(-self.lens[c] // self.page)
                need = -(-(self.lens[c] + tokens) // self.page) - held
                ok = asked + need <= len(free) or need == 0
            if ok:
                for j in range(need):
                    self.table[c, held + j] = free[asked + j]
                    self.refs[free[asked + j]] = 1
                self.lens[c] += tokens
            asked += need
            granted.append(int(ok))
        return granted

    def append(self, k, v, seqs):
        tokens = k.shape[1]
        for i, c in enumerate(seqs):
            for t in range(tokens):
                pos = self.lens[c] - tokens + t
                self.pool[0, self.table[c, pos // self.page], pos % self.page] = k[i, t]
                self.pool[1, self.table[c, pos // self.page], pos % self.page] = v[i, t]

    def fork(self, parents, children):
        free, asked, granted, todo = self._free(), 0, [], []
        for i, (p, c) in enumerate(zip(parents, children)):
            ok = 0 <= p < len(self.lens) and self._valid(list(children), i)
            if ok and p != c:
                n, row = self.lens[p], self.table[p].copy()
                if n % self.page:
                    ok = asked < len(free)
                    if ok:
                        todo.append((c, n, row, free[asked]))
                    asked += 1
                else:
                    todo.append((c, n, row, None))
            granted.append(int(ok))
        new = []
        for c, n, row, page in todo:
            if page is not None:
                self.pool[:, page] = self.pool[:, row[n // self.page]]
                row[n // self.page] = page
            row[-(-n // self.page):] = -1
            new.append((c, n, row))
        for c, n, row in new:
            for p in row[row >= 0]:
                self.refs[p] += 1
        for c, n, row in new:
            for p in self.table[c][self.table[c] >= 0]:
                self.refs[p] -= 1
            self.table[c], self.lens[c] = row, n
        return granted

    def free(self, seqs):
        for c in seqs:
            if not 0 <= c < len(self.lens):
                continue
            if self.lens[c]:
                for p in self.table[c][self.table[c] >= 0]:
                    self.refs[p] -= 1
                self.table[c] = -1
            self.lens[c] = 0

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] <= 0]
        for p in range(live, len(self.refs)):
            if self.refs[p] > 0:
                to = holes.pop(0)
                self.pool[:, to] = self.pool[:, p]
                self.refs[to], self.refs[p] = self.refs[p], 0
                self.table[self.table == p] = to
        return live


# ------------------------------------------------------------ logits
def penalize_logits(logits, prompt, output, repetition, presence, frequency, bias_ids, bias_values, mask):
    """mask: bool [rows, vocab] (True: allowed) or None; the rest as in the operator, None where absent."""
    x = logits.copy()
    rows, vocab = x.shape
    for b in range(rows):
        count = np.zeros(vocab, dtype=np.int64)
        seen = np.zeros(vocab, dtype=bool)
        if output is not None:
            ids = output[b][(output[b] >= 0) & (output[b] < vocab)]
            np.add.at(count, ids, 1)
            seen[ids] = True
        if prompt is not None:
            seen[prompt[b][(prompt[b] >= 0) & (prompt[b] < vocab)]] = True
        if repetition is not None:
            x[b] = np.where(seen, np.where(x[b] > 0, x[b] / repetition[b], x[b] * repetition[b]), x[b])
        if frequency is not None:
            x[b] = np.where(count > 0, x[b] - frequency[b] * count, x[b])
        if presence is not None:
            x[b] = np.where(count > 0, x[b] - presence[b], x[b])
        if bias_ids is not None:
            last = {int(v): float(z) for v, z in zip(bias_ids[b], bias_values[b]) if 0 <= v < vocab}
            for v, z in last.items():
                x[b, v] += z
        if mask is not None:
            x[b] = np.where(mask[b], x[b], -np.inf)
    return x
