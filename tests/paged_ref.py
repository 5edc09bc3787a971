"""The paged cache in plain Python, and attention over it in 64 bits.

`Model` keeps what g4hip.h says of a cache (table, lengths, refs, contents) and does the
bookkeeping calls on it one list entry at a time; the tests compare the library's
device tensors with it exactly."""
import numpy as np
import torch


class Model:
    def __init__(self, cache):
        """A copy of a cache's device state."""
        self.page, self.pages = cache.page_tokens, cache.n_pages
        self.k, self.v = cache.k.cpu().clone(), cache.v.cpu().clone()
        self.table = cache.table.cpu().numpy().copy()
        self.lengths = cache.lengths.cpu().numpy().copy()
        self.refs = cache.refs.cpu().numpy().copy()

    def same_books(self, cache):
        assert int(cache.status_word.cpu()[0]) == 0
        assert np.array_equal(cache.lengths.cpu().numpy(), self.lengths)
        assert np.array_equal(cache.table.cpu().numpy(), self.table)
        assert np.array_equal(cache.refs.cpu().numpy(), self.refs)

    def same_contents(self, cache):
        """Bit for bit, pages of no sequence included."""
        for mine, theirs in ((self.k, cache.k), (self.v, cache.v)):
            a, b = (t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)
                    for t in (mine, theirs.cpu()))
            assert torch.equal(a, b)

    def used(self, n):
        return -(-n // self.page)

    def free_pages(self):
        return [p for p in range(self.pages) if self.refs[p] == 0]

    def extend(self, seqs, counts):
        free = iter(self.free_pages())
        for s, c in zip(seqs, counts):
            for j in range(self.used(self.lengths[s]), self.used(self.lengths[s] + c)):
                self.table[s, j] = next(free)
                self.refs[self.table[s, j]] = 1
            self.lengths[s] += c

    def move(self, src, dst, prefix, keep):
        """fork (keep None) and compact."""
        free = iter(self.free_pages())
        table, lengths, refs = self.table.copy(), self.lengths.copy(), self.refs.copy()
        k, v = self.k.clone(), self.v.clone()
        rows = []
        for i, (s, d) in enumerate(zip(src, dst)):
            n = lengths[s] if prefix is None and keep is None else 0 if prefix is None else prefix[i]
            tokens = [] if keep is None else list(keep[i])
            shared = n // self.page
            if n % self.page and s == d and not tokens and refs[table[s, shared]] == 1:
                shared += 1
            row = list(table[s, :shared])
            old = list(range(shared * self.page, n)) + tokens
            for at in range(0, len(old), self.page):
                p = next(free)
                row.append(p)
                for y, t in enumerate(old[at:at + self.page]):
                    for mine, was in ((self.k, k), (self.v, v)):
                        mine[:, p, :, y] = was[:, table[s, t // self.page], :, t % self.page]
            rows.append((d, row, n + len(tokens)))
        for d, row, n in rows:
            for p in table[d]:
                if p >= 0:
                    self.refs[p] -= 1
            for p in row:
                if p >= 0:
                    self.refs[p] += 1
            self.table[d] = row + [-1] * (self.table.shape[1] - len(row))
            self.lengths[d] = n

    def release(self, seqs, first=None, window=None):
        for s in seqs:
            n = int(self.lengths[s])
            for j in range(self.used(n)):
                if window is None or (j * self.page >= first and (j + 1) * self.page - 1 <= n - window):
                    if self.table[s, j] >= 0:
                        self.refs[self.table[s, j]] -= 1
                    self.table[s, j] = -1
            if window is None:
                self.lengths[s] = 0

    def write(self, layer, seq, pos, k, v):
        p, y = self.table[seq, pos // self.page], pos % self.page
        self.k[layer, p, :, y] = k.to(self.k.dtype)
        self.v[layer, p, :, y] = v.to(self.v.dtype)

    def rows(self, layer, seq, upto):
        """Keys and values of tokens 0 .. upto - 1 in float64 [tokens, kv heads, head size], and which are there."""
        t = np.arange(upto)
        p = self.table[seq, t // self.page] if upto else np.zeros(0, np.int64)
        there = (p >= 0) & (p < self.pages)
        at, y = torch.from_numpy(np.where(there, p, 0).astype(np.int64)), torch.from_numpy(t % self.page)
        return self.k[layer, at, :, y].double(), self.v[layer, at, :, y].double(), there


def attend(model, layer, q, seq, pos, scale, window, sinks):
    """(out, bound) of one row [heads, head size] at `pos` in 64 bits.  bound: the sum of
    w |v| times (1 + 2 max_t sum |scale q k|), what a relative error of every product
    moves the result by at most (weights move by at most twice their scores' error)."""
    heads, hs = q.shape
    q = q.double()
    out, bound = torch.zeros(heads, hs, dtype=torch.float64), torch.zeros(heads, hs, dtype=torch.float64)
    k, v, there = model.rows(layer, seq, pos + 1)
    t = np.arange(pos + 1)
    see = there.copy()
    if window:
        see &= (t > pos - window) | (t < sinks)
    if not see.any():
        return out, bound
    see = torch.from_numpy(see)
    k, v = k[see], v[see]
    group = heads // k.shape[1]
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = kh @ q[h] * scale
        w = torch.softmax(s, 0)
        out[h] = w @ vh
        bound[h] = w @ vh.abs() * (1 + 2 * float((kh.abs() @ q[h].abs()).max() * abs(scale)))
    return out, bound
