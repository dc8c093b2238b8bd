"""A plain model of the paged 8-bit cache for the tests: numpy on the host, one
token and one page at a time; attention in 64 bits."""
import numpy as np

F = np.float32
TINY = F(1e-30)


def quantise_block(old_codes, old_scale, x):
    """A block's codes [tokens, d] and scale after rows x (f32) follow old_codes:
    s = max(s0, amax * (1 / 127)), code = rint(x * (1 / s)); older codes rint(code * (s0 / s))."""
    mag = np.where(np.isfinite(x), np.abs(x), F(0))
    a = F(mag.max()) if mag.size else F(0)
    s0 = F(old_scale) if len(old_codes) else F(0)
    s = max(s0, F(a * (F(1) / F(127))) if a >= TINY else F(0))
    if len(old_codes) and s > s0:
        old_codes = np.rint(old_codes.astype(F) * F(s0 / s)).astype(np.int8)
    with np.errstate(invalid="ignore", over="ignore"):
        r = np.rint(x * (F(1) / s if s > 0 else F(0)))
    new = np.clip(np.nan_to_num(r, nan=0.0, posinf=127, neginf=-127), -127, 127).astype(np.int8)
    return np.concatenate([old_codes, new]), s


class RefCache:
    def __init__(self, n_layers, n_pages, kv, d, n_seqs, max_pages, page, block):
        self.kv, self.d, self.page, self.block = kv, d, page, block
        self.n_layers, self.n_pages, self.n_seqs, self.max_pages = n_layers, n_pages, n_seqs, max_pages
        self.codes = np.zeros((2, n_layers, n_pages, kv, page, d), np.int8)
        self.scale = np.zeros((2, n_layers, n_pages, kv, page // block), F)
        self.table = np.full((n_seqs, max_pages), -1, np.int32)
        self.length = np.zeros(n_seqs, np.int32)
        self.refs = np.zeros(n_pages, np.int32)

    # ---- pages ----
    def _np(self, n):
        return -(-int(n) // self.page)

    def _free(self):
        return list(np.nonzero(self.refs == 0)[0])

    def reserve(self, seqs, counts):
        """True if it could be served."""
        need = [self._np(self.length[s] + c) - self._np(self.length[s]) for s, c in zip(seqs, counts)]
        if any(self.length[s] + c > self.max_pages * self.page for s, c in zip(seqs, counts)):
            return False
        free = self._free()
        if sum(need) > len(free):
            return False
        for s, c, n in zip(seqs, counts, need):
            at = self._np(self.length[s])
            for j in range(n):
                p = free.pop(0)
                self.table[s, at + j] = p
                self.refs[p] = 1
            self.length[s] += c
        return True

    def fork(self, parents, children):
        old, length = self.table.copy(), self.length.copy()
        free = self._free()
        need = [p != c and length[p] % self.page != 0 and old[p, length[p] // self.page] >= 0
                for p, c in zip(parents, children)]
        if sum(need) > len(free):
            return False
        for p, c, fresh in zip(parents, children, need):
            for e in self.table[c]:
                if e >= 0:
                    self.refs[e] -= 1
        for p, c, fresh in zip(parents, children, need):
            row = np.full(self.max_pages, -1, np.int32)
            row[:self._np(length[p])] = old[p, :self._np(length[p])]
            if fresh:
                q = free.pop(0)
                last = self._np(length[p]) - 1
                u = length[p] % self.page
                nb = -(-u // self.block)
                self.codes[:, :, q, :, :u] = self.codes[:, :, row[last], :, :u]
                self.scale[:, :, q, :, :nb] = self.scale[:, :, row[last], :, :nb]
                row[last] = q
            for e in row:
                if e >= 0:
                    self.refs[e] += 1
            self.table[c], self.length[c] = row, length[p]
        return True

    def release(self, seqs):
        for s in seqs:
            for j in range(self.max_pages):
                if self.table[s, j] >= 0:
                    self.refs[self.table[s, j]] -= 1
                self.table[s, j] = -1
            self.length[s] = 0

    def slide(self, window, sinks, seqs):
        for s in seqs:
            for j in range(self.max_pages):
                if (j + 1) * self.page <= self.length[s] - window and j * self.page >= sinks and self.table[s, j] >= 0:
                    self.refs[self.table[s, j]] -= 1
                    self.table[s, j] = -1

    def compact(self):
        live = int((self.refs > 0).sum())
        src = [p for p in range(live, self.n_pages) if self.refs[p] > 0]
        dst = [p for p in range(live) if self.refs[p] == 0]
        for a, b in zip(src, dst):
            self.table[self.table == a] = b
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.codes[:, :, b], self.scale[:, :, b] = self.codes[:, :, a], self.scale[:, :, a]

    # ---- rows ----
    def append(self, layer, seqs, rows_k, rows_v):
        """rows_k[i], rows_v[i]: f32 [n_i, kv, d], the last tokens of sequence seqs[i]."""
        for s, *rows in zip(seqs, rows_k, rows_v):
            for z, x in enumerate(rows):
                first = int(self.length[s]) - len(x)
                if first < 0:
                    x, first = x[-first:], 0
                t = first
                while t < self.length[s]:
                    b0 = t // self.block * self.block
                    end = min(b0 + self.block, int(self.length[s]))
                    p, slot, b = self.table[s, t // self.page], b0 % self.page, b0 % self.page // self.block
                    for h in range(self.kv):
                        c, sc = quantise_block(self.codes[z, layer, p, h, slot:slot + t - b0],
                                               self.scale[z, layer, p, h, b], x[t - first:end - first, h])
                        self.codes[z, layer, p, h, slot:slot + end - b0] = c
                        self.scale[z, layer, p, h, b] = sc
                    t = end

    def values(self, layer, s, z):
        """f64 [length, kv, d]; tokens without a page: NaN."""
        n = int(self.length[s])
        out = np.full((n, self.kv, self.d), np.nan)
        for t in range(n):
            p = self.table[s, t // self.page]
            if p >= 0:
                sc = self.scale[z, layer, p, :, t % self.page // self.block].astype(np.float64)
                out[t] = self.codes[z, layer, p, :, t % self.page].astype(np.float64) * sc[:, None]
        return out

    def attend(self, layer, s, q, scale, window=0, sinks=0):
        """q f64 [n, heads, d], the last tokens of s: (out, lse, bound), where bound [n, heads] holds
        sum_d |q k| of the row's largest key times scale and the largest |v| it sees."""
        k, v = self.values(layer, s, 0), self.values(layer, s, 1)
        n, heads = q.shape[:2]
        g = heads // self.kv
        out, lse = np.zeros((n, heads, self.d)), np.full((n, heads), -np.inf)
        size, top = np.zeros((n, heads)), np.zeros((n, heads))
        t = np.arange(len(k))
        held = ~np.isnan(k[:, 0, 0]) if len(k) else np.zeros(0, bool)
        for i in range(n):
            p = int(self.length[s]) - n + i
            see = held & (t <= p)
            if window:
                see &= (t > p - window) | (t < sinks)
            idx = np.nonzero(see)[0]
            if not len(idx):
                continue
            for h in range(heads):
                w = k[idx, h // g] @ q[i, h] * scale
                m = w.max()
                e = np.exp(w - m)
                lse[i, h] = m + np.log(e.sum())
                out[i, h] = (e / e.sum()) @ v[idx, h // g]
                size[i, h] = (np.abs(k[idx, h // g]) @ np.abs(q[i, h])).max() * abs(scale)
                top[i, h] = np.abs(v[idx, h // g]).max()
        return out, lse, size, top
