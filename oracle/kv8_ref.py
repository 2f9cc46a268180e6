"""Plain restatement of the 8-bit paged K/V cache (aion_kv8_* of include/aion.h)
on the CPU: NumPy, 64-bit sums, one sequence and one page at a time.  Only
tests use it."""
from __future__ import annotations

import numpy as np

F = np.float32


class Cache:
    """State and calls under the library's names; every list is a plain list."""

    def __init__(self, n_layers, n_pages, n_kv, hd, max_seqs, max_pages, page):
        self.k = np.zeros((n_layers, n_pages, n_kv, page, hd), np.int8)
        self.v = np.zeros_like(self.k)
        self.k_scale = np.zeros((n_layers, n_pages, n_kv), F)
        self.v_scale = np.zeros_like(self.k_scale)
        self.tables = np.full((max_seqs, max_pages), -1, np.int32)
        self.lens = np.zeros(max_seqs, np.int32)
        self.refs = np.zeros(n_pages, np.int32)
        self.page = page
        self.status = set()

    def _ok(self, slot, seen):
        if not 0 <= slot < len(self.lens) or slot in seen:
            self.status.add("ARG")
            return False
        return True

    def _pages(self, tokens):
        return -(-int(tokens) // self.page)

    # -- pages ----------------------------------------------------------------
    def grow(self, seqs, n_new):
        seen, asked, plan = set(), 0, []
        free = [int(p) for p in np.flatnonzero(self.refs == 0)]
        shared = self.refs > 1
        for slot, n in zip(seqs, n_new):
            if not self._ok(slot, seen):
                plan.append(None)
                continue
            seen.add(slot)
            old = int(self.lens[slot])
            if n < 0 or old + n > self.tables.shape[1] * self.page:
                self.status.add("ARG")
                plan.append(None)
                continue
            have, want = self._pages(old), self._pages(old + n)
            copy = n > 0 and old % self.page > 0 and bool(shared[self.tables[slot, have - 1]])
            need = want - have + copy
            asked += need
            if need and asked > len(free):
                self.status.add("OOM")
                plan.append(None)
                continue
            plan.append((slot, n, old, have, want, copy, free[asked - need:asked]))
        pos0, moves = [], []
        for p in plan:
            if p is None:
                pos0.append(-1)
                continue
            slot, n, old, have, want, copy, pages = p
            if copy:
                moves.append((int(self.tables[slot, have - 1]), pages[0]))
                self.refs[moves[-1][0]] -= 1
                self.tables[slot, have - 1] = pages[0]
            self.tables[slot, have:want] = pages[copy:]
            self.refs[pages] = 1
            self.lens[slot] = old + n
            pos0.append(old)
        for s, d in moves:
            self._move(s, d)
        return pos0

    def _move(self, s, d):
        for a in (self.k, self.v, self.k_scale, self.v_scale):
            a[:, d] = a[:, s]

    def _drop(self, slot, keep):
        a, b = self._pages(keep), self._pages(self.lens[slot])
        for j in range(a, b):
            self.refs[self.tables[slot, j]] -= 1
            self.tables[slot, j] = -1
        self.lens[slot] = keep

    def trim(self, seqs, keep=None):
        seen = set()
        for i, slot in enumerate(seqs):
            n = 0 if keep is None else keep[i]
            if not self._ok(slot, seen):
                continue
            seen.add(slot)
            if n < 0:
                self.status.add("ARG")
                continue
            self._drop(slot, min(int(self.lens[slot]), n))

    def fork(self, src, dst, keep=None):
        seen = set()
        for i, (s, d) in enumerate(zip(src, dst)):
            n = 1 << 30 if keep is None else keep[i]
            bad = d in src or n < 0 or not 0 <= s < len(self.lens)
            if not self._ok(d, seen) or bad:
                self.status.add("ARG")
                seen.add(d)
                continue
            seen.add(d)
            self._drop(d, 0)
            n = min(int(self.lens[s]), n)
            used = self._pages(n)
            self.tables[d, :used] = self.tables[s, :used]
            self.refs[self.tables[s, :used]] += 1
            self.lens[d] = n

    def compact(self):
        used = self.refs > 0
        u = int(used.sum())
        src, dst = np.flatnonzero(used[u:]) + u, np.flatnonzero(~used[:u])
        for s, d in zip(src, dst):
            self._move(s, d)
            self.refs[d], self.refs[s] = self.refs[s], 0
            for slot in range(len(self.lens)):
                row = self.tables[slot, :self._pages(self.lens[slot])]
                row[row == s] = d
        return u

    # -- rows -----------------------------------------------------------------
    def append(self, layer, k, v, seqs, pos0, cu):
        seen = set()
        for i, slot in enumerate(seqs):
            n = cu[i + 1] - cu[i]
            if pos0[i] < 0 or n <= 0:
                continue
            if not self._ok(slot, seen):
                continue
            seen.add(slot)
            done = 0
            while done < n:
                pos = pos0[i] + done
                take = min(n - done, self.page - pos % self.page)
                pg = int(self.tables[slot, pos // self.page]) if pos // self.page < self.tables.shape[1] else -1
                if pg < 0 or self.refs[pg] != 1:
                    self.status.add("STATE")
                else:
                    at = slice(cu[i] + done, cu[i] + done + take)
                    for x, pool, scale in ((k, self.k, self.k_scale), (v, self.v, self.v_scale)):
                        self._write(pool[layer, pg], scale[layer, pg], x[at].astype(F), pos % self.page)
                done += take

    def _write(self, pool, scale, x, row):
        """pool [head][token][hd], scale [head]; x [token][head][hd] fp32."""
        for h in range(pool.shape[0]):
            top = np.abs(x[:, h]).max()
            need = F(np.float64(top) / 127) if np.isfinite(top) else F(np.nan)
            s0, s = scale[h], need
            if row:
                s = s0 if need <= s0 else F(np.nan) if np.isnan(need) or np.isnan(s0) else max(need, F(F(1.25) * s0))
                if not s == s0:
                    ratio = F(s0 / s) if s > 0 else F(0)
                    pool[h, :row] = np.rint(pool[h, :row].astype(F) * ratio).astype(np.int8)
            scale[h] = s
            with np.errstate(all="ignore"):
                q = np.rint(x[:, h].astype(np.float64) / np.float64(s)) if s > 0 else np.zeros_like(x[:, h])
            pool[h, row:row + len(x)] = np.clip(q, -127, 127).astype(np.int8)

    def rows(self, layer, slot, n):
        """The first n K and V rows of a slot in 64 bits: [n][head][hd] each."""
        pos = np.arange(n)
        pg = self.tables[slot, pos // self.page]
        return [pool[layer][pg, :, pos % self.page].astype(np.float64) * sc[layer][pg].astype(np.float64)[:, :, None]
                for pool, sc in ((self.k, self.k_scale), (self.v, self.v_scale))]

    def attention(self, layer, q, seqs, pos0, cu, scale=None):
        """(out, bound) in 64 bits; bound[row][head] = (max |q|, largest sum |k| of a
        position seen, largest |v|, positions seen): what tolerances are made of."""
        heads, hd = q.shape[1:]
        group = heads // self.k.shape[2]
        scale = 1 / np.sqrt(hd) if scale is None else scale
        out, info = np.zeros(q.shape), np.zeros((q.shape[0], heads, 4))
        for i, slot in enumerate(seqs):
            n = cu[i + 1] - cu[i]
            if pos0[i] < 0 or n <= 0:
                continue
            k, v = self.rows(layer, slot, pos0[i] + n)
            for r in range(n):
                seen = pos0[i] + r + 1
                for h in range(heads):
                    x, kk, vv = q[cu[i] + r, h].astype(np.float64), k[:seen, h // group], v[:seen, h // group]
                    s = kk @ x * scale
                    w = np.exp(s - s.max())
                    out[cu[i] + r, h] = w @ vv / w.sum()
                    info[cu[i] + r, h] = np.abs(x).max(), np.abs(kk).sum(1).max(), np.abs(vv).max(), seen
        return out, info
