"""The paged 8-bit cache by the words of include/b200_kv8.h, in numpy and 64 bits, page by page and head by head."""
import numpy as np


class Pool:
    """A layer's pages: ints k, v [n_pages][heads][page][size], scales f32, and the bytes of a record."""

    def __init__(self, n_pages, page, heads, dim, vdim, seed=0):
        self.n_pages, self.page, self.heads, self.dim, self.vdim = n_pages, page, heads, dim, vdim
        self.bytes = -(-(heads * page * (dim + vdim) + 8 * heads) // 128) * 128
        rng = np.random.default_rng(seed)
        self.raw = rng.integers(0, 256, (n_pages, self.bytes), dtype=np.uint8)  # padding too: nobody may touch it
        nk, nv = heads * page * dim, heads * page * vdim
        self.at = nk, nk + nv
        self.put(np.clip(np.round(rng.standard_normal((n_pages, heads, page, dim)) * 40), -127, 127), np.clip(np.round(rng.standard_normal((n_pages, heads, page, vdim)) * 40), -127, 127),
                 np.exp(0.4 * rng.standard_normal((n_pages, heads))) * 0.02, np.exp(0.4 * rng.standard_normal((n_pages, heads))) * 0.02)

    def put(self, k, v, ks, vs):
        self.k, self.v = k.astype(np.int8), v.astype(np.int8)
        self.ks, self.vs = ks.astype(np.float32), vs.astype(np.float32)

    def records(self):
        out = self.raw.copy()
        n, (a, b) = self.n_pages, self.at
        out[:, :a] = self.k.reshape(n, -1).view(np.uint8)
        out[:, a:b] = self.v.reshape(n, -1).view(np.uint8)
        out[:, b:b + 4 * self.heads] = self.ks.view(np.uint8).reshape(n, -1)
        out[:, b + 4 * self.heads:b + 8 * self.heads] = self.vs.view(np.uint8).reshape(n, -1)
        return out

    # ------------------------------------------------------------------ store
    def _store(self, ints, scales, entries, x, held):
        m = x.shape[0]
        if m == 0:
            return
        for e in range(held // self.page, -(-(held + m) // self.page)):
            p = entries[e] if e < len(entries) else -1
            if not 0 <= p < self.n_pages:
                continue
            lo, hi = max(held, e * self.page), min(held + m, (e + 1) * self.page)
            used = lo - e * self.page
            for h in range(self.heads):
                part = x[lo - held:hi - held, h].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    loud = np.abs(part).max()
                old = scales[p, h] if used else np.float32(0)
                if not np.isfinite(loud) or not np.isfinite(old):
                    scales[p, h] = np.nan
                    ints[p, h, used:used + hi - lo] = 0
                    continue
                want = np.float32(loud / 127)
                if want < 2.0 ** -126:
                    want = np.float32(0)
                if used == 0:
                    now = want
                elif want <= old:
                    now = old
                else:
                    now = max(want, np.float32(1.25 * np.float64(old)))
                if used and now != old:
                    ints[p, h, :used] = np.round(ints[p, h, :used].astype(np.float64) * np.float64(old) / np.float64(now))
                scales[p, h] = now
                ints[p, h, used:used + hi - lo] = np.clip(np.round(part / np.float64(now)), -127, 127) if now > 0 else 0

    def store(self, entries, k, v, held):
        """New rows k [m][heads][dim], v of the sequence whose pages are `entries`, which held `held` tokens."""
        self._store(self.k, self.ks, entries, k, held)
        self._store(self.v, self.vs, entries, v, held)

    # ------------------------------------------------------------------ reading
    def rows(self, entries, n, which):
        """Values of the first n tokens, 64 bits [n][heads][size]; and which tokens have a page."""
        ints, scales, size = (self.k, self.ks, self.dim) if which == "k" else (self.v, self.vs, self.vdim)
        out, there = np.zeros((n, self.heads, size)), np.zeros(n, bool)
        for e in range(-(-n // self.page)):
            p = entries[e] if e < len(entries) else -1
            if 0 <= p < self.n_pages:
                hi = min(n, (e + 1) * self.page) - e * self.page
                out[e * self.page:e * self.page + hi] = (ints[p].astype(np.float64) * scales[p].astype(np.float64)[:, None, None])[:, :hi].transpose(1, 0, 2)
                there[e * self.page:e * self.page + hi] = True
        return out, there

    def attend(self, entries, q, held, scale, window=0, keep=0, sink=None, softcap=0.0):
        """q [m][n_head][dim] at positions held ..: results [m][n_head][vdim]; and for bounds sum_j p_j |v_j| and max_j scale sum_d |q_d k_jd| over what a
        query sees."""
        m, n_head, _ = q.shape
        n = held + m
        k, there = self.rows(entries, n, "k")
        v, _ = self.rows(entries, n, "v")
        pos, key = held + np.arange(m)[:, None], np.arange(n)[None]
        sees = (key <= pos) & there
        if window:
            sees &= (pos - key < window) | (key < keep)
        out, mass, size = np.zeros((m, n_head, self.vdim)), np.zeros((m, n_head, self.vdim)), np.zeros((m, n_head))
        for h in range(n_head):
            g = h // (n_head // self.heads)
            qh, kk, vv = q[:, h].astype(np.float64), k[:, g], v[:, g]
            with np.errstate(invalid="ignore", over="ignore"):
                s = qh @ np.where(there[:, None], kk, 0.0).T * scale
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                s = np.where(sees, s, -np.inf)
                top = s.max(axis=1) if n else np.full(m, -np.inf)
                if sink is not None:
                    top = np.maximum(top, sink[h])
                top = np.where(top == -np.inf, 0.0, top)
                p = np.where(sees, np.exp(s - top[:, None]), 0.0)
                total = p.sum(axis=1) + (np.exp(sink[h] - top) if sink is not None else 0.0)
                p = p / np.where(total == 0, 1.0, total)[:, None]
                for i in range(m):  # only what a query sees takes part: elsewhere there may be NaN
                    out[i, h] = p[i, sees[i]] @ vv[sees[i]]
                    mass[i, h] = p[i, sees[i]] @ np.abs(vv[sees[i]])
                    size[i, h] = (np.abs(qh[i]) @ np.abs(kk[sees[i]]).T).max(initial=0.0) * abs(scale)
        return out, mass, size


class Pages:
    """Tables, lengths and counts of holders, and the four calls that change them."""

    def __init__(self, n_rows, stride, n_pages, page):
        self.table = np.full((n_rows, stride), -1, np.int32)
        self.len, self.refs = np.zeros(n_rows, np.int32), np.zeros(n_pages, np.int32)
        self.n_rows, self.stride, self.n_pages, self.page = n_rows, stride, n_pages, page

    def cover(self, tokens):
        return -(-int(tokens) // self.page)

    def cut(self, rows, keep):
        for i, r in enumerate(rows):
            if not 0 <= r < self.n_rows or r in rows[:i]:
                continue
            left = min(int(self.len[r]), max(0, int(keep[i])) if keep is not None else 0)
            for e in range(self.cover(left), self.cover(self.len[r])):
                if self.table[r, e] >= 0:
                    self.refs[self.table[r, e]] -= 1
                self.table[r, e] = -1
            self.len[r] = left

    def fork(self, src, dst):
        refused = 0
        had = self.len.copy()
        for i, (a, b) in enumerate(zip(src, dst)):
            if not (0 <= a < self.n_rows and 0 <= b < self.n_rows) or b in dst[:i] or a in dst or had[b]:
                refused += 1
                continue
            n = self.cover(self.len[a])
            for p in self.table[a, :n]:
                if p >= 0:
                    self.refs[p] += 1
            self.table[b, :n] = self.table[a, :n]
            self.len[b] = self.len[a]
        return refused

    def grow(self, rows, new):
        """(seq_info, refused, copies)"""
        n, plan, before = len(rows), [], 0
        refs0 = self.refs.copy()
        free = [p for p in range(self.n_pages) if refs0[p] == 0]
        for i, (r, m) in enumerate(zip(rows, new)):
            ok = 0 <= r < self.n_rows and m >= 0 and r not in rows[:i]
            held = int(self.len[r]) if ok else 0
            ok = ok and held + m <= min(self.stride * self.page, 2 ** 31 - 1)
            tail = -1
            if ok and m > 0 and held % self.page:
                p = self.table[r, held // self.page]
                tail = p if p >= 0 and refs0[p] > 1 else -1
            need = self.cover(held + m) - self.cover(held) + (tail >= 0) if ok else 0
            plan.append([ok, held, tail, need, before])
            before += need
        info, refused, copies, first = np.zeros((4, n), np.int32), 0, [], 0
        for i, (r, m) in enumerate(zip(rows, new)):
            ok, held, tail, need, start = plan[i]
            info[0, i], info[2, i], info[3, i] = first, r, held
            first += max(0, int(m))
            if not ok or (need and start + need > len(free)):
                refused += 1
                continue
            info[1, i] = m
            got = free[start:start + need]
            if tail >= 0:
                copies.append((tail, got[0]))
                self.refs[tail] -= 1
                self.table[r, held // self.page] = got[0]
                self.refs[got[0]] = 1
                got = got[1:]
            for e, p in enumerate(got):
                self.table[r, self.cover(held) + e] = p
                self.refs[p] = 1
            self.len[r] = held + m
        return info, refused, copies

    def compact(self):
        """(live pages, moves)"""
        live = [p for p in range(self.n_pages) if self.refs[p] > 0]
        n = len(live)
        moves = list(zip([p for p in live if p >= n], [p for p in range(n) if self.refs[p] <= 0]))
        for a, b in moves:
            self.table[self.table == a] = b
            self.refs[b], self.refs[a] = self.refs[a], 0
        return n, moves
