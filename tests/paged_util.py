"""Paged-cache inputs, attention in 64 bits on the CPU with its error bound, and a model of the page bookkeeping in plain
Python: what the paged-cache tests compare the library with."""
import math

import numpy as np

U32 = 2 ** 32 - 1


def ceil_div(a, b):
    return -(-a // b)


def make_case(seed, lens, n_new, n_q, n_kv, hd, page, f16, spare=3, q_gain=1.5, garbage=np.nan):
    """lens: tokens each sequence holds, n_new: how many of them are this call's rows.  Pages in random order, cache rows
    that nobody holds full of `garbage`, table entries that nobody needs out of range."""
    r = np.random.default_rng([77, seed])
    counts = [ceil_div(n, page) for n in lens]
    n_pages = sum(counts) + spare
    order = r.permutation(n_pages)
    width = max(counts + [0]) + 2
    table = np.full((len(lens), width), -1, np.int32)
    K = np.full((n_pages * page, n_kv * hd), garbage, np.float16)
    V = K.copy()
    at = 0
    for s, (c, n) in enumerate(zip(counts, lens)):
        table[s, :c] = order[at:at + c]
        at += c
        rows = slots_of(table[s], n, page)
        K[rows] = r.standard_normal((n, n_kv * hd)).astype(np.float16)
        V[rows] = r.standard_normal((n, n_kv * hd)).astype(np.float16)
    q_off = np.concatenate([[0], np.cumsum(n_new)]).astype(np.int32)
    q = (r.standard_normal((int(q_off[-1]), n_q * hd)) * q_gain).astype(np.float16 if f16 else np.float32)
    return dict(q=q, K=K, V=V, table=table, kv_len=np.array(lens, np.int32), q_off=q_off, page=page, n_q=n_q, n_kv=n_kv, hd=hd, n_pages=n_pages)


def slots_of(table_row, n, page):
    j = np.arange(n)
    return table_row[j // page].astype(np.int64) * page + j % page


def attention64(c, scale, window=0):
    """(out, tol) in float64.  tol bounds the distance of a result computed as the library documents it, from rounding
    errors alone.  With A = sum_j w_j |v_j| (w the softmax weights), u16 = 2^-11 and u32 = 2^-24 the half steps of fp16 and f32:
      a score carries hd + 8 roundings of f32 sums and products, and for f32 queries 2^-22 of every product (an f32 query
      is held in 22 bits), each relative to scale * sum |q||k|; a score error e moves a weight by the factor e;
      exp2 of the hardware and the scaling of its argument (of magnitude up to |x|): 2^-21 + 4 |x| u32;
      a weight is rounded to u16 (fp16 rows) or 2^-22 (f32 rows); the two sums over n keys: n u32 each, and the sums of the
      parts: below 2^-20 together;
      the result is rounded once: u16 or u32 of it, and half the smallest subnormal step of fp16.
    Weight errors come in twice, through the sum of the values and through the sum of the weights."""
    hd, g, page = c["hd"], c["n_q"] // c["n_kv"], c["page"]
    f16 = c["q"].dtype == np.float16
    q = c["q"].astype(np.float64)
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(len(c["kv_len"])):
        n, a, b = int(c["kv_len"][s]), int(c["q_off"][s]), int(c["q_off"][s + 1])
        rows = slots_of(c["table"][s], n, page)
        k, v = c["K"][rows].astype(np.float64), c["V"][rows].astype(np.float64)
        for r in range(a, b):
            p = n - (b - a) + (r - a)
            lo = max(0, p - window + 1) if window else 0
            if p < 0:
                continue
            for h in range(c["n_q"]):
                sl = slice((h // g) * hd, (h // g + 1) * hd)
                qq, kk, vv = q[r, h * hd:(h + 1) * hd], k[lo:p + 1, sl], v[lo:p + 1, sl]
                x = scale * (kk @ qq)
                w = np.exp(x - x.max())
                w /= w.sum()
                o = w @ vv
                A = w @ np.abs(vv)
                eps = abs(scale) * (np.abs(kk) @ np.abs(qq)).max() * ((hd + 8) * 2.0 ** -24 + (0 if f16 else 2.0 ** -22))
                eps += 2.0 ** -21 + 4 * np.abs(x).max() * 2.0 ** -24 + (p + 1 - lo) * 2.0 ** -24 + 2.0 ** -20
                u_p, u_o = (2.0 ** -11, 2.0 ** -11) if f16 else (2.0 ** -22, 2.0 ** -24)
                out[r, h * hd:(h + 1) * hd] = o
                tol[r, h * hd:(h + 1) * hd] = A * (u_p + 2 * eps) + u_o * np.abs(o) + (2.0 ** -25 if f16 else 2.0 ** -149)
    return out, tol


class PageModel:
    """The bookkeeping of the pages as the header describes it, one sequence after the other."""

    def __init__(self, n_pages, page, n_seq, max_pages):
        self.n_pages, self.page, self.n_seq, self.max_pages = n_pages, page, n_seq, max_pages
        self.refs = [0] * n_pages
        self.table = [[] for _ in range(n_seq)]
        self.kv_len = [0] * n_seq

    def free(self):
        return [p for p in range(self.n_pages) if not self.refs[p]]

    def extend(self, n_new, rows):
        """None: refused; else (q_off, positions, slots, pairs)"""
        P = self.page
        free, pairs, grown = self.free(), [], []
        refs = list(self.refs)
        sharers = {}
        for s, new in enumerate(n_new):
            if new and self.kv_len[s] % P and self.refs[self.table[s][-1]] > 1:
                sharers.setdefault(self.table[s][-1], []).append(s)
        for s, new in enumerate(n_new):
            t = list(self.table[s])
            if new and self.kv_len[s] % P and self.refs[t[-1]] > 1:
                old = t[-1]
                if not (len(sharers[old]) == self.refs[old] and sharers[old][-1] == s):
                    if not free:
                        return None
                    t[-1] = free.pop(0)
                    refs[t[-1]] = 1
                    refs[old] -= 1
                    pairs.append((t[-1], old))
            while len(t) < ceil_div(self.kv_len[s] + new, P):
                if not free:
                    return None
                t.append(free.pop(0))
                refs[t[-1]] = 1
            if len(t) > self.max_pages:
                return None
            grown.append(t)
        if sum(n_new) > rows:
            return None
        self.refs, self.table = refs, grown
        q_off, positions, slots = [0], [], []
        for s, new in enumerate(n_new):
            for j in range(self.kv_len[s], self.kv_len[s] + new):
                positions.append(j)
                slots.append(self.table[s][j // P] * P + j % P)
            self.kv_len[s] += new
            q_off.append(q_off[-1] + new)
        return q_off, positions, slots, pairs

    def fork(self, src, dst):
        """True where a pair was left out"""
        lens, tables, bad, named = list(self.kv_len), [list(t) for t in self.table], False, set()
        for a, b in zip(src, dst):
            if not (0 <= a < self.n_seq and 0 <= b < self.n_seq) or a == b or b in named or lens[b]:
                bad = True
            else:
                self.table[b], self.kv_len[b] = list(tables[a]), lens[a]
                for p in tables[a]:
                    self.refs[p] += 1
            named.add(b)
        return bad

    def truncate(self, new_len):
        for s, n in enumerate(new_len):
            if n < self.kv_len[s]:
                keep = ceil_div(n, self.page)
                for p in self.table[s][keep:]:
                    self.refs[p] -= 1
                self.table[s], self.kv_len[s] = self.table[s][:keep], n

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if not self.refs[p]]
        strays = [p for p in range(live, self.n_pages) if self.refs[p]]
        name = dict(zip(strays, holes))
        for a, b in name.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[name.get(p, p) for p in t] for t in self.table]
        return list(zip(holes, strays))
