"""A paged cache on the device for tests, and the operators on it from their definitions in 64 bits."""
from __future__ import annotations

import numpy as np

from cera_amd import hip_api as A

SENTINEL = np.float32(-12345.5)


class Pool:
    """Sequences in pages of a pool whose other slots hold NaN.  k, v: per sequence [len][n_kv][hd] as the cache holds them."""

    def __init__(self, hip, lens, n_kv, hd, f16=True, page=16, seed=0, max_pages=None, interleaved=False, fill=np.nan, spare=2, k=None, v=None):
        r = np.random.default_rng(seed)
        self.hip, self.lens, self.n_kv, self.hd, self.page, self.f16 = hip, list(lens), n_kv, hd, page, f16
        self.dtype = np.float16 if f16 else np.float32
        need = [-(-n // page) for n in lens]
        self.cols = max_pages or max(need + [1])
        self.n_pages = sum(need) + spare
        order = list(r.permutation(self.n_pages))
        self.table = np.full((len(lens), self.cols), -7, np.int32)      # entries behind a sequence's pages are no page numbers
        for s, c in enumerate(need):
            self.table[s, :c] = [order.pop() for _ in range(c)]
        self.k = k or [r.standard_normal((n, n_kv, hd)).astype(self.dtype) for n in lens]
        self.v = v or [r.standard_normal((n, n_kv, hd)).astype(self.dtype) for n in lens]
        both = np.full((self.n_pages, 2, n_kv, page, hd), fill, self.dtype)
        for s, n in enumerate(lens):
            for t in range(n):
                both[self.table[s, t // page], 0, :, t % page] = self.k[s][t]
                both[self.table[s, t // page], 1, :, t % page] = self.v[s][t]
        self.per_page = n_kv * page * hd
        self.bufs = []
        if interleaved:      # a page's values behind its keys
            base = self.dev(both)
            self.dk, self.dv, self.stride = base, base + self.per_page * self.dtype().itemsize, 2 * self.per_page
        else:
            self.dk, self.dv, self.stride = self.dev(both[:, 0]), self.dev(both[:, 1]), 0
        self.interleaved = interleaved
        self.d_table, self.d_lens = self.dev(self.table), self.dev(np.array(lens, np.uint32))

    def dev(self, a):
        p = self.hip.to_device(np.ascontiguousarray(a))
        self.bufs.append(p)
        return p

    def kv(self, **more):
        f = dict(kv_type=int(self.f16), n_kv_heads=self.n_kv, head_dim=self.hd, page_size=self.page, n_pages=self.n_pages, n_seqs=len(self.lens),
                 max_pages=self.cols, page_stride=self.stride, k=self.dk, v=self.dv, table=self.d_table, lens=self.d_lens)
        f.update(more)
        return A.PagedKV(**f)

    def pages(self):
        """(k, v) of the pool: [n_pages][n_kv][page][hd]."""
        shape = (self.n_pages, self.n_kv, self.page, self.hd)
        if self.interleaved:
            both = self.hip.download(self.dk, (self.n_pages, 2) + shape[1:], self.dtype)
            return both[:, 0], both[:, 1]
        return self.hip.download(self.dk, shape, self.dtype), self.hip.download(self.dv, shape, self.dtype)

    def rows(self, s, n):
        """(k, v) of sequence s's first n positions as they lie in the pool."""
        k, v = self.pages()
        at = [(self.table[s, t // self.page], t % self.page) for t in range(n)]
        return tuple(np.stack([x[p, :, o] for p, o in at]) if n else np.zeros((0, self.n_kv, self.hd), self.dtype) for x in (k, v))

    def close(self):
        for b in self.bufs:
            self.hip.free(b)
        self.bufs = []


def seen(P, window, sinks):
    t = np.arange(P + 1)
    return t[(t < sinks) | (window == 0) | (t > P - window)]


def attn_ref(q, k, v, n_new, scale, window, sinks):
    """q [n_new][heads][hd]; k, v [len][n_kv][hd].  (out, bound of a kernel's error, weights [n_kv][len] of the rows).

    The bound: K and V enter as they are.  A query's value is held in two halves of 11 bits (2^-20 relative at most, with the
    discarded products), a score sums hd products in f32 (2^-24 for each): |ds| <= (2^-20 + hd 2^-24) scale sum |q k|.  A weight's
    relative error is at most 2 |ds| (itself and the sum of all) plus its own rounding to two halves and the exponential's, 2^-20;
    a sum of n weights, and of n weighted values, adds n 2^-24."""
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    n, heads, G = k.shape[0], q.shape[1], q.shape[1] // k.shape[1]
    out, bound, mass = np.zeros_like(q), np.zeros_like(q), np.zeros((k.shape[1], n))
    mass_bound = np.zeros_like(mass)
    for i in range(n_new):
        ids = seen(n - n_new + i, window, sinks)
        if not len(ids):
            continue
        for h in range(heads):
            kk, vv = k[ids, h // G], v[ids, h // G]
            s = kk @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vv
            ds = (2.0 ** -20 + q.shape[2] * 2.0 ** -24) * abs(scale) * (np.abs(kk) @ np.abs(q[i, h])).max()
            rel = np.expm1(2 * ds) + 2.0 ** -20 + len(ids) * 2.0 ** -24
            bound[i, h] = rel * (p @ np.abs(vv)) + 1e-30
            mass[h // G, ids] += p
            mass_bound[h // G, ids] += rel * p
    return out, bound, mass, mass_bound


class Rows:
    """Device rows of q, out and the new keys and values, dense or with strides, guard values around what is written."""

    def __init__(self, pool, n_rows, heads, seed, pad=0, new=False, extra=2):
        r = np.random.default_rng(seed + 1000)
        self.pool, self.heads, self.n = pool, heads, n_rows
        hd, kvd = pool.hd, pool.n_kv * pool.hd
        self.q = (r.standard_normal((n_rows, heads, hd)) * 1.5).astype(np.float32)
        self.qs, self.ks, self.os = heads * hd + pad, kvd + pad, heads * hd + 2 * pad
        qb = np.full((n_rows, self.qs), np.nan, np.float32)
        qb[:, :heads * hd] = self.q.reshape(n_rows, -1)
        self.d_q = pool.dev(qb)
        self.extra = extra
        self.d_out = pool.dev(np.full((n_rows + extra, self.os), SENTINEL, np.float32))
        self.k_new = r.standard_normal((n_rows, pool.n_kv, hd)).astype(np.float32) if new else None
        self.v_new = r.standard_normal((n_rows, pool.n_kv, hd)).astype(np.float32) if new else None
        self.d_kn = self.d_vn = None
        if new:
            kb, vb = np.full((n_rows, self.ks), np.nan, np.float32), np.full((n_rows, self.ks), np.nan, np.float32)
            kb[:, :kvd], vb[:, :kvd] = self.k_new.reshape(n_rows, -1), self.v_new.reshape(n_rows, -1)
            self.d_kn, self.d_vn = pool.dev(kb), pool.dev(vb)

    def op(self, **more):
        f = dict(q=self.d_q, k_new=self.d_kn, v_new=self.d_vn, out=self.d_out, q_stride=self.qs, kv_stride=self.ks, out_stride=self.os, n_rows=self.n,
                 n_heads=self.heads, scale=1 / np.sqrt(self.pool.hd))
        f.update(more)
        return A.PagedAttn(**f)

    def result(self):
        """out [n_rows][heads][hd], after a look at the guard values."""
        o = self.pool.hip.download(self.d_out, (self.n + self.extra, self.os), np.float32)
        w = self.heads * self.pool.hd
        assert (o[:, w:] == SENTINEL).all() and (o[self.n:] == SENTINEL).all()
        return o[:self.n, :w].reshape(self.n, self.heads, self.pool.hd)
