"""Inputs of paged attention whose result tells every part of a number that the kernels hold in several.

Three positions have all the weight; the others' scores are 500 below, so that their weights are 0 and no sum rounds for them.  Queries
have five dims that are not 0 and values are positive, so the bound below is near 2^-18, where a part that is left out shows: a
half has 11 bits, two bfloat16 have 16."""
import numpy as np

DIMS = (2, 7, 33, 60)


def make(seed, lens, n_rows, heads, n_kv, hd, f16, last):
    """(k, v) of the sequences, q [n_rows][heads][hd]; the three positions lie before the last `last`."""
    r = np.random.default_rng(seed)
    dtype = np.float16 if f16 else np.float32
    k, v, where = [], [], []
    for n in lens:
        kk, vv = np.zeros((n, n_kv, hd)), 0.5 + r.random((n, n_kv, hd))
        kk[:, :, 0] = -4000
        ids = np.sort(r.choice(n - last, 3, replace=False))
        kk[ids] = 0
        kk[np.ix_(ids, range(n_kv), DIMS)] = r.standard_normal((3, n_kv, 4))
        k.append(kk.astype(dtype))
        v.append(vv.astype(dtype))
        where.append(ids)
    q = np.zeros((n_rows, heads, hd), np.float32)
    q[:, :, 0] = 1
    q[:, :, DIMS] = (0.3 + 0.6 * r.random((n_rows, heads, 4))) * r.choice([-1, 1], (n_rows, heads, 4))
    return k, v, q, where


def exact(q, k, v, ids, scale):
    """(out, relative bound) of rows q [n][heads][hd] over the three positions.

    A score: products of q and k off by 2^-21 at most (q, k and what is left out), five of them added.  A weight: its exponent, up to 16,
    is rounded by 2^-21 at most, times ln 2, and the exponential by 2^-22; both enter twice, over the value's and over the weights' sum.  Its
    parts and the value's: 2^-21.  Sums: 18 products at most, two joins of two roundings and an exponential each, the inverse: 26 times 2^-24
    and twice 2^-22."""
    G = q.shape[1] // k.shape[1]
    q, k, v = q.astype(np.float64), k[ids].astype(np.float64), v[ids].astype(np.float64)
    out, bound = np.zeros(q.shape), np.zeros(q.shape[:2])
    for h in range(q.shape[1]):
        s = q[:, h] @ k[:, h // G].T * scale
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h] = p @ v[:, h // G]
        size = scale * (np.abs(q[:, h]) @ np.abs(k[:, h // G]).T).max(1)
        bound[:, h] = 2 * (2.0 ** -21 + 5 * 2.0 ** -24) * size + 2 * (2.0 ** -21 * np.log(2) + 2.0 ** -22) + 2.0 ** -21 + 26 * 2.0 ** -24 + 2 * 2.0 ** -22
    return out, bound[..., None]


def thirds(x):
    """Three bfloat16 each, rounded towards 0."""
    out, x = [], x.astype(np.float32)
    for _ in range(3):
        a = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        out.append(a.astype(np.float64))
        x = x - a
    return out


def halves(x):
    """Two halves each."""
    hi = x.astype(np.float32).astype(np.float16).astype(np.float64)
    return [hi, (x.astype(np.float64) - hi).astype(np.float16).astype(np.float64)]
