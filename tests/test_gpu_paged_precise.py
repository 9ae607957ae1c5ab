"""Attention over a paged cache at f32's accuracy: inputs at which a part of a number that was left out would show (paged_precise)."""
import numpy as np
import pytest

import paged_precise as Q
import paged_util as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,n_kv,counts", [(16, 2, [1, 1, 1]), (14, 1, [1, 1, 1]), (30, 1, [1, 1, 1]), (4, 2, [2, 1, 2]), (4, 1, [4, 3, 4]), (4, 1, [8, 7, 5]), (4, 1, [40, 33, 37]), (32, 8, [50, 40, 1])])
@pytest.mark.parametrize("lens", [[60, 70, 90], [2500, 3100, 90]])
def test_every_part_counts(hip, f16, hd, heads, n_kv, counts, lens):
    print("precise", f16, hd, heads, n_kv, counts, lens, flush=True)
    k, v, q, where = Q.make(7, lens, sum(counts), heads, n_kv, hd, f16, max(counts))
    pool = P.Pool(hip, lens, n_kv, hd, f16, 32, seed=3, k=k, v=v)
    rows = P.Rows(pool, sum(counts), heads, seed=5)
    rows.q[:] = q
    hip.upload(rows.d_q, q)
    more = {} if max(counts) == 1 else dict(q_first=pool.dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)), max_queries=max(counts))
    hip.paged_attn(pool.kv(), rows.op(**more))
    got, at, worst = rows.result(), 0, 0.0
    for s, m in enumerate(counts):
        out, bound = Q.exact(q[at:at + m], k[s], v[s], where[s], 1 / np.sqrt(hd))
        worst = max(worst, (np.abs(got[at:at + m] - out) / (bound * out)).max())
        at += m
    print("largest error over its bound", worst, flush=True)
    assert worst <= 1
    pool.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("counts", [[1], [3], [40]])
def test_keys_of_an_f32_cache_to_their_last_bits(hip, hd, counts):
    """Two scores of 1024 and 1024.5 and a little, in powers of two, that f32 holds: the key is off by half a step of its second half, 2^-23,
    so the score by 2^-13, and the weight's share of the two, p = 0.59, by ln 2 p (1 - p) times that; the rest, as in paged_precise, is
    below 2^-18."""
    n, m = 60, counts[0]
    scale = np.float32(np.log(2))
    assert np.float32(scale * np.float32(1.44269504088896340736)) == 1
    k, v = np.zeros((n, 1, hd), np.float32), np.zeros((n, 1, hd), np.float32)
    k[:, 0, 3] = -4
    k[7, 0, 3], k[12, 0, 3] = 1 + 2.0 ** -11 + 3 * 2.0 ** -23, 1
    v[7] = 1
    pool = P.Pool(hip, [n], 1, hd, False, 32, seed=3, k=[k], v=[v])
    rows = P.Rows(pool, m, 4, seed=5)
    rows.q[:] = 0
    rows.q[..., 3] = 1024
    hip.upload(rows.d_q, rows.q)
    more = {} if m == 1 else dict(q_first=pool.dev(np.array([0, m], np.uint32)))
    hip.paged_attn(pool.kv(), rows.op(scale=float(scale), **more))
    w = 2.0 ** (0.5 + 3 * 2.0 ** -13)
    p = w / (1 + w)
    err = np.abs(rows.result() - p).max()
    print("share off by", err, flush=True)
    assert err <= np.log(2) * p * (1 - p) * 2.0 ** -13 + 2.0 ** -18
    pool.close()
