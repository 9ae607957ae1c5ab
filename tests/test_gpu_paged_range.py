"""Scores and values far from 1: what the contract allows has the definition's result."""
import numpy as np
import pytest

import paged_util as P

pytestmark = pytest.mark.gpu


def _first(pool, counts):
    return pool.dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32))


@pytest.mark.parametrize("counts", [[1], [3], [50]])
def test_a_mean_of_large_values(hip, counts):
    """A scale of 0 over 40000 positions of an f32 cache: no sum on the way may leave f32's range."""
    n = 40000
    r = np.random.default_rng(2)
    k, v = r.standard_normal((n, 1, 64)).astype(np.float32), ((0.5 + r.random((n, 1, 64))) * 6e29).astype(np.float32)
    pool = P.Pool(hip, [n], 1, 64, False, 256, seed=3, k=[k], v=[v])
    rows = P.Rows(pool, counts[0], 4, seed=5)
    hip.paged_attn(pool.kv(), rows.op(scale=0.0, **({} if counts == [1] else dict(q_first=_first(pool, counts)))))
    got = rows.result().astype(np.float64)
    v64 = v[:, 0].astype(np.float64)
    total = v64.cumsum(0)
    for i in range(counts[0]):
        m = n - counts[0] + i + 1
        assert (np.abs(got[i] - total[m - 1] / m) <= (m * 2.0 ** -24 + 2.0 ** -20) * total[m - 1] / m).all(), i
    # and of weights that differ
    hip.paged_attn(pool.kv(), rows.op(**({} if counts == [1] else dict(q_first=_first(pool, counts)))))
    out, bound, _, _ = P.attn_ref(rows.q, k, v, counts[0], 0.125, 0, 0)
    assert (np.abs(rows.result() - out) <= bound).all()
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("counts", [[1, 1], [3, 2], [5, 6], [50, 40], [80, 60]])
@pytest.mark.parametrize("lens", [[90, 60], [1900, 1500]])
@pytest.mark.parametrize("size,scale", [(3e5, 1.0), (1e6, 0.7), (3e6, 1.0), (1e9, 1.0), (1e12, -1.0), (1e31, 0.3), (-1e6, 1.3), (-2e6, -0.9), (-1e9, 1.3), (-1e12, 0.125), (-1e31, 1.0), (-1e35, 0.7)])
def test_scores_of_which_the_largest_is_all(hip, f16, counts, lens, size, scale):
    """Scores of up to 30 times `size`, size / 64 apart: the largest has all the weight, whatever was seen before it, and where a part of a
    cut sequence sees nothing of a column."""
    heads = 1 if counts == [80, 60] else 4                   # one head: a workgroup has rows of many positions
    size = max(size, -1e31) if f16 else size                 # queries of 10^30 at most
    r = np.random.default_rng(2)
    dtype = np.float16 if f16 else np.float32
    share = 1.0 if f16 else np.sqrt(abs(size)) / 64          # of the size, in the keys
    k, v = [], [r.standard_normal((n, 1, 64)).astype(dtype) for n in lens]
    for n in lens:
        x = np.zeros((n, 1, 64), dtype)
        x[:, 0, 3] = np.sign(size) * share * (64 + r.permutation(n))
        k.append(x)
    pool = P.Pool(hip, lens, 1, 64, f16, 16, seed=3, k=k, v=v)
    rows = P.Rows(pool, sum(counts), heads, seed=5)
    rows.q[:] = 0
    rows.q[..., 3] = abs(size) / 64 / share
    hip.upload(rows.d_q, rows.q)
    for window, sinks in ((0, 0), (25, 2)):
        more = {} if counts == [1, 1] else dict(q_first=_first(pool, counts), max_queries=max(counts))
        hip.paged_attn(pool.kv(), rows.op(scale=scale, window=window, n_sink=sinks, **more))
        got, at = rows.result(), 0
        for s, m in enumerate(counts):
            for i in range(m):
                ids = P.seen(lens[s] - m + i, window, sinks)
                best = ids[np.argmax(scale * k[s][ids, 0, 3].astype(np.float64))]
                # The weight, its parts' products with the value and its inverse: up to sixteen roundings of 2^-24.  From 2^24 on a score less
                # 14 may round to 16 less, and a half holds 65504 of 2^16: with few columns the weight may then lack 2^-11.
                few = f16 and max(counts) * heads <= 32 and abs(size) * 30 >= 1e7
                assert (np.abs(got[at + i] - v[s][best, 0].astype(np.float64)) <= (2.0 ** -20 + few * 2.0 ** -11) * np.abs(v[s][best, 0].astype(np.float64))).all(), (s, i, window)
            at += m
    pool.close()
