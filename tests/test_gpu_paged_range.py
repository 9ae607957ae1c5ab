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
