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
