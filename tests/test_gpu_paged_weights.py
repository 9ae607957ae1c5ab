"""Weights by position where something is not in order: a head that is no number, positions that are given again."""
import numpy as np
import pytest

import paged_util as P
from cera_amd import hip_api as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("heads,n_kv", [(8, 2), (3, 1), (40, 1)])
@pytest.mark.parametrize("fresh", [0, 1])
@pytest.mark.parametrize("every", [False, True])
def test_a_head_that_is_no_number_adds_nothing(hip, f16, heads, n_kv, fresh, every):
    """The other heads of its kv head add theirs, and the new position starts at 0 all the same."""
    lens = [1, 40, 2600, 300]
    pool = P.Pool(hip, lens, n_kv, 64, f16, 32, seed=11)
    cap = pool.cols * pool.page
    before = np.random.default_rng(5).random((4, n_kv, cap)).astype(np.float32)
    d_mass = pool.dev(before)
    rows = P.Rows(pool, 4, heads, seed=12, new=True)
    G = heads // n_kv
    odd = range(G) if every else [1]           # of the first kv head
    for s, value in ((0, np.nan), (1, np.inf), (2, np.nan)):
        rows.q[s, list(odd), 3] = value
    hip.upload(rows.d_q, rows.q)
    hip.paged_attn(pool.kv(), rows.op(mass=d_mass, mass_stride=cap, mass_fresh=fresh))
    got, out = hip.download(d_mass, before.shape, np.float32), rows.result()
    for s, n in enumerate(lens):
        pool.k[s][n - 1], pool.v[s][n - 1] = rows.k_new[s].astype(pool.dtype), rows.v_new[s].astype(pool.dtype)
        for g in range(n_kv):
            good = [h for h in range(g * G, (g + 1) * G) if s == 3 or g or h not in odd]
            want, bound = before[s, g, :n].astype(np.float64), np.zeros(n)
            if fresh:
                want[n - 1] = 0
            for h in good:                         # a head by itself
                _, _, mass, mb = P.attn_ref(rows.q[s:s + 1, h:h + 1], pool.k[s][:, g:g + 1], pool.v[s][:, g:g + 1], 1, 0.125, 0, 0)
                want, bound = want + mass[0], bound + mb[0]
            assert (np.abs(got[s, g, :n] - want) <= bound + (1 + G) * 2.0 ** -24 * (want + 1)).all(), (s, g)
            assert np.array_equal(got[s, g, n:], before[s, g, n:])
            for h in range(g * G, (g + 1) * G):
                assert np.isnan(out[s, h]).all() == (h not in good)
    pool.close()


@pytest.mark.parametrize("fresh", [0, 1])
def test_a_bad_page_adds_nothing(hip, fresh):
    lens = [100, 100]
    pool = P.Pool(hip, lens, 2, 64, True, 16, seed=11)
    cap = pool.cols * pool.page
    before = np.random.default_rng(5).random((2, 2, cap)).astype(np.float32)
    d_mass = pool.dev(before)
    rows = P.Rows(pool, 2, 4, seed=12, new=True)
    table = pool.table.copy()
    table[0, 2] = -1
    hip.paged_attn(pool.kv(table=pool.dev(table)), rows.op(mass=d_mass, mass_stride=cap, mass_fresh=fresh))
    got = hip.download(d_mass, before.shape, np.float32)
    assert np.isnan(rows.result()[0]).all() and np.array_equal(got[0, :, :99], before[0, :, :99])
    assert (got[1, :, :99] > before[1, :, :99]).all()
    pool.close()
