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


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("heads,n_kv,counts", [(4, 2, [3, 1, 0, 2, 3]), (8, 1, [50, 1, 0, 40, 3]), (24, 8, [2, 2, 0, 2, 2])])
@pytest.mark.parametrize("lens", [[60, 1, 5, 44, 30], [2500, 3, 0, 900, 30]])
def test_a_chunk_s_positions_start_at_nothing(hip, f16, heads, n_kv, counts, lens):
    """Theirs only: neither those before them, nor those of a sequence whose rows are out of order."""
    counts = [min(m, n) for m, n in zip(counts, lens)]
    pool = P.Pool(hip, lens, n_kv, 64, f16, 32, seed=11)
    cap = pool.cols * pool.page + 3
    before = np.random.default_rng(5).random((5, n_kv, cap)).astype(np.float32)
    d_mass = pool.dev(before)
    rows = P.Rows(pool, sum(counts), heads, seed=12, new=True)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    bad = np.array(lens, np.uint32)
    bad[4] = pool.cols * pool.page + 1
    hip.paged_attn(pool.kv(lens=pool.dev(bad)), rows.op(q_first=pool.dev(first), max_queries=max(counts), mass=d_mass, mass_stride=cap, mass_fresh=1))
    want = before.copy()
    for s in range(4):
        want[s, :, lens[s] - counts[s]:lens[s]] = 0
    assert np.array_equal(hip.download(d_mass, before.shape, np.float32), want)
    got = rows.result()
    assert np.isnan(got[first[4]:]).all() and np.isfinite(got[:first[4]]).all()
    pool.close()


@pytest.mark.parametrize("many", [False, True])
def test_evictions_with_chunks_between_rank_by_the_weights_of_what_is_there(hip, many):
    """Weights, an eviction, a chunk in the positions that became free, weights again and a second eviction."""
    n_kv, heads, hd = 2, 4, 64
    pool = P.Pool(hip, [200, 150], n_kv, hd, True, 32, seed=3)
    cap = pool.cols * pool.page
    before = (np.random.default_rng(4).random((2, n_kv, cap)) * 50).astype(np.float32)     # what many steps have collected
    d_mass, d_lens, d_new = pool.dev(before), pool.dev(np.array([200, 150], np.uint32)), pool.dev(np.zeros(2, np.uint32))
    hip.paged_evict(pool.kv(lens=d_lens), A.PagedEvict(mass=d_mass, mass_stride=cap, new_lens=d_new, budget=64, n_first=2, n_recent=4))
    kept = hip.download(d_mass, before.shape, np.float32)[:, :, :64]
    m = 40 if many else 4
    rows = P.Rows(pool, 2 * m, heads, seed=5, new=True)
    hip.upload(d_lens, np.array([64 + m] * 2, np.uint32))
    hip.paged_attn(pool.kv(lens=d_lens), rows.op(q_first=pool.dev(np.array([0, m, 2 * m], np.uint32)), max_queries=m, mass=d_mass, mass_stride=cap, mass_fresh=1))
    one = P.Rows(pool, 2, heads, seed=6, new=True)
    hip.upload(d_lens, np.array([65 + m] * 2, np.uint32))
    hip.paged_attn(pool.kv(lens=d_lens), one.op(mass=d_mass, mass_stride=cap, mass_fresh=1))
    got = hip.download(d_mass, before.shape, np.float32)
    # a step adds at most one for each query head, where positions that are gone had up to 50
    G = heads // n_kv
    assert (got[:, :, 64:65 + m] <= G * (1 + 2.0 ** -20)).all() and (got[:, :, 64:65 + m] > 0).all()
    assert (got[:, :, :64] >= kept).all() and (got[:, :, :64] <= kept + G * (1 + 2.0 ** -20)).all()
    d_newer, d_kept = pool.dev(np.zeros(2, np.uint32)), pool.dev(np.zeros((2, n_kv, 32), np.int32))
    hip.paged_evict(pool.kv(lens=d_lens), A.PagedEvict(mass=d_mass, mass_stride=cap, new_lens=d_newer, kept=d_kept, budget=32, n_first=2, n_recent=4))
    stays = hip.download(d_kept, (2, n_kv, 32), np.int32)
    for s in range(2):
        for g in range(n_kv):
            mid = sorted(range(2, 61 + m), key=lambda t: (-got[s, g, t], t))[:26]
            assert list(stays[s, g]) == [0, 1] + sorted(mid) + list(range(61 + m, 65 + m))
            assert max(mid) < 64            # the old ones weigh more: no new position has a gone one's weight
    pool.close()
