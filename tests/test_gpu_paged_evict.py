"""Eviction from a paged cache through the C ABI, against the definition: what stays is equal, bit for bit."""
import numpy as np
import pytest

import paged_util as P
from cera_amd import hip_api as A

pytestmark = pytest.mark.gpu


def _kept(w, n, budget, first, recent):
    if n <= budget:
        return np.arange(n)
    key = np.where(np.isnan(w), np.inf, w.astype(np.float64)) + 0.0
    nan = np.isnan(w)
    mid = sorted(range(first, n - recent), key=lambda t: (not nan[t], -key[t], t))[:budget - first - recent]
    return np.array(sorted(list(range(first)) + mid + list(range(n - recent, n))), np.int64)


def _run(hip, pool, mass, budget, first, recent, table=None, lens=None, kept=True, max_len=0):
    n = len(pool.lens)
    d_mass, d_new = pool.dev(mass), pool.dev(np.full(n + 1, 77, np.uint32))
    d_kept = pool.dev(np.full((n, pool.n_kv, budget), -9, np.int32)) if kept else None
    more = {}
    if table is not None:
        more["table"] = pool.dev(table)
    if lens is not None:
        more["lens"] = pool.dev(lens)
    hip.paged_evict(pool.kv(**more), A.PagedEvict(mass=d_mass, mass_stride=mass.shape[2], new_lens=d_new, kept=d_kept, budget=budget, n_first=first, n_recent=recent, max_len=max_len))
    new = hip.download(d_new, n + 1, np.uint32)
    assert new[n] == 77
    return new[:n], hip.download(d_kept, (n, pool.n_kv, budget), np.int32) if kept else None, hip.download(d_mass, mass.shape, np.float32)


def _check(pool, mass, budget, first, recent, new, kept, got_mass, skip=()):
    before_k, before_v = pool.k, pool.v
    for s, n in enumerate(pool.lens):
        if s in skip:
            continue
        m = min(n, budget)
        assert new[s] == m
        gk, gv = pool.rows(s, m)
        for g in range(pool.n_kv):
            ids = _kept(mass[s, g, :n], n, budget, first, recent)
            assert np.array_equal(kept[s, g, :m], ids) and (kept[s, g, m:] == -1).all(), (s, g)
            assert np.array_equal(gk[:, g], before_k[s][ids, g]) and np.array_equal(gv[:, g], before_v[s][ids, g]), (s, g)
            assert np.array_equal(got_mass[s, g, :m].view(np.uint32), mass[s, g, ids].view(np.uint32))
            assert np.array_equal(got_mass[s, g, n:].view(np.uint32), mass[s, g, n:].view(np.uint32))


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("n_kv,hd,page", [(2, 128, 16), (3, 64, 64), (1, 128, 256), (8, 64, 32)])
@pytest.mark.parametrize("budget,first,recent", [(1, 0, 0), (37, 4, 8), (64, 0, 64), (64, 64, 0), (300, 4, 50), (700, 1, 0), (1200, 4, 100)])
def test_what_stays(hip, f16, n_kv, hd, page, budget, first, recent):
    print("evict", f16, n_kv, hd, page, budget, first, recent, flush=True)
    lens = [0, 1, budget - 1, budget, budget + 1, budget + 17, 1100, 64]
    pool = P.Pool(hip, lens, n_kv, hd, f16, page, seed=budget, interleaved=hd == 64)
    r = np.random.default_rng(budget)
    cap = pool.cols * pool.page
    mass = r.random((len(lens), n_kv, cap)).astype(np.float32) ** 8
    new, kept, got = _run(hip, pool, mass, budget, first, recent)
    _check(pool, mass, budget, first, recent, new, kept, got)
    pool.close()


@pytest.mark.parametrize("kind", ["equal", "two values", "zeros of both signs", "nan", "negative", "infinite", "tiny"])
def test_ties_and_odd_weights(hip, kind):
    lens, budget, first, recent = [3000, 2049, 1025], 1000, 3, 11
    pool = P.Pool(hip, lens, 2, 64, True, 32, seed=5)
    r = np.random.default_rng(3)
    shape = (3, 2, pool.cols * 32)
    mass = {"equal": np.full(shape, 0.25), "two values": r.integers(0, 2, shape) * 1.0, "zeros of both signs": np.where(r.integers(0, 2, shape), 0.0, -0.0),
            "nan": np.where(r.random(shape) < 0.1, np.nan, r.random(shape)), "negative": r.standard_normal(shape), "infinite": np.where(r.random(shape) < 0.2, np.inf, -np.inf),
            "tiny": r.random(shape) * 1e-42}[kind].astype(np.float32)
    new, kept, got = _run(hip, pool, mass, budget, first, recent)
    _check(pool, mass, budget, first, recent, new, kept, got)
    pool.close()


def test_a_long_sequence_and_without_the_list(hip):
    lens = [20000, 9000]
    pool = P.Pool(hip, lens, 1, 64, True, 256, seed=5)
    mass = np.random.default_rng(3).random((2, 1, pool.cols * 256)).astype(np.float32)
    new, _, got = _run(hip, pool, mass, 8192, 4, 1000, kept=False, max_len=20000)
    kept = np.full((2, 1, 8192), -1, np.int32)
    for s, n in enumerate(lens):
        kept[s, 0] = _kept(mass[s, 0, :n], n, 8192, 4, 1000)
    _check(pool, mass, 8192, 4, 1000, new, kept, got)
    pool.close()


def test_bad_pages_and_lengths_leave_their_sequence(hip):
    lens = [300, 400, 200, 250]
    pool = P.Pool(hip, lens, 2, 64, True, 16, seed=9)
    mass = np.random.default_rng(3).random((4, 2, pool.cols * 16)).astype(np.float32)
    table, bad = pool.table.copy(), np.array(lens, np.uint32)
    table[0, 3], table[2, 12] = -1, pool.n_pages
    bad[3] = pool.cols * 16 + 1
    before = pool.pages()
    new, kept, got = _run(hip, pool, mass, 100, 4, 10, table=table, lens=bad)
    assert list(new) == [300, 100, 200, bad[3]]
    _check(pool, mass, 100, 4, 10, new, kept, got, skip=(0, 2, 3))
    after = pool.pages()
    for s in (0, 2, 3):
        assert (kept[s] == -1).all() and np.array_equal(got[s], mass[s])
        for t in range(lens[s]):
            for x, y in zip(before, after):
                assert np.array_equal(x[pool.table[s, t // 16], :, t % 16], y[pool.table[s, t // 16], :, t % 16])
    pool.close()


def test_two_calls_in_a_row(hip):
    """The second on what the first left, with its lengths."""
    lens = [900, 500]
    pool = P.Pool(hip, lens, 2, 128, True, 64, seed=4)
    mass = np.random.default_rng(3).random((2, 2, pool.cols * 64)).astype(np.float32)
    d_mass, d_new, d_newer = pool.dev(mass), pool.dev(np.zeros(2, np.uint32)), pool.dev(np.zeros(2, np.uint32))
    kept = [pool.dev(np.zeros((2, 2, b), np.int32)) for b in (400, 150)]
    op = dict(mass=d_mass, mass_stride=mass.shape[2], n_first=4, n_recent=32)
    hip.paged_evict(pool.kv(), A.PagedEvict(new_lens=d_new, kept=kept[0], budget=400, **op))
    hip.paged_evict(pool.kv(lens=d_new), A.PagedEvict(new_lens=d_newer, kept=kept[1], budget=150, **op))
    assert list(hip.download(d_newer, 2, np.uint32)) == [150, 150]
    k1, k2 = hip.download(kept[0], (2, 2, 400), np.int32), hip.download(kept[1], (2, 2, 150), np.int32)
    for s, n in enumerate(lens):
        gk, gv = pool.rows(s, 150)
        for g in range(2):
            a = _kept(mass[s, g, :n], n, 400, 4, 32)
            b = _kept(mass[s, g, a], 400, 150, 4, 32)
            assert np.array_equal(k1[s, g], a) and np.array_equal(k2[s, g], b)
            assert np.array_equal(gk[:, g], pool.k[s][a[b], g]) and np.array_equal(gv[:, g], pool.v[s][a[b], g])
    pool.close()


def test_refusals(hip):
    pool = P.Pool(hip, [40], 2, 64, True, 16, seed=2)
    d = pool.dev(np.zeros((1, 2, 64), np.float32))
    ok = dict(mass=d, mass_stride=64, new_lens=d, budget=8, n_first=4, n_recent=4)
    for more, status in ((dict(mass=None), 6), (dict(budget=0, n_first=0, n_recent=0), 4), (dict(n_recent=5), 4), (dict(mass_stride=47), 4), (dict(new_lens=pool.d_lens), 6)):
        with pytest.raises(A.HipError) as e:
            hip.paged_evict(pool.kv(), A.PagedEvict(**{**ok, **more}))
        assert e.value.status == status
    pool.close()
