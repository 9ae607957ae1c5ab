"""Attention over a paged cache through the C ABI, against the definition in 64 bits (tolerances: paged_util.attn_ref)."""
import numpy as np
import pytest

import paged_util as P
from cera_amd import hip_api as A

pytestmark = pytest.mark.gpu

SCALE = {64: 0.125, 128: 128 ** -0.5}


def _new_rows(pool, rows, lens, counts):
    """The reference's cache with the call's own rows in it."""
    at = 0
    for s, (n, m) in enumerate(zip(lens, counts)):
        if m and n:
            pool.k[s][n - m:] = rows.k_new[at:at + m].astype(pool.dtype)
            pool.v[s][n - m:] = rows.v_new[at:at + m].astype(pool.dtype)
        at += m


def _check(pool, rows, counts, window, sinks, got=None, skip=()):
    got = rows.result() if got is None else got
    at, masses = 0, []
    for s, m in enumerate(counts):
        if s not in skip:
            out, bound, mass, mb = P.attn_ref(rows.q[at:at + m], pool.k[s], pool.v[s], m, 1 / np.sqrt(pool.hd), window, sinks)
            bad = ~(np.abs(got[at:at + m] - out) <= bound)
            assert not bad.any(), (s, np.argwhere(bad)[:4], np.abs(got[at:at + m] - out).max(), bound.max())
            masses.append((mass, mb))
        else:
            masses.append(None)
        at += m
    return masses


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 64, 100, 255, 257, 700]


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("heads,n_kv,hd,page", [(32, 8, 128, 64), (28, 4, 128, 16), (12, 2, 64, 32), (4, 4, 64, 256), (8, 1, 128, 128), (18, 2, 64, 16), (20, 1, 128, 32), (40, 1, 64, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4), (16, 0), (1, 33), (300, 70)])
def test_one_token_of_every_sequence(hip, f16, heads, n_kv, hd, page, window, sinks):
    print("decode", f16, heads, n_kv, hd, page, window, sinks, flush=True)
    pool = P.Pool(hip, LENS, n_kv, hd, f16, page, seed=heads + page)
    rows = P.Rows(pool, len(LENS), heads, seed=7, pad=8, new=True)
    hip.paged_attn(pool.kv(), rows.op(window=window, n_sink=sinks))
    _new_rows(pool, rows, LENS, [1] * len(LENS))
    _check(pool, rows, [1] * len(LENS), window, sinks)
    for s in (1, 5, len(LENS) - 1):    # what was written, bit for bit, and nothing else
        k, v = pool.rows(s, LENS[s])
        assert np.array_equal(k, pool.k[s]) and np.array_equal(v, pool.v[s])
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
def test_a_long_sequence_beside_short_ones(hip, f16):
    lens = [9001, 3, 5000, 1, 777]
    pool = P.Pool(hip, lens, 2, 128, f16, 64, seed=3)
    rows = P.Rows(pool, len(lens), 8, seed=4)
    for window, sinks in ((0, 0), (2500, 5)):
        hip.paged_attn(pool.kv(), rows.op(window=window, n_sink=sinks))
        first = rows.result().copy()
        _check(pool, rows, [1] * len(lens), window, sinks, first)
        hip.paged_attn(pool.kv(), rows.op(window=window, n_sink=sinks, max_len=9001))
        assert np.array_equal(first.view(np.uint32), rows.result().view(np.uint32))      # the same call again has the same bits
    pool.close()


@pytest.mark.parametrize("heads,n_kv,hd,f16", [(32, 8, 128, True), (14, 2, 64, True), (8, 2, 128, False), (20, 1, 64, True), (40, 1, 128, True), (36, 1, 64, False)])
@pytest.mark.parametrize("window,sinks,fresh", [(0, 0, 0), (0, 0, 1), (100, 6, 1)])
def test_weights_add_up_by_position(hip, heads, n_kv, hd, f16, window, sinks, fresh):
    lens = [1, 0, 33, 700, 2600]
    pool = P.Pool(hip, lens, n_kv, hd, f16, 32, seed=11)
    cap = pool.cols * pool.page + 5
    r = np.random.default_rng(5)
    before = r.random((len(lens), n_kv, cap)).astype(np.float32)
    d_mass = pool.dev(before)
    rows = P.Rows(pool, len(lens), heads, seed=12, new=True)
    _new_rows(pool, rows, lens, [1] * len(lens))
    steps = 2
    for _ in range(steps):
        hip.paged_attn(pool.kv(), rows.op(window=window, n_sink=sinks, mass=d_mass, mass_stride=cap, mass_fresh=fresh))
    masses = _check(pool, rows, [1] * len(lens), window, sinks)
    got = hip.download(d_mass, before.shape, np.float32)
    for s, n in enumerate(lens):
        mass, mb = masses[s]
        want = before[s, :, :n] + steps * mass
        if n and fresh:
            want[:, n - 1] = mass[:, n - 1]        # the new position's weight starts at nothing, in each of the calls
        bound = steps * mb + (steps + heads // n_kv) * 2.0 ** -24 * (want + 1)
        assert (np.abs(got[s, :, :n] - want) <= bound).all()
        assert np.array_equal(got[s, :, n:], before[s, :, n:])
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("heads,n_kv,hd,page", [(32, 8, 128, 64), (14, 2, 64, 16), (3, 1, 128, 32), (16, 16, 64, 128), (20, 2, 128, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 4), (7, 0), (130, 40)])
def test_chunks_of_new_tokens(hip, f16, heads, n_kv, hd, page, window, sinks):
    print("chunk", f16, heads, n_kv, hd, page, window, sinks, flush=True)
    lens, counts = [5, 64, 0, 333, 90, 17, 130], [5, 3, 0, 1, 77, 16, 65]
    pool = P.Pool(hip, lens, n_kv, hd, f16, page, seed=heads, interleaved=True)
    rows = P.Rows(pool, sum(counts), heads, seed=8, pad=4, new=True)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    hip.paged_attn(pool.kv(), rows.op(q_first=pool.dev(first), window=window, n_sink=sinks, max_queries=77))
    _new_rows(pool, rows, lens, counts)
    _check(pool, rows, counts, window, sinks)
    for s, n in enumerate(lens):
        k, v = pool.rows(s, n)
        assert np.array_equal(k, pool.k[s]) and np.array_equal(v, pool.v[s])
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 4)])
def test_a_long_chunk(hip, f16, window, sinks):
    lens, counts = [1500, 400], [300, 400]
    pool = P.Pool(hip, lens, 2, 128, f16, 32, seed=2)
    rows = P.Rows(pool, sum(counts), 8, seed=9)
    first = np.array([0, 300, 700], np.uint32)
    hip.paged_attn(pool.kv(), rows.op(q_first=pool.dev(first), window=window, n_sink=sinks))
    _check(pool, rows, counts, window, sinks)
    pool.close()


def test_rows_of_no_sequence_stay(hip):
    pool = P.Pool(hip, [40, 20], 2, 64, True, 16, seed=2)
    rows = P.Rows(pool, 12, 4, seed=9)
    hip.paged_attn(pool.kv(), rows.op(q_first=pool.dev(np.array([2, 5, 9], np.uint32))))
    got = rows.result()
    assert (got[:2] == P.SENTINEL).all() and (got[9:] == P.SENTINEL).all()
    for s, (a, b) in enumerate(((2, 5), (5, 9))):
        out, bound, _, _ = P.attn_ref(rows.q[a:b], pool.k[s], pool.v[s], b - a, 0.125, 0, 0)
        assert (np.abs(got[a:b] - out) <= bound).all()
    pool.close()


@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("f16", [True, False])
def test_bad_pages_and_lengths_give_nan_to_their_own_sequence(hip, chunk, f16):
    lens = [40, 70, 300, 33, 20]
    pool = P.Pool(hip, lens, 2, 64, f16, 16, seed=6)
    rows = P.Rows(pool, len(lens), 4, seed=3, new=True)
    table = pool.table.copy()
    table[0, 1], table[2, 0], table[4, 0] = -1, pool.n_pages, 0x7FFFFFFF
    bad_lens = np.array(lens, np.uint32)
    bad_lens[3] = pool.cols * pool.page + 1
    kv = pool.kv(table=pool.dev(table), lens=pool.dev(bad_lens))
    more = dict(q_first=pool.dev(np.arange(len(lens) + 1, dtype=np.uint32))) if chunk else {}
    hip.paged_attn(kv, rows.op(**more))
    _new_rows(pool, rows, lens, [1] * len(lens))
    got = rows.result()
    for s in (0, 2, 3, 4):
        assert np.isnan(got[s]).all(), s
    _check(pool, rows, [1] * len(lens), 0, 0, got, skip=(0, 2, 3, 4))
    # behind a window the bad first page is out of sight
    hip.paged_attn(kv, rows.op(window=16, **more))
    got = rows.result()
    out, bound, _, _ = P.attn_ref(rows.q[2:3], pool.k[2], pool.v[2], 1, 0.125, 16, 0)
    assert (np.abs(got[2:3] - out) <= bound).all() and np.isnan(got[3]).all()
    pool.close()


def test_rows_out_of_order_give_nan(hip):
    pool = P.Pool(hip, [40, 20, 30, 8], 2, 64, True, 16, seed=2)
    rows = P.Rows(pool, 20, 4, seed=9, new=True)
    before = pool.pages()
    # rows that decrease, more rows than positions, more than max_queries, an end behind n_rows
    hip.paged_attn(pool.kv(), rows.op(q_first=pool.dev(np.array([3, 1, 8, 11, 21], np.uint32)), max_queries=6))
    got = rows.result()
    assert np.isnan(got[1:8]).all() and np.isnan(got[11:]).all() and (got[0] == P.SENTINEL).all()
    out, bound, _, _ = P.attn_ref(rows.q[8:11], np.concatenate([pool.k[2][:27], rows.k_new[8:11].astype(np.float16)]),
                                  np.concatenate([pool.v[2][:27], rows.v_new[8:11].astype(np.float16)]), 3, 0.125, 0, 0)
    assert (np.abs(got[8:11] - out) <= bound).all()
    after = pool.pages()
    for s in (0, 1, 3):
        for t in range(pool.lens[s]):
            p = pool.table[s, t // 16]
            for x, y in zip(before, after):
                assert np.array_equal(x[p, :, t % 16], y[p, :, t % 16])
    pool.close()


@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("f16", [True, False])
def test_large_and_small_queries(hip, f16, chunk):
    """Queries far from 1 lose nothing to their halves, and none are zeros."""
    lens = [70] * 5
    pool = P.Pool(hip, lens, 1, 64, f16, 16, seed=6)
    rows = P.Rows(pool, 5, 2, seed=3)
    for s, f in enumerate((1e-20, 300, 1e4, 0, 1e-3)):
        rows.q[s] *= np.float32(f)
    hip.upload(rows.d_q, rows.q)
    hip.paged_attn(pool.kv(), rows.op(**(dict(q_first=pool.dev(np.arange(6, dtype=np.uint32))) if chunk else {})))
    _check(pool, rows, [1] * 5, 0, 0)
    pool.close()


@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 17, 30]])
def test_f32_rows_of_very_different_size(hip, counts):
    """Keys and values that no half can hold, and rows 2^40 apart: the bound is relative to the weighted values' sizes."""
    lens = [90, 60, 45]
    r = np.random.default_rng(1)
    k = [(r.standard_normal((n, 2, 64)) * (2.0 ** r.integers(-20, 3, (n, 2, 1)))).astype(np.float32) for n in lens]
    v = [(r.standard_normal((n, 2, 64)) * (2.0 ** r.integers(-20, 20, (n, 2, 1)))).astype(np.float32) for n in lens]
    k[1] *= np.float32(1e6)
    v[2] *= np.float32(1e20)
    pool = P.Pool(hip, lens, 2, 64, False, 16, seed=3, k=k, v=v)
    rows = P.Rows(pool, sum(counts), 8, seed=5)
    at = counts[0]
    rows.q[at:at + counts[1]] *= np.float32(1e-6)
    hip.upload(rows.d_q, rows.q)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    for window in (0, 20):
        hip.paged_attn(pool.kv(), rows.op(q_first=pool.dev(first), window=window))
        got, at = rows.result(), 0
        for s, m in enumerate(counts):
            out, bound, _, _ = P.attn_ref(rows.q[at:at + m], k[s], v[s], m, 0.125, window, 0)
            assert (np.abs(got[at:at + m] - out) <= bound).all(), (s, window)
            at += m
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("heads,n_kv,hd", [(2, 2, 64), (8, 1, 64), (6, 2, 128), (4, 1, 128), (40, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_infinities_reach_only_the_rows_that_see_them(hip, f16, heads, n_kv, hd, window, sinks):
    """Infinities and NaN among the values, and in keys that no earlier row may see: chunks of few and of many rows."""
    lens, counts = [70, 150, 40], [6, 50, 3]
    pool = P.Pool(hip, lens, n_kv, hd, f16, 16, seed=3)
    k, v = [x.copy() for x in pool.k], [x.copy() for x in pool.v]
    pool.close()
    v[0][66, :, 3] = np.inf
    v[0][67, :, 5] = np.nan
    v[1][120, :, 7] = -np.inf
    v[1][140, 0, :] = np.nan
    k[1][149] = np.nan               # the last row's own key: only it sees it
    v[2][38, :, hd - 1] = np.inf
    v[2][39, :, hd - 1] = -np.inf
    pool = P.Pool(hip, lens, n_kv, hd, f16, 16, seed=3, k=k, v=v)
    rows = P.Rows(pool, sum(counts), heads, seed=5)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    hip.paged_attn(pool.kv(), rows.op(q_first=pool.dev(first), window=window, n_sink=sinks))
    got, at = rows.result(), 0
    with np.errstate(invalid="ignore"):
        for s, m in enumerate(counts):
            out, bound, _, _ = P.attn_ref(rows.q[at:at + m], k[s], v[s], m, 1 / np.sqrt(hd), window, sinks)
            g = got[at:at + m]
            if s == 1:
                assert np.isnan(g[-1]).all()          # its own key is no number
                g, out, bound = g[:-1], out[:-1], bound[:-1]
            fine = np.isfinite(out)
            assert fine.any() and not fine.all()
            assert (np.abs(g - out)[fine] <= bound[fine]).all(), s
            # an infinity times a weight's low part of 0 is NaN: what the row sees makes its value not finite, of either kind
            assert not np.isfinite(g[~fine]).any(), s
            at += m
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("heads,n_kv,n_seqs,window,sinks", [(32, 8, 12, 0, 0), (32, 8, 12, 40, 3), (24, 8, 15, 0, 0), (8, 8, 64, 0, 0), (16, 4, 70, 0, 0), (72, 4, 9, 100, 0)])
def test_chunks_of_many_sequences(hip, f16, heads, n_kv, n_seqs, window, sinks):
    """Uncut groups of columns of ragged sequences, longest first (up to 64 of them) or in order, with empty and faulty ones among them."""
    print("many", f16, heads, n_kv, n_seqs, window, sinks, flush=True)
    r = np.random.default_rng(n_seqs)
    lens = [int(x) for x in r.integers(1, 260, n_seqs)]
    counts = [int(min(n, c)) for n, c in zip(lens, r.integers(0, 130 if n_seqs < 20 else 40, n_seqs))]
    lens[2], counts[2] = 0, 0
    counts[4], lens[4] = 33, 259
    counts[6] = min(lens[6], 5)
    pool = P.Pool(hip, lens, n_kv, 64, f16, 32, seed=3)
    rows = P.Rows(pool, sum(counts), heads, seed=4, new=True)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    bad = np.array(lens, np.uint32)
    bad[6] = pool.cols * pool.page + 1            # longer than its row of the table
    hip.paged_attn(pool.kv(lens=pool.dev(bad)), rows.op(q_first=pool.dev(first), max_queries=max(counts), window=window, n_sink=sinks))
    _new_rows(pool, rows, lens, counts)
    got = rows.result()
    _check(pool, rows, counts, window, sinks, got, skip=(6,))
    assert np.isnan(got[first[6]:first[7]]).all()
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("heads,n_kv,hd", [(2, 2, 64), (8, 1, 64), (4, 1, 128), (40, 1, 128)])
@pytest.mark.parametrize("window", [0, 2])
def test_new_values_that_are_not_finite(hip, f16, heads, n_kv, hd, window):
    """Among a chunk's own rows, one of them infinite only as the cache holds it."""
    lens, counts = [70, 53, 4], [5, 40, 2]
    pool = P.Pool(hip, lens, n_kv, hd, f16, 16, seed=3)
    rows = P.Rows(pool, sum(counts), heads, seed=5, new=True)
    rows.v_new[2, :, 3] = np.inf
    rows.v_new[3, :, 5] = 1e6
    rows.v_new[4, :, 6] = np.nan
    rows.v_new[5 + 30, 0, :9] = -np.inf
    rows.v_new[46, :, hd - 1] = -1e6
    hip.upload(rows.d_vn, rows.v_new)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    with np.errstate(over="ignore", invalid="ignore"):
        _new_rows(pool, rows, lens, counts)
        hip.paged_attn(pool.kv(), rows.op(q_first=pool.dev(first), window=window))
        got, at = rows.result(), 0
        for s, m in enumerate(counts):
            out, bound, _, _ = P.attn_ref(rows.q[at:at + m], pool.k[s], pool.v[s], m, 1 / np.sqrt(hd), window, 0)
            fine = np.isfinite(out)
            assert fine.any() and (fine.all() if s == 2 and not f16 else not fine.all())
            assert (np.abs(got[at:at + m] - out)[fine] <= bound[fine]).all() and not np.isfinite(got[at:at + m][~fine]).any(), s
            at += m
    for s, n in enumerate(lens):
        k, v = pool.rows(s, n)
        assert np.array_equal(k, pool.k[s]) and np.array_equal(v, pool.v[s], equal_nan=True)
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("chunk", [False, True])
def test_more_sequences_than_a_wavefront_has_lanes(hip, f16, chunk):
    """150 ragged sequences in equal shares, with empty ones among them, cut and whole."""
    r = np.random.default_rng(4)
    lens = [int(x) for x in r.integers(0, 200, 150)]
    lens[5], lens[77], lens[149], lens[70], lens[0] = 1500, 900, 640, 0, 0
    counts = [min(n, int(c)) if chunk else 1 for n, c in zip(lens, r.integers(0, 4, 150))]
    pool = P.Pool(hip, lens, 1, 64, f16, 16, seed=3)
    rows = P.Rows(pool, sum(counts), 4, seed=4, new=True)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    hip.paged_attn(pool.kv(), rows.op(**(dict(q_first=pool.dev(first), max_queries=3) if chunk else {})))
    _new_rows(pool, rows, lens, counts)
    _check(pool, rows, counts, 0, 0)
    pool.close()


@pytest.mark.parametrize("heads,n_kv,f16", [(130, 2, True), (130, 2, False), (300, 1, True)])
def test_more_heads_of_a_kv_head_than_a_workgroup_has_columns(hip, heads, n_kv, f16):
    lens = [700, 0, 33, 1]
    pool = P.Pool(hip, lens, n_kv, 64, f16, 32, seed=11)
    cap = pool.cols * pool.page
    d_mass = pool.dev(np.zeros((len(lens), n_kv, cap), np.float32))
    rows = P.Rows(pool, len(lens), heads, seed=12, new=True)
    hip.paged_attn(pool.kv(), rows.op(mass=d_mass, mass_stride=cap))
    _new_rows(pool, rows, lens, [1] * len(lens))
    masses = _check(pool, rows, [1] * len(lens), 0, 0)
    for s, n in enumerate(lens):
        k, v = pool.rows(s, n)
        assert np.array_equal(k, pool.k[s]) and np.array_equal(v, pool.v[s])
        mass, mb = masses[s]
        got = hip.download(d_mass, (len(lens), n_kv, cap), np.float32)[s, :, :n]
        assert (np.abs(got - mass) <= mb + (1 + heads // n_kv) * 2.0 ** -24 * (mass + 1)).all()
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.25, 1e-9, -3.0])
def test_scales(hip, f16, chunk, scale):
    """A scale of 0 gives the mean of what is seen; a negative one turns the order round."""
    lens, counts = [70, 500, 1], [20, 60, 1] if chunk else [1, 1, 1]
    pool = P.Pool(hip, lens, 1, 64, f16, 16, seed=6)
    rows = P.Rows(pool, sum(counts), 4, seed=3)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    hip.paged_attn(pool.kv(), rows.op(scale=scale, window=300, **(dict(q_first=pool.dev(first)) if chunk else {})))
    got, at = rows.result(), 0
    for s, m in enumerate(counts):
        out, bound, _, _ = P.attn_ref(rows.q[at:at + m], pool.k[s], pool.v[s], m, scale, 300, 0)
        assert (np.abs(got[at:at + m] - out) <= bound).all(), s
        at += m
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("counts", [[3, 2], [30, 20]])
def test_a_query_that_is_no_number_is_its_row_s_alone(hip, f16, counts):
    lens = [90, 60]
    pool = P.Pool(hip, lens, 1, 64, f16, 16, seed=6)
    rows = P.Rows(pool, sum(counts), 4, seed=3)
    rows.q[1, 2, 5] = np.nan
    rows.q[counts[0], 0, 0] = np.inf
    hip.upload(rows.d_q, rows.q)
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    hip.paged_attn(pool.kv(), rows.op(q_first=pool.dev(first)))
    got = rows.result().copy()
    assert np.isnan(got[1, 2]).all() and np.isnan(got[counts[0], 0]).all()
    for row, h in ((1, 2), (counts[0], 0)):
        rows.q[row, h] = 0
        hip.upload(rows.d_q, rows.q)
    hip.paged_attn(pool.kv(), rows.op(q_first=pool.dev(first)))
    want = rows.result()
    got[1, 2], got[counts[0], 0] = want[1, 2], want[counts[0], 0]
    assert np.array_equal(got, want)
    pool.close()


def test_without_room_for_parts(hip):
    """A limit on workspaces: sequences are not cut then, and weights, which need theirs, are refused."""
    ctx = A.Context(0)
    lens = [3000, 0, 20]
    pool = P.Pool(ctx, lens, 2, 64, True, 32, seed=11)
    cap = pool.cols * pool.page
    rows = P.Rows(pool, len(lens), 8, seed=12)
    before = np.ones((len(lens), 2, cap), np.float32)
    d_mass = pool.dev(before)
    ctx.set_workspace_limit(4096)
    ctx.paged_attn(pool.kv(), rows.op())
    _check(pool, rows, [1] * 3, 0, 0)
    with pytest.raises(A.HipError) as e:
        ctx.paged_attn(pool.kv(), rows.op(mass=d_mass, mass_stride=cap))
    assert e.value.status == 2 and e.value.message
    assert np.array_equal(ctx.download(d_mass, before.shape, np.float32), before)
    ctx.set_workspace_limit(0)
    ctx.paged_attn(pool.kv(), rows.op(mass=d_mass, mass_stride=cap))
    _check(pool, rows, [1] * 3, 0, 0)
    got = ctx.download(d_mass, before.shape, np.float32) - 1
    assert abs(got[0].sum() - 8) < 1e-3 and np.count_nonzero(got[1]) == 0
    pool.close()
    ctx.close()


def test_two_contexts_and_calls_of_other_sizes_between(hip):
    """Each context has its own stream and workspaces, and a call's results owe nothing to the calls before it."""
    import threading
    ctxs = [A.Context(0), A.Context(0)]
    work = []
    for i, ctx in enumerate(ctxs):
        mine = []
        for lens in ([2000 + 300 * i, 5, 700], [40, 1, 9 + i], [1200, 1300, 0]):
            pool = P.Pool(ctx, lens, 2, 128, True, 32, seed=i)
            rows = P.Rows(pool, 3, 8, seed=i + 5)
            cap = pool.cols * pool.page
            mass = pool.dev(np.zeros((3, 2, cap), np.float32))
            mine.append((pool, rows, mass, cap))
        work.append(mine)
    once = [[], []]
    for i, ctx in enumerate(ctxs):        # each by itself, in order
        for pool, rows, mass, cap in work[i]:
            ctx.paged_attn(pool.kv(), rows.op(mass=mass, mass_stride=cap))
            _check(pool, rows, [1] * 3, 0, 0)
            once[i].append((rows.result().copy(), ctx.download(mass, (3, 2, cap), np.float32)))
    wrong = []

    def run(i):
        try:
            for k in (2, 1, 0, 1, 2) * 4:
                pool, rows, mass, cap = work[i][k]
                ctxs[i].upload(mass, np.zeros((3, 2, cap), np.float32))
                ctxs[i].paged_attn(pool.kv(), rows.op(mass=mass, mass_stride=cap))
                out, m = rows.result(), ctxs[i].download(mass, (3, 2, cap), np.float32)
                if not (np.array_equal(out, once[i][k][0]) and np.array_equal(m, once[i][k][1])):
                    wrong.append((i, k))
        except Exception as e:      # a thread's failure is the test's
            wrong.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for mine in work:
        for pool, _, _, _ in mine:
            pool.close()
    for ctx in ctxs:
        ctx.close()


def test_offsets_beyond_32_bits(hip):
    """Pages 2^31 elements apart: byte and element offsets past 32 bits."""
    stride, n_kv, hd, page = (1 << 31) + 8, 2, 128, 16
    base = hip.malloc(3 * stride * 2)
    r = np.random.default_rng(0)
    n = 40
    k, v = (r.standard_normal((n, n_kv, hd)).astype(np.float16) for _ in range(2))
    table = np.array([[2, 0, 1]], np.int32)
    per = n_kv * page * hd
    for i, p in enumerate(table[0]):
        for x, off in ((k, 0), (v, per)):
            block = np.zeros((n_kv, page, hd), np.float16)
            part = x[i * page:(i + 1) * page]
            block[:, :len(part)] = part.transpose(1, 0, 2)
            hip.upload(base + (int(p) * stride + off) * 2, block)
    q = r.standard_normal((1, 8, hd)).astype(np.float32)
    bufs = [hip.to_device(x) for x in (table, np.array([n], np.uint32), q)]
    d_out = hip.malloc(q.nbytes)
    hip.paged_attn(A.PagedKV(kv_type=1, n_kv_heads=n_kv, head_dim=hd, page_size=page, n_pages=3, n_seqs=1, max_pages=3, page_stride=stride, k=base, v=base + per * 2,
                             table=bufs[0], lens=bufs[1]), A.PagedAttn(q=bufs[2], out=d_out, n_rows=1, n_heads=8, scale=SCALE[hd]))
    got = hip.download(d_out, q.shape, np.float32)
    out, bound, _, _ = P.attn_ref(q, k, v, 1, SCALE[hd], 0, 0)
    assert (np.abs(got - out) <= bound).all()
    for b in bufs + [d_out, base]:
        hip.free(b)


def test_sequences_that_share_pages(hip):
    """Two sequences with the same first pages: reading them needs no copies."""
    pool = P.Pool(hip, [96, 96], 2, 64, True, 32, seed=1)
    table = pool.table.copy()
    table[1, :2] = table[0, :2]
    rows = P.Rows(pool, 2, 4, seed=3)
    hip.paged_attn(pool.kv(table=pool.dev(table)), rows.op())
    for x in (pool.k, pool.v):
        x[1][:64] = x[0][:64]
    _check(pool, rows, [1, 1], 0, 0)
    pool.close()


def test_refusals(hip):
    pool = P.Pool(hip, [40, 20], 2, 64, True, 16, seed=2)
    rows = P.Rows(pool, 2, 4, seed=9)
    for kv, op, status in ((pool.kv(head_dim=96), rows.op(), 4), (pool.kv(page_size=24), rows.op(), 4), (pool.kv(kv_type=2), rows.op(), 3), (pool.kv(), rows.op(n_heads=3), 4),
                           (pool.kv(), rows.op(out=None), 6), (pool.kv(), rows.op(scale=float("nan")), 6), (pool.kv(), rows.op(q=rows.d_q + 4), 6), (pool.kv(), rows.op(n_rows=1), 4),
                           (pool.kv(), rows.op(k_new=rows.d_q), 6), (pool.kv(k=None), rows.op(), 6)):
        with pytest.raises(A.HipError) as e:
            hip.paged_attn(kv, op)
        assert e.value.status == status and e.value.message
    assert (rows.result() == P.SENTINEL).all()
    hip.paged_attn(pool.kv(n_seqs=0), rows.op(n_rows=0))
    pool.close()
