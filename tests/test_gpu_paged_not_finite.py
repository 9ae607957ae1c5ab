"""Infinities and NaN among queries and keys: every row that has or sees one is NaN, whatever the sign of its product; others keep their values."""
import numpy as np
import pytest

import paged_util as P

pytestmark = pytest.mark.gpu


def _first(pool, counts):
    return pool.dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32))


def _check(pool, rows, counts, window, sinks, odd, k=None, v=None):
    """odd: per sequence {position: kv heads} with keys that are not finite."""
    k, v = k or pool.k, v or pool.v
    got, at = rows.result(), 0
    G = rows.heads // pool.n_kv
    for s, m in enumerate(counts):
        n = k[s].shape[0]
        clean = k[s].astype(np.float64)
        clean[~np.isfinite(clean)] = 0
        out, bound, _, _ = P.attn_ref(rows.q[at:at + m], clean, v[s], m, 1 / np.sqrt(pool.hd), window, sinks)
        for i in range(m):
            ids = set(P.seen(n - m + i, window, sinks).tolist())
            for h in range(rows.heads):
                g = got[at + i, h]
                if any(t in ids and h // G in heads for t, heads in odd[s].items()):
                    assert np.isnan(g).all(), (s, i, h, g[:4])
                else:
                    assert (np.abs(g - out[i, h]) <= bound[i, h]).all(), (s, i, h)
        at += m


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("heads,n_kv,hd,counts", [(8, 2, 64, [1, 1, 1]), (40, 1, 64, [1, 1, 1]), (8, 2, 128, [2, 3, 1]), (4, 1, 64, [5, 6, 2]), (8, 1, 128, [40, 17, 3]), (4, 2, 64, [40, 70, 3])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 3)])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_keys(hip, f16, heads, n_kv, hd, counts, window, sinks, sign):
    """Queries are positive in one dim and negative in another, keys infinite in these: products of both signs."""
    print("infinite keys", f16, heads, n_kv, hd, counts, window, sign, flush=True)
    lens = [90, 150, 7]
    pool = P.Pool(hip, lens, n_kv, hd, f16, 16, seed=3)
    k = [x.copy() for x in pool.k]
    pool.close()
    last = n_kv - 1
    k[0][60, 0, 5] = sign * np.inf
    k[0][88, last, 9] = sign * np.inf          # behind the first of a chunk's rows
    k[1][1, last, 5] = sign * np.inf           # a first position, or one that a window hides
    k[1][100, 0, 5] = k[1][100, 0, 9] = sign * np.inf
    k[2][6, 0, 9] = -sign * np.inf             # the last row's own
    odd = [{60: {0}, 88: {last}}, {1: {last}, 100: {0}}, {6: {0}}]
    pool = P.Pool(hip, lens, n_kv, hd, f16, 16, seed=3, k=k)
    rows = P.Rows(pool, sum(counts), heads, seed=5)
    rows.q[..., 5], rows.q[..., 9] = np.abs(rows.q[..., 5]) + 0.3, -np.abs(rows.q[..., 9]) - 0.3
    hip.upload(rows.d_q, rows.q)
    more = {} if counts == [1, 1, 1] else dict(q_first=_first(pool, counts), max_queries=max(counts))
    hip.paged_attn(pool.kv(), rows.op(window=window, n_sink=sinks, **more))
    _check(pool, rows, counts, window, sinks, odd)
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("counts", [[1, 1], [3, 2], [60, 50]])
def test_an_infinite_key_in_a_sequence_that_is_cut(hip, f16, counts):
    """One part of many holds it: the whole row is NaN, and the other kv head's rows are not."""
    lens = [3000, 2500]
    pool = P.Pool(hip, lens, 2, 64, f16, 64, seed=3)
    k = [x.copy() for x in pool.k]
    pool.close()
    k[0][700, 0, 5] = -np.inf
    k[1][2400, 1, 5] = -np.inf
    pool = P.Pool(hip, lens, 2, 64, f16, 64, seed=3, k=k)
    rows = P.Rows(pool, sum(counts), 8, seed=5)
    rows.q[..., 5] = np.abs(rows.q[..., 5]) + 0.3
    hip.upload(rows.d_q, rows.q)
    more = {} if counts == [1, 1] else dict(q_first=_first(pool, counts), max_queries=max(counts))
    hip.paged_attn(pool.kv(), rows.op(**more))
    _check(pool, rows, counts, 0, 0, [{700: {0}}, {2400: {1}}])
    pool.close()


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("chunk", [0, 3, 40])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_a_query_that_is_no_number_and_one_position(hip, f16, chunk, value):
    """A row that sees itself alone has one score, of either sign."""
    lens, m = [60, 60, 1], chunk or 1
    counts = [m, m, 1]
    pool = P.Pool(hip, lens, 1, 64, f16, 16, seed=6)
    rows = P.Rows(pool, sum(counts), 4, seed=3)
    ends = np.cumsum(counts) - 1
    for e in ends:
        rows.q[e, 1, 7] = rows.q[e, 2, 8] = value
    hip.upload(rows.d_q, rows.q)
    more = dict(q_first=_first(pool, counts), max_queries=m) if chunk else {}
    hip.paged_attn(pool.kv(), rows.op(window=1, **more))
    got = rows.result()
    assert np.isnan(got[ends][:, 1:3]).all()
    at = 0
    for s, c in enumerate(counts):
        for i in range(c):
            for h in range(4):
                if at + i in ends and h in (1, 2):
                    continue
                assert np.abs(got[at + i, h] - pool.v[s][lens[s] - c + i, 0].astype(np.float64)).max() <= 2.0 ** -20 * 6, (s, i, h)
        at += c
    pool.close()


@pytest.mark.parametrize("counts", [[1, 1], [3, 2], [50, 40]])
@pytest.mark.parametrize("sign", [1, -1])
def test_new_keys_that_a_half_cannot_hold(hip, counts, sign):
    """Infinite as the cache holds them, which no position may be lost to silently."""
    lens = [80, 60]
    pool = P.Pool(hip, lens, 2, 64, True, 16, seed=6)
    rows = P.Rows(pool, sum(counts), 4, seed=3, new=True)
    rows.q[..., 5] = np.abs(rows.q[..., 5]) + 0.3
    hip.upload(rows.d_q, rows.q)
    rows.k_new[counts[0] - 1, 1, 5] = sign * 1e6       # the first sequence's last position
    hip.upload(rows.d_kn, np.pad(rows.k_new.reshape(sum(counts), -1), ((0, 0), (0, rows.ks - 128))))
    more = {} if counts == [1, 1] else dict(q_first=_first(pool, counts), max_queries=max(counts))
    hip.paged_attn(pool.kv(), rows.op(**more))
    at = 0
    with np.errstate(over="ignore"):
        for s, m in enumerate(counts):
            pool.k[s][lens[s] - m:] = rows.k_new[at:at + m].astype(np.float16)
            pool.v[s][lens[s] - m:] = rows.v_new[at:at + m].astype(np.float16)
            at += m
    _check(pool, rows, counts, 0, 0, [{79: {1}}, {}])
    pool.close()
