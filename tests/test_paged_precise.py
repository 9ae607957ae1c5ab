"""What the bound of the precise inputs (paged_precise) tells apart, on the CPU: all parts pass it, and without any one of them it fails."""
import numpy as np
import pytest

import paged_precise as Q

SCALE = 0.125


def _error(f16, q_parts, k_parts, pairs):
    """Largest error against the bound with these parts of q and k (None: as they are) and these products (weight part, value part)."""
    k, v, q, ids = Q.make(5, [60], 40, 4, 1, 64, f16, 1)
    k, v, ids = k[0], v[0], ids[0]
    out, bound = Q.exact(q, k, v, ids, SCALE)
    qq = q.astype(np.float64) if q_parts is None else sum(Q.halves(q)[:q_parts])
    kk = k[ids, 0].astype(np.float64) if k_parts is None else sum(Q.halves(k[ids, 0])[:k_parts])
    s = qq @ kk.T * SCALE
    w = np.exp2((s - s.max(-1, keepdims=True)) * np.log2(np.e))
    wp, vp = (Q.halves(w * 2.0 ** 14), [v[ids, 0].astype(np.float64)]) if f16 else (Q.thirds(w), Q.thirds(v[ids, 0]))
    o = sum(wp[i] @ vp[j] for i, j in pairs) / (w.sum(-1, keepdims=True) * (2.0 ** 14 if f16 else 1))
    return (np.abs(o - out) / (bound * out)).max()


SIX = [(0, 0), (1, 0), (0, 1), (2, 0), (1, 1), (0, 2)]


def test_all_parts_pass():
    assert _error(True, 2, None, [(0, 0), (1, 0)]) < 0.5
    assert _error(False, 2, 2, SIX) < 0.5
    assert _error(False, None, None, SIX) < 0.5


@pytest.mark.parametrize("q_parts,k_parts,pairs", [(1, 2, SIX), (2, 1, SIX)] + [(2, 2, [p for p in SIX if p != gone]) for gone in SIX])
def test_a_part_that_is_left_out_of_an_f32_cache(q_parts, k_parts, pairs):
    assert _error(False, q_parts, k_parts, pairs) > 1.5


@pytest.mark.parametrize("q_parts,pairs", [(1, [(0, 0), (1, 0)]), (2, [(0, 0)])])
def test_a_part_that_is_left_out_of_a_half_cache(q_parts, pairs):
    assert _error(True, q_parts, None, pairs) > 1.5
