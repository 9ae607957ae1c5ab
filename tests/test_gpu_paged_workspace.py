"""The workspace of weights by position, whose size follows the longest sequence."""
import ctypes as C

import numpy as np
import pytest

import paged_util as P
from cera_amd import hip_api as A

pytestmark = pytest.mark.gpu


def _free_bytes():
    rt = C.CDLL("libamdhip64.so")
    free, total = C.c_size_t(), C.c_size_t()
    assert rt.hipMemGetInfo(C.byref(free), C.byref(total)) == 0
    return free.value


def test_a_max_len_that_rises_from_call_to_call(hip):
    """Memory is taken anew a few times, not with every call: each time waits for all queued work."""
    ctx = A.Context(0)
    lens, heads, n_kv = [20] * 16, 64, 4
    pool = P.Pool(ctx, lens, n_kv, 64, True, 256, seed=3, max_pages=136)
    cap = pool.cols * pool.page
    d_mass = pool.dev(np.zeros((16, n_kv, cap), np.float32))
    rows = P.Rows(pool, 16, heads, seed=4)
    taken, before = 0, None
    for max_len in range(1024, cap, 512):          # 4 KB of scores a position: 2 MB more each time
        ctx.paged_attn(pool.kv(), rows.op(mass=d_mass, mass_stride=cap, max_len=max_len))
        now = _free_bytes()
        taken += before is not None and now != before
        before = now
    print("taken anew", taken, flush=True)
    assert 1 <= taken <= 10                        # each time at least half as large again: 34 < 1.5^9
    got = rows.result()
    for s in range(16):
        out, bound, _, _ = P.attn_ref(rows.q[s:s + 1], pool.k[s], pool.v[s], 1, 0.125, 0, 0)
        assert (np.abs(got[s:s + 1] - out) <= bound).all()
    pool.close()
    ctx.close()
