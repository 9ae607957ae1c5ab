"""Verification at temperature 0, which reads neither random numbers nor a draft's distribution."""
import numpy as np
import pytest

from cera_amd import hip_api as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,D,V", [(1, 1, 5), (5, 4, 32000), (3, 64, 1025)])
def test_without_random_numbers(hip, S, D, V):
    r = np.random.default_rng(S)
    target = r.standard_normal((S, D + 1, V)).astype(np.float32)
    best = target.argmax(2)
    tokens = best[:, :D].astype(np.int32)
    n = [D, 0, D // 2, D, 1][:S]
    for s in range(S):
        if n[s] < D:
            tokens[s, n[s]] = (tokens[s, n[s]] + 1) % V
    bufs = [hip.to_device(x) for x in (target, tokens, np.zeros(S, np.uint32), np.zeros((S, D + 1), np.int32))]
    hip.verify_draft(A.VerifyDraft(n_seqs=S, max_draft=D, vocab=V, temperature=0.0, target=bufs[0], tokens=bufs[1], accepted=bufs[2], out_tokens=bufs[3]))
    acc, out = hip.download(bufs[2], S, np.uint32), hip.download(bufs[3], (S, D + 1), np.int32)
    for s in range(S):
        assert acc[s] == n[s] and list(out[s]) == list(best[s, :n[s] + 1]) + [-1] * (D - n[s])
    for b in bufs:
        hip.free(b)
