"""Verification of drafted tokens through the C ABI, against the definition in 64 bits: tokens and counts are equal."""
import numpy as np
import pytest

from cera_amd import hip_api as A

pytestmark = pytest.mark.gpu


def _softmax(z, t):
    z = z.astype(np.float64) / float(np.float32(t))
    e = np.exp(z - z.max())
    return e / e.sum()


def _ok(z):
    return not np.isnan(z).any() and not (z == np.inf).any() and (z > -np.inf).any()


def _ref(target, draft, tokens, n, uniform, t):
    """(accepted, tokens, distance of the nearest decision from its border) of one sequence."""
    D = len(tokens)
    out, near = [-1] * (D + 1), 1.0
    if n > D:
        return 0, out, near
    for j in range(n + 1):
        if not _ok(target[j]):
            return j, out, near
        if t == 0:
            best = int(np.argmax(target[j]))
            if j < n and tokens[j] == best:
                out[j] = best
                continue
            out[j] = best
            return j, out, near
        p = weight = _softmax(target[j], t)
        if j < n:
            x = int(tokens[j])
            inside = 0 <= x < len(p)
            if draft is None:
                q = np.zeros_like(p)
                if inside:
                    q[x] = 1.0
            else:
                if not _ok(draft[j]):
                    return j, out, near
                q = _softmax(draft[j], t)
            if inside:
                near = min(near, abs(float(uniform[j]) * q[x] - p[x]) / max(p[x], 1e-300))
                if float(uniform[j]) * q[x] < p[x]:
                    out[j] = x
                    continue
            weight = np.maximum(p - q, 0)
            if not weight.sum() > 0:
                weight = p
        c = np.cumsum(weight)
        want = float(uniform[D]) * c[-1]
        hit = np.argmax(c > want) if (c > want).any() else np.flatnonzero(weight)[-1]
        near = min(near, np.abs(c - want).min() / c[-1])
        out[j] = int(hit)
        return j, out, near


def _run(hip, target, draft, tokens, counts, uniform, t, stride=0):
    S, D1, V = target.shape
    D, bufs = D1 - 1, []

    def dev(a, fill=None):
        if a is None:
            return None
        if stride and a.ndim == 3:
            b = np.full(a.shape[:2] + (stride,), np.nan, np.float32)
            b[..., :V] = a
            a = b
        bufs.append(hip.to_device(np.ascontiguousarray(a)))
        return bufs[-1]

    acc, nxt = dev(np.full(S + 1, 99, np.uint32)), dev(np.full((S + 1, D1), -99, np.int32))
    hip.verify_draft(A.VerifyDraft(n_seqs=S, max_draft=D, vocab=V, temperature=t, row_stride=stride, target=dev(target.astype(np.float32)),
                                   draft=dev(None if draft is None else draft.astype(np.float32)), tokens=dev(tokens.astype(np.int32)),
                                   n_draft=dev(None if counts is None else np.array(counts, np.uint32)), uniform=dev(uniform.astype(np.float32)),
                                   accepted=acc, out_tokens=nxt))
    a, n = hip.download(acc, S + 1, np.uint32), hip.download(nxt, (S + 1, D1), np.int32)
    assert a[S] == 99 and (n[S] == -99).all()
    for b in bufs:
        hip.free(b)
    return a[:S], n[:S]


def _case(seed, S, D, V, lookup, sharp=2.5):
    r = np.random.default_rng(seed)
    target = (r.standard_normal((S, D + 1, V)) * sharp).astype(np.float32)
    draft = None if lookup else (target[:, :D] + r.standard_normal((S, D, V))).astype(np.float32)
    tokens = ((target[:, :D] if lookup else draft) * (2 if lookup else 1) + r.gumbel(size=(S, D, V))).argmax(-1)
    return target, draft, tokens, r.random((S, D + 1)).astype(np.float32), r


def _check(hip, target, draft, tokens, counts, uniform, t, stride=0):
    S, D1, _ = target.shape
    acc, nxt = _run(hip, target, draft, tokens, counts, uniform, t, stride)
    for s in range(S):
        n = D1 - 1 if counts is None else counts[s]
        a, out, near = _ref(target[s], None if draft is None else draft[s], tokens[s], n, uniform[s], t)
        if near < 1e-12:        # 64-bit sums in another order may fall on the other side
            continue
        assert acc[s] == a and list(nxt[s]) == out, (s, acc[s], a, list(nxt[s]), out, near)


@pytest.mark.parametrize("lookup", [True, False])
@pytest.mark.parametrize("t", [0.0, 0.3, 1.0, 4.0])
@pytest.mark.parametrize("S,D,V", [(1, 1, 1), (3, 2, 2), (5, 4, 63), (4, 8, 1000), (3, 3, 4096), (3, 3, 4097), (7, 5, 32000), (2, 4, 128256), (70, 1, 513), (2, 64, 300)])
def test_decisions(hip, lookup, t, S, D, V):
    print("verify", lookup, t, S, D, V, flush=True)
    target, draft, tokens, uniform, r = _case(S * 7 + D + V, S, D, V, lookup)
    counts = [int(x) for x in r.integers(0, D + 1, S)]
    _check(hip, target, draft, tokens, None, uniform, t)
    _check(hip, target, draft, tokens, counts, uniform, t, stride=V + 3)


@pytest.mark.parametrize("lookup", [True, False])
def test_random_numbers_at_their_ends(hip, lookup):
    target, draft, tokens, uniform, _ = _case(3, 8, 3, 5000, lookup)
    for u in (0.0, 1 - 2.0 ** -24):
        uniform[:] = u
        _check(hip, target, draft, tokens, None, uniform, 0.7)


@pytest.mark.parametrize("t", [1e-3, 1e-6, 1e-20, 1e-38, 1e-44])
@pytest.mark.parametrize("lookup", [True, False])
def test_temperatures_at_which_the_largest_logit_is_all(hip, lookup, t):
    """Logits a quarter apart around -1000 and 3e37: weights of 1 and 0, whatever (logit / temperature) overflows or loses."""
    r = np.random.default_rng(2)
    S, D, V = 4, 3, 3000
    target = np.stack([[r.permutation(V) * 0.25 - 1000 for _ in range(D + 1)] for _ in range(S)]).astype(np.float32)
    target[0] = np.where(target[0] > -600, 3e37, -3e37) * (1 + (target[0] + 1000) / 4000)
    draft = target[:, :D].copy()
    draft[1, 2] = np.roll(draft[1, 2], 5)
    draft[2, 0] = np.roll(draft[2, 0], 1)
    tokens = draft.argmax(2).astype(np.int32)
    uniform = np.full((S, D + 1), 0.75, np.float32)
    acc, out = _run(hip, target, None if lookup else draft, tokens, None, uniform, t)
    best = target.argmax(2)
    for s, n in enumerate((3, 2, 0, 3)):
        assert acc[s] == n and list(out[s]) == list(best[s, :n + 1]) + [-1] * (D - n), (s, acc[s], out[s], best[s])


@pytest.mark.parametrize("t", [0.0, 1.0])
@pytest.mark.parametrize("lookup", [True, False])
def test_masked_tokens_and_bad_rows(hip, lookup, t):
    S, D, V = 9, 3, 9000
    target, draft, tokens, uniform, r = _case(4, S, D, V, lookup)
    keep = tokens[0, 0]
    target[0, 0, :] = -np.inf; target[0, 0, keep] = 1.5        # all weight on one token, the drafted one
    target[1, 0, tokens[1, 0]] = -np.inf                        # the drafted token is masked
    target[2, 1, 77] = np.nan
    target[3, 0, :] = -np.inf
    target[4, 2, 8999] = np.inf
    target[5, :, :4200] = -np.inf                               # the first chunk of the row has nothing
    tokens[6, 1] = V
    tokens[7, 0] = -1
    if draft is not None:
        draft[8, 1, :] = -np.inf
    _check(hip, target, draft, tokens, None, uniform, t)
    _check(hip, target, draft, tokens, [0, 3, 2, 1, 3, 2, 3, 3, 4], uniform, t)   # 4: more than there can be


def test_equal_distributions_and_ties(hip):
    target, draft, tokens, uniform, _ = _case(5, 6, 4, 3000, False)
    draft = target[:, :4].copy()                               # p = q: nothing is ever rejected
    acc, _ = _run(hip, target, draft, tokens, None, uniform, 1.0)
    assert (acc == 4).all()
    target[:] = 0
    target[:, :, [5, 900, 2999]] = 3                           # equal maxima: the lowest index
    tokens[:] = 5
    tokens[3:] = 900
    acc, nxt = _run(hip, target, None, tokens, None, uniform, 0.0)
    assert list(acc) == [4, 4, 4, 0, 0, 0] and (nxt[:3] == 5).all() and (nxt[3:, 0] == 5).all() and (nxt[3:, 1:] == -1).all()


def test_draws_follow_the_distribution(hip):
    """Accepted or drawn, the first token of many trials has the target's law: every count within five standard deviations."""
    V, N = 16, 40000
    r = np.random.default_rng(8)
    z, y = r.standard_normal(V), r.standard_normal(V)
    p, q = _softmax(z.astype(np.float32), 1), _softmax(y.astype(np.float32), 1)
    tokens = r.choice(V, size=(N, 1), p=q)
    acc, nxt = _run(hip, np.broadcast_to(z, (N, 2, V)).copy(), np.broadcast_to(y, (N, 1, V)).copy(), tokens, None, r.random((N, 2)), 1.0)
    got = np.bincount(nxt[:, 0], minlength=V)
    assert (np.abs(got - N * p) <= 5 * np.sqrt(N * p * (1 - p))).all()


def test_refusals(hip):
    ok = dict(n_seqs=1, max_draft=1, vocab=4, temperature=1.0, target=hip.malloc(64), tokens=hip.malloc(64), uniform=hip.malloc(64), accepted=hip.malloc(64), out_tokens=hip.malloc(64))
    for more, status in ((dict(target=None), 6), (dict(temperature=-0.5), 6), (dict(vocab=0), 4), (dict(max_draft=65), 4), (dict(row_stride=3), 4), (dict(n_seqs=65536), 4)):
        with pytest.raises(A.HipError) as e:
            hip.verify_draft(A.VerifyDraft(**{**ok, **more}))
        assert e.value.status == status
    hip.verify_draft(A.VerifyDraft(**{**ok, "n_seqs": 0}))


def test_the_same_call_many_times(hip):
    """A sequence's token is drawn by whichever of its workgroups is done last: the same one every time."""
    r = np.random.default_rng(8)
    S, D, V = 6, 3, 128256
    target = (r.standard_normal((S, D + 1, V)) * 2).astype(np.float32)
    draft = (target[:, :D] + r.standard_normal((S, D, V))).astype(np.float32)
    tokens = draft.argmax(2).astype(np.int32)
    bufs = [hip.to_device(x) for x in (target, draft, tokens)]
    d_u, d_acc, d_out = hip.malloc(S * (D + 1) * 4), hip.malloc(S * 4), hip.malloc(S * (D + 1) * 4)
    for k in range(40):
        u = r.random((S, D + 1)).astype(np.float32)
        hip.upload(d_u, u)
        hip.verify_draft(A.VerifyDraft(n_seqs=S, max_draft=D, vocab=V, temperature=0.9, target=bufs[0], draft=bufs[1], tokens=bufs[2], uniform=d_u, accepted=d_acc, out_tokens=d_out))
        got = hip.download(d_out, (S, D + 1), np.int32)
        if k % 10 == 0:
            for s in range(S):
                _, want, near = _ref(target[s], draft[s], tokens[s], D, u[s], 0.9)
                assert near > 1e-12 and list(got[s]) == list(want), (k, s)
        for _ in range(5):
            hip.verify_draft(A.VerifyDraft(n_seqs=S, max_draft=D, vocab=V, temperature=0.9, target=bufs[0], draft=bufs[1], tokens=bufs[2], uniform=d_u, accepted=d_acc, out_tokens=d_out))
            assert np.array_equal(got, hip.download(d_out, (S, D + 1), np.int32)), k
    for b in bufs + [d_u, d_acc, d_out]:
        hip.free(b)
