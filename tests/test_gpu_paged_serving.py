"""A server's steps on one paged cache: prompts, decoding with weights, eviction, drafts and their verification, a roll-back.

The reference runs the same steps in 64 bits on its own cache (keys and values as the cache holds them) and takes over only the
decisions that it checked: what an eviction kept and which drafts were accepted."""
import numpy as np
import pytest

import paged_util as P
from cera_amd import hip_api as A
from test_gpu_verify_draft import _ref as verify_ref

pytestmark = pytest.mark.gpu

HEADS, KV = 6, 2


class Server:
    def __init__(self, hip, f16, hd, page, window, sinks, seed):
        self.hip, self.r = hip, np.random.default_rng(seed)
        self.window, self.sinks = window, sinks
        self.lens = [0, 0, 0]
        self.pool = P.Pool(hip, [160, 160, 160], KV, hd, f16, page, seed=seed)      # room for 160 positions each
        self.pool.k = [np.zeros((0, KV, hd), self.pool.dtype) for _ in self.lens]
        self.pool.v = [np.zeros((0, KV, hd), self.pool.dtype) for _ in self.lens]
        self.cap = self.pool.cols * page
        self.mass = np.zeros((3, KV, self.cap))
        self.mass_bound = np.zeros_like(self.mass)
        self.d_mass = self.pool.dev(np.zeros((3, KV, self.cap), np.float32))

    def step(self, counts, decode):
        """New rows of every sequence, their attention against the reference; the device's out."""
        pool, hip = self.pool, self.hip
        rows = P.Rows(pool, sum(counts), HEADS, seed=int(self.r.integers(1 << 30)), new=True)
        self.lens = [n + m for n, m in zip(self.lens, counts)]
        hip.upload(pool.d_lens, np.array(self.lens, np.uint32))
        if decode:
            op = rows.op(window=self.window, n_sink=self.sinks, mass=self.d_mass, mass_stride=self.cap, mass_fresh=1)
        else:
            first = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
            op = rows.op(window=self.window, n_sink=self.sinks, q_first=pool.dev(first), max_queries=max(counts))
        hip.paged_attn(pool.kv(), op)
        got, at = rows.result(), 0
        for s, m in enumerate(counts):
            pool.k[s] = np.concatenate([pool.k[s][:self.lens[s] - m], rows.k_new[at:at + m].astype(pool.dtype)])
            pool.v[s] = np.concatenate([pool.v[s][:self.lens[s] - m], rows.v_new[at:at + m].astype(pool.dtype)])
            out, bound, mass, mb = P.attn_ref(rows.q[at:at + m], pool.k[s], pool.v[s], m, 1 / np.sqrt(pool.hd), self.window, self.sinks)
            assert (np.abs(got[at:at + m] - out) <= bound).all(), s
            if decode:
                n = self.lens[s]
                self.mass[s, :, n - 1] = self.mass_bound[s, :, n - 1] = 0
                self.mass[s, :, :n] += mass
                # the step's weights, their sum over the heads and its sum with what was there
                self.mass_bound[s, :, :n] += mb + (1 + HEADS // KV) * 2.0 ** -24 * (self.mass[s, :, :n] + 1)
                dev = hip.download(self.d_mass, (3, KV, self.cap), np.float32)[s, :, :n]
                assert (np.abs(dev - self.mass[s, :, :n]) <= self.mass_bound[s, :, :n]).all(), s
            at += m
        return got

    def evict(self, budget, first, recent):
        pool, hip = self.pool, self.hip
        d_new, d_kept = pool.dev(np.zeros(3, np.uint32)), pool.dev(np.zeros((3, KV, budget), np.int32))
        hip.paged_evict(pool.kv(), A.PagedEvict(mass=self.d_mass, mass_stride=self.cap, new_lens=d_new, kept=d_kept, budget=budget, n_first=first, n_recent=recent))
        kept, new = hip.download(d_kept, (3, KV, budget), np.int32), hip.download(d_new, 3, np.uint32)
        for s, n in enumerate(self.lens):
            m = min(n, budget)
            assert new[s] == m
            k, v = pool.k[s][:m].copy(), pool.v[s][:m].copy()
            for g in range(KV):
                ids = kept[s, g, :m]
                assert (np.diff(ids) > 0).all() and (kept[s, g, m:] == -1).all()
                if n > budget:
                    assert list(ids[:first]) == list(range(first)) and list(ids[m - recent:]) == list(range(n - recent, n))
                    gone = np.setdiff1d(np.arange(n), ids)
                    mid = ids[first:m - recent]
                    w, e = self.mass[s, g], self.mass_bound[s, g]
                    # none that went weighs surely more than one that stayed
                    assert (w[gone] - e[gone]).max() <= (w[mid] + e[mid]).min()
                k[:, g], v[:, g] = pool.k[s][ids, g], pool.v[s][ids, g]
                self.mass[s, g, :m], self.mass_bound[s, g, :m] = self.mass[s, g, ids], self.mass_bound[s, g, ids]
            pool.k[s], pool.v[s] = k, v
            self.lens[s] = m
        self.same_rows()

    def same_rows(self):
        for s, n in enumerate(self.lens):
            k, v = self.pool.rows(s, n)
            assert np.array_equal(k, self.pool.k[s][:n]) and np.array_equal(v, self.pool.v[s][:n])

    def drafts(self, D, temperature):
        """A chunk of drafts and the row behind them, verified; the rejected ones' positions are given back."""
        pool, hip, r = self.pool, self.hip, self.r
        out = self.step([D + 1] * 3, decode=False)
        V = 1500
        head = r.standard_normal((HEADS * pool.hd, V)).astype(np.float32) * np.float32(0.5)
        target = (out.reshape(3 * (D + 1), -1) @ head).reshape(3, D + 1, V)
        draft = (target[:, :D] + r.standard_normal((3, D, V)) * 0.5).astype(np.float32)
        tokens = np.array([[int(np.argmax(draft[s, i])) for i in range(D)] for s in range(3)], np.int32)
        u = r.random((3, D + 1)).astype(np.float32)
        d_acc, d_out = pool.dev(np.zeros(3, np.uint32)), pool.dev(np.zeros((3, D + 1), np.int32))
        hip.verify_draft(A.VerifyDraft(n_seqs=3, max_draft=D, vocab=V, temperature=temperature, target=pool.dev(target), draft=pool.dev(draft), tokens=pool.dev(tokens),
                                       uniform=pool.dev(u), accepted=d_acc, out_tokens=d_out))
        acc, got = hip.download(d_acc, 3, np.uint32), hip.download(d_out, (3, D + 1), np.int32)
        for s in range(3):
            want, toks, near = verify_ref(target[s], draft[s], tokens[s], D, u[s], temperature)
            assert near > 1e-9 and acc[s] == want and list(got[s]) == list(toks), s
            self.lens[s] -= D - int(acc[s])      # the next token's row is written by the next step
        return acc


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd,page,window,sinks,temperature", [(64, 16, 0, 0, 0.8), (128, 32, 24, 4, 0.0)])
def test_a_server_s_steps(hip, f16, hd, page, window, sinks, temperature):
    sv = Server(hip, f16, hd, page, window, sinks, seed=hd + f16)
    sv.step([40, 9, 70], decode=False)        # prompts
    for _ in range(3):
        sv.step([1, 1, 1], decode=True)
    sv.evict(32, 2, 8)
    assert sv.lens == [32, 12, 32]
    for _ in range(2):
        sv.step([1, 1, 1], decode=True)
    total = 0
    for _ in range(3):
        total += int(sv.drafts(4, temperature).sum())
        sv.step([1, 1, 1], decode=True)       # over a rejected draft's rows
    assert 0 < total < 36                     # some of the drafts went each way
    sv.step([0, 20, 0], decode=False)         # one sequence gets more to read
    sv.evict(16, 0, 4)
    assert sv.lens == [16, 16, 16]
    sv.step([1, 1, 1], decode=True)
    sv.same_rows()
    sv.pool.close()
