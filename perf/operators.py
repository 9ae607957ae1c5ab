"""The timed operators of a server that keeps many sequences in one pool of cache pages.

``attn`` cases are one layer's attention of a step: the new tokens' key and value rows go into the pages, then every new token
attends to its sequence (one token a sequence: the decode form, which may add its weights up per position; or a chunk of new
tokens a sequence), with or without a sliding window and first positions that stay visible.  ``evict`` cases bring every sequence
back to a budget of positions by those weights.  ``verify`` cases decide about drafted tokens and draw the next one.

``run`` computes them in plain torch operations, or with ``own`` set by the framework's entry points.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
SHAPES = {"32/8/128": (32, 8, 128), "24/8/128": (24, 8, 128), "28/4/128": (28, 4, 128), "32/8/64": (32, 8, 64), "12/2/128": (12, 2, 128),
          "16/16/64": (16, 16, 64), "8/1/128": (8, 1, 128), "40/8/128": (40, 8, 128)}


def _attn(shape, f16, page, seqs, longest, new, window, sinks, weights, spread):
    """new 0: the decode form; else the most new tokens of a sequence.  spread: lengths between longest / spread and longest."""
    return {"op": "attn", "shape": shape, "f16": f16, "page": page, "seqs": seqs, "longest": longest, "new": new, "window": window, "sinks": sinks,
            "weights": weights, "spread": spread}


def _evict(shape, f16, page, seqs, longest, budget, first, recent, spread):
    return {"op": "evict", "shape": shape, "f16": f16, "page": page, "seqs": seqs, "longest": longest, "budget": budget, "first": first, "recent": recent,
            "spread": spread}


def _verify(seqs, drafts, vocab, temperature, lookup):
    return {"op": "verify", "seqs": seqs, "drafts": drafts, "vocab": vocab, "temperature": temperature, "lookup": lookup}


def listed():
    return [
        # the first words of one reply: nothing but latency
        {"name": "decode_one", **_attn("32/8/64", True, 16, 1, 300, 0, 0, 0, False, 1)},
        # a step of a busy server: chats of very different lengths, weights collected for eviction
        {"name": "decode_batch", **_attn("32/8/128", True, 64, 32, 8000, 0, 0, 0, True, 16)},
        # two questions about long documents in a full-precision cache
        {"name": "decode_long", **_attn("32/8/128", False, 256, 2, 60001, 0, 0, 0, False, 2)},
        # endless chats: a window and the first four positions, seven query heads a key head
        {"name": "decode_window", **_attn("28/4/128", True, 32, 48, 20000, 0, 1024, 4, False, 8)},
        # a round of speculative decoding: up to five tokens a sequence to be verified
        {"name": "chunk_drafts", **_attn("32/8/128", True, 64, 16, 4000, 5, 0, 0, False, 4)},
        # a long prompt's chunk in the middle of a document
        {"name": "chunk_prompt", **_attn("32/8/128", True, 64, 1, 6000, 2048, 0, 0, False, 1)},
        # the same behind a window with four first positions
        {"name": "chunk_window", **_attn("24/8/128", True, 128, 2, 9001, 1500, 1024, 4, False, 2)},
        # prompts of several users side by side, full precision, heads of 64
        {"name": "chunk_users", **_attn("32/8/64", False, 16, 6, 700, 700, 0, 0, False, 8)},
        # one chat cut by a few positions
        {"name": "evict_one", **_evict("32/8/64", False, 32, 1, 600, 512, 4, 64, 1)},
        # all chats of a server brought back to half of the longest
        {"name": "evict_batch", **_evict("32/8/128", True, 64, 16, 8192, 4096, 4, 512, 2)},
        # drafts found in the prompt, one sequence, a large vocabulary
        {"name": "verify_one", **_verify(1, 4, 128256, 0.8, True)},
        # drafts of a small model for a batch
        {"name": "verify_batch", **_verify(64, 5, 32000, 1.0, False)},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "chunk", "chunk", "chunk", "evict", "evict", "verify", "verify"])
    shape, f16, page = rng.choice(sorted(SHAPES)), rng.random() < 0.6, rng.choice([16, 32, 64, 128, 256])
    window, sinks = rng.choice([(0, 0), (_log_int(rng, 16, 4096), rng.choice([0, 1, 4, 33]))])
    if op == "attn":
        longest = _log_int(rng, 1, 60000)
        seqs = _log_int(rng, 1, max(1, min(64, 80000 // longest)))
        return _attn(shape, f16, page, seqs, longest, 0, window, sinks, rng.random() < 0.4, rng.choice([1, 2, 16]))
    if op == "chunk":
        longest = _log_int(rng, 2, 8000)
        new = _log_int(rng, 2, min(longest, 1500))
        seqs = _log_int(rng, 1, max(1, min(24, 6_000_000 // (longest * new))))
        return _attn(shape, f16, page, seqs, longest, new, window, sinks, False, rng.choice([1, 2, 16]))
    if op == "evict":
        longest = _log_int(rng, 64, 30000)
        seqs = _log_int(rng, 1, max(1, min(32, 50000 // longest)))
        budget = _log_int(rng, max(8, longest // 16), longest)
        first = rng.choice([0, 1, 4])
        return _evict(shape, f16, page, seqs, longest, budget, first, rng.randint(0, (budget - first) // 2), rng.choice([1, 2, 4]))
    vocab, drafts = _log_int(rng, 1000, 152064), rng.randint(1, 8)
    return _verify(_log_int(rng, 1, max(1, min(64, 20_000_000 // (vocab * (2 * drafts + 1))))), drafts, vocab, rng.choice([0.0, 0.6, 1.0]), rng.random() < 0.4)


def _plan(case):
    """Lengths and counts of new tokens by sequence: a matter of the case, so that its work is known without the inputs."""
    r = random.Random(case["longest"] * 131 + case["seqs"])
    lens = [case["longest"]] + [_log_int(r, max(1, case["longest"] // case["spread"]), case["longest"]) for _ in range(case["seqs"] - 1)]
    most = max(1, case.get("new", 0))
    new = [min(lens[0], most)] + [min(n, r.randint(max(1, most // 2), most)) for n in lens[1:]]
    return lens, new


def _seen(position, window, sinks):
    """Positions that a query at `position` sees."""
    return position + 1 if not window else min(position + 1, window + min(sinks, max(0, position + 1 - window)))


def work(case):
    if case["op"] == "verify":
        rows = case["seqs"] * (case["drafts"] + 1 + (0 if case["lookup"] or not case["temperature"] else case["drafts"]))
        return {"bytes": 4 * rows * case["vocab"], "flops": 4 * rows * case["vocab"]}
    heads, kv, hd = SHAPES[case["shape"]]
    row = 2 * kv * hd * (2 if case["f16"] else 4)          # a position's keys and values
    lens, new = _plan(case)
    if case["op"] == "evict":
        cut = [n for n in lens if n > case["budget"]]
        # weights read; what is kept behind the first positions read and written
        return {"bytes": sum(4 * kv * n + 2 * (case["budget"] - case["first"]) * (row + 4 * kv) for n in cut) + 8 * kv * len(lens), "flops": kv * sum(lens)}
    w, k = case["window"], case["sinks"]
    read = sum(_seen(n - 1, w, k) if m == 1 else min(n, _seen(n - m, w, k) + m - 1) for n, m in zip(lens, new))
    pairs = sum(_seen(p, w, k) for n, m in zip(lens, new) for p in range(n - m, n))
    fresh = sum(new)
    return {"bytes": read * row + fresh * (2 * heads * hd * 4 + 2 * kv * hd * 4 + row) + (8 * kv * read if case["weights"] else 0),
            "flops": 4 * pairs * heads * hd}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s, dtype=torch.float32: torch.randn(*s, generator=g, device=DEV, dtype=torch.float32).to(dtype)  # noqa: E731
    st = {"case": case}
    if case["op"] == "verify":
        n, d, v = case["seqs"], case["drafts"], case["vocab"]
        st["target"] = randn(n, d + 1, v) * 2.5
        st["draft"] = None if case["lookup"] else st["target"][:, :d].contiguous() + randn(n, d, v)
        # a lookup's tokens are often the likely ones; a draft model's come from its own distribution
        gumbel = -torch.log(-torch.log(torch.rand(n, d, v, generator=g, device=DEV).clamp(1e-30, 1 - 1e-7)))
        st["tokens"] = ((st["target"][:, :d] * 4 if case["lookup"] else st["draft"] / (case["temperature"] or 0.05)) + gumbel).argmax(-1).int().contiguous()
        st["counts"] = torch.tensor([d - i % 2 if d > 1 else d for i in range(n)], device=DEV, dtype=torch.int32)
        st["uniform"] = torch.rand(n, d + 1, generator=g, device=DEV)
        st["accepted"] = torch.zeros(n, device=DEV, dtype=torch.int32)
        st["next"] = torch.zeros(n, d + 1, device=DEV, dtype=torch.int32)
        return st
    heads, kv, hd = SHAPES[case["shape"]]
    page, n = case["page"], case["seqs"]
    lens, new = _plan(case)
    need = [-(-x // page) for x in lens]
    cols = max(need)
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = [[order.pop() for _ in range(c)] + [-1] * (cols - c) for c in need]
    st["table"] = torch.tensor(table, device=DEV, dtype=torch.int32)
    st["lens"] = torch.tensor(lens, device=DEV, dtype=torch.int32)
    e = torch.float16 if case["f16"] else torch.float32
    st["k"], st["v"] = randn(pages, kv, page, hd, dtype=e), randn(pages, kv, page, hd, dtype=e)
    cap = cols * page
    if case["op"] == "evict":
        # collected weights: a few positions have most of it
        st["collected"] = torch.rand(n, kv, cap, generator=g, device=DEV) ** 8 * 20
        st["mass"] = st["collected"].clone()
        st["new_lens"] = torch.zeros(n, device=DEV, dtype=torch.int32)
        st["kept"] = torch.zeros(n, kv, case["budget"], device=DEV, dtype=torch.int32)
        return st
    rows = sum(new)
    st["q"] = randn(rows, heads, hd) * 1.5
    st["k_new"], st["v_new"] = randn(rows, kv, hd), randn(rows, kv, hd)
    st["first"] = torch.tensor([sum(new[:i]) for i in range(n + 1)], device=DEV, dtype=torch.int32) if case["new"] else None
    st["mass"] = torch.zeros(n, kv, cap, device=DEV) if case["weights"] else None
    st["out"] = torch.zeros(rows, heads, hd, device=DEV)
    return st


# ---- the framework's entry points ------------------------------------------------------------------------------------

_ctx = None


def _own(st):
    global _ctx
    from cera_amd import hip_api as A

    if _ctx is None:
        _ctx = A.Context(0)
    case = st["case"]
    at = lambda name: st[name].data_ptr() if st.get(name) is not None else None  # noqa: E731
    if case["op"] == "verify":
        _ctx.verify_draft(A.VerifyDraft(n_seqs=case["seqs"], max_draft=case["drafts"], vocab=case["vocab"], row_stride=case["vocab"],
                                        temperature=case["temperature"], target=at("target"), draft=at("draft"), tokens=at("tokens"),
                                        n_draft=at("counts"), uniform=at("uniform"), accepted=at("accepted"), out_tokens=at("next")))
        return st["accepted"], st["next"]
    heads, kv, hd = SHAPES[case["shape"]]
    cache = A.PagedKV(kv_type=1 if case["f16"] else 0, n_kv_heads=kv, head_dim=hd, page_size=case["page"], n_pages=st["k"].shape[0],
                      n_seqs=case["seqs"], max_pages=st["table"].shape[1], k=at("k"), v=at("v"), table=at("table"), lens=at("lens"))
    if case["op"] == "evict":
        st["mass"].copy_(st["collected"])           # as decode steps have collected it
        _ctx.paged_evict(cache, A.PagedEvict(mass=at("mass"), mass_stride=st["mass"].shape[2], budget=case["budget"], n_first=case["first"],
                                             n_recent=case["recent"], max_len=case["longest"], new_lens=at("new_lens"), kept=at("kept")))
        return {"lens": st["new_lens"], "kept": st["kept"], "k": st["k"], "v": st["v"], "mass": st["mass"]}
    _ctx.paged_attn(cache, A.PagedAttn(q=at("q"), k_new=at("k_new"), v_new=at("v_new"), out=at("out"), mass=at("mass"), q_first=at("first"),
                                       mass_stride=st["mass"].shape[2] if case["weights"] else 0, n_rows=st["q"].shape[0],
                                       max_queries=max(1, case["new"]), n_heads=heads, scale=1 / math.sqrt(hd), window=case["window"],
                                       n_sink=case["sinks"], max_len=case["longest"]))
    return {"out": st["out"], "k": st["k"], "v": st["v"], **({"mass": st["mass"]} if case["weights"] else {})}


# ---- the plain forms -------------------------------------------------------------------------------------------------


def _slots(st, positions):
    """(page, slot) of [sequence, position] pairs; a page that a table does not name is page 0, for positions that are masked."""
    page = st["case"]["page"]
    at = torch.gather(st["table"].long(), 1, (positions // page).clamp(0, st["table"].shape[1] - 1))
    return at.clamp(min=0), positions % page


def _plain_attn(st):
    case = st["case"]
    heads, kv, hd = SHAPES[case["shape"]]
    n, longest, lens = case["seqs"], case["longest"], st["lens"].long()
    rows = st["q"].shape[0]
    first = st["first"].long() if st["first"] is not None else torch.arange(n + 1, device=DEV)
    counts = first[1:] - first[:-1]
    # every row's sequence and position; its key and value go into their page
    row = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(first[1:].contiguous(), row, right=True)
    pos = (lens - counts)[seq] + row - first[seq]
    page, slot = st["table"].long()[seq, pos // case["page"]], pos % case["page"]
    st["k"][page, :, slot] = st["k_new"].to(st["k"].dtype)
    st["v"][page, :, slot] = st["v_new"].to(st["v"].dtype)
    # all sequences padded to the longest, all chunks to the largest
    key = torch.arange(longest, device=DEV)
    page, slot = _slots(st, key.expand(n, longest))
    k = st["k"][page, :, slot].float().transpose(1, 2)                       # [n][kv][longest][hd]
    v = st["v"][page, :, slot].float().transpose(1, 2)
    most = max(1, case["new"])
    padded = torch.zeros(n, most, heads, hd, device=DEV)
    padded[seq, row - first[seq]] = st["q"]
    where = (lens - counts)[:, None] + torch.arange(most, device=DEV)        # [n][most] positions of the queries
    near = key > where[..., None] - case["window"] if case["window"] else torch.ones(1, dtype=torch.bool, device=DEV)
    seen = (key <= where[..., None]) & (near | (key < case["sinks"])) & (key < lens[:, None, None])      # [n][most][longest]
    q = padded.view(n, most, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, hd)          # [n][kv][group * most][hd]
    s = torch.matmul(q, k.transpose(2, 3)).view(n, kv, heads // kv, most, longest) * (1 / math.sqrt(hd))
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(s - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p.reshape(n, kv, -1, longest), v).view(n, kv, heads // kv, most, hd).permute(0, 3, 1, 2, 4).reshape(n, most, heads, hd)
    out = {"out": o[seq, row - first[seq]], "k": st["k"], "v": st["v"]}
    if case["weights"]:
        st["mass"][:, :, :longest] += p.sum(dim=(2, 3))
        out["mass"] = st["mass"]
    return out


def _plain_evict(st):
    case = st["case"]
    st["mass"].copy_(st["collected"])               # as decode steps have collected it
    kv = SHAPES[case["shape"]][1]
    n, budget, longest, lens = case["seqs"], case["budget"], case["longest"], st["lens"].long()
    key = torch.arange(longest, device=DEV)
    mass = st["mass"][:, :, :longest]
    middle = (key >= case["first"]) & (key < (lens - case["recent"])[:, None])
    cut = (lens > budget)[:, None]
    # rank of a position: the ones that stay in any case, then by weight, the lowest index first among equals, then what is no position
    order = torch.where(middle[:, None], mass, torch.where(key < lens[:, None], math.inf, -math.inf)[:, None])
    ranked = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.sort(ranked, dim=-1).values                                                  # [n][kv][budget], the order of positions
    slots = torch.arange(min(budget, longest), device=DEV)
    kept = torch.where(cut[..., None], kept, slots.expand(n, kv, -1))
    live = (slots < lens[:, None])[:, None].expand_as(kept)
    head = torch.arange(kv, device=DEV)[None, :, None].expand_as(kept)
    src, at = _slots(st, kept.reshape(n, -1))
    dst, to = _slots(st, slots.expand(n, kv, -1).reshape(n, -1))
    src, at, dst, to = (x.view_as(kept)[live] for x in (src, at, dst, to))
    rows_k, rows_v = st["k"][src, head[live], at], st["v"][src, head[live], at]
    st["k"][dst, head[live], to] = rows_k
    st["v"][dst, head[live], to] = rows_v
    moved = torch.gather(mass, 2, kept)
    mass[:, :, :slots.numel()] = torch.where(live, moved, mass[:, :, :slots.numel()])
    st["kept"].fill_(-1)
    st["kept"][:, :, :slots.numel()] = torch.where(live, kept, -1).int()
    st["new_lens"].copy_(lens.clamp(max=budget))
    return {"lens": st["new_lens"], "kept": st["kept"], "k": st["k"], "v": st["v"], "mass": st["mass"]}


def _plain_verify(st):
    case = st["case"]
    n, d, t = case["seqs"], case["drafts"], case["temperature"]
    count, x = st["counts"].long(), st["tokens"].long()
    live = torch.arange(d, device=DEV) < count[:, None]
    if not t:
        best = st["target"].argmax(-1)
        good = (best[:, :d] == x) & live
        accepted = good.long().cumprod(1).sum(1)
        following = best.gather(1, accepted[:, None])
    else:
        # 64 bits: a draw next to a border between two tokens
        z = st["target"].double() / t
        p = torch.exp(z - z.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        if st["draft"] is None:
            q = torch.zeros_like(p[:, :d]).scatter_(2, x[..., None], 1.0)
        else:
            y = st["draft"].double() / t
            q = torch.exp(y - y.amax(-1, keepdim=True))
            q = q / q.sum(-1, keepdim=True)
        px, qx = p[:, :d].gather(2, x[..., None])[..., 0], q.gather(2, x[..., None])[..., 0]
        good = (st["uniform"][:, :d].double() * qx < px) & live
        accepted = good.long().cumprod(1).sum(1)
        at = torch.arange(n, device=DEV)
        rest = (p[at, accepted] - q[at, accepted.clamp(max=d - 1)]).clamp(min=0)
        weight = torch.where((accepted < count)[:, None], rest, p[at, accepted])
        sums = weight.cumsum(-1)
        following = torch.searchsorted(sums, (st["uniform"][:, d:].double() * sums[:, -1:]).contiguous(), right=True).clamp(max=case["vocab"] - 1)
    tokens = torch.cat([x, x[:, :1]], 1)
    slot = torch.arange(d + 1, device=DEV)
    tokens = torch.where(slot < accepted[:, None], tokens, torch.where(slot == accepted[:, None], following, -1))
    return accepted.int(), tokens.int()


def run(st):
    if own:
        return _own(st)
    return {"attn": _plain_attn, "evict": _plain_evict, "verify": _plain_verify}[st["case"]["op"]](st)


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "verify":
        return _exact_verify(st)
    lens = st["lens"].tolist()
    table, page = st["table"].tolist(), case["page"]
    places = [torch.tensor([[table[s][t // page], t % page] for t in range(n)], device=DEV).T for s, n in enumerate(lens)]
    heads, kv, hd = SHAPES[case["shape"]]
    k, v = st["k"].double(), st["v"].double()
    if case["op"] == "evict":
        mass, kept = st["collected"].double(), torch.full((case["seqs"], kv, case["budget"]), -1, dtype=torch.int32)
        for s, n in enumerate(lens):
            for h in range(kv):
                ids = list(range(n))
                if n > case["budget"]:
                    w = st["collected"][s, h].tolist()
                    mid = sorted(range(case["first"], n - case["recent"]), key=lambda t: (-w[t], t))[: case["budget"] - case["first"] - case["recent"]]
                    ids = list(range(case["first"])) + sorted(mid) + list(range(n - case["recent"], n))
                kept[s, h, : len(ids)] = torch.tensor(ids, dtype=torch.int32)
                i = torch.tensor(ids, device=DEV)
                (a, b), (c, d) = places[s][:, i], places[s][:, : len(ids)]
                k[c, h, d], v[c, h, d] = k[a, h, b], v[a, h, b]
                mass[s, h, : len(ids)] = mass[s, h, i]
        return {"lens": [min(n, case["budget"]) for n in lens], "kept": kept, "k": k, "v": v, "mass": mass}
    _, new = _plan(case)
    out = torch.zeros(sum(new), heads, hd, device=DEV, dtype=torch.float64)
    mass = torch.zeros(st["mass"].shape, device=DEV, dtype=torch.float64) if case["weights"] else None
    at = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        a, b = places[s]
        k[a[n - m:], :, b[n - m:]] = st["k_new"][at: at + m].to(st["k"].dtype).double()
        v[a[n - m:], :, b[n - m:]] = st["v_new"][at: at + m].to(st["v"].dtype).double()
        t, P = torch.arange(n, device=DEV), torch.arange(n - m, n, device=DEV)[:, None]
        hidden = t > P
        if case["window"]:
            hidden = hidden | ((t <= P - case["window"]) & (t >= case["sinks"]))
        for h in range(heads):
            kk, vv = k[a, h * kv // heads, b], v[a, h * kv // heads, b]
            w = torch.softmax((st["q"][at: at + m, h].double() @ kk.T / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1)
            out[at: at + m, h] = w @ vv
            if mass is not None:
                mass[s, h * kv // heads, :n] += w.sum(0)
        at += m
    return {"out": out, "k": k, "v": v, **({"mass": mass} if mass is not None else {})}


def _exact_verify(st):
    case = st["case"]
    d, temperature = case["drafts"], case["temperature"]
    accepted, tokens = [], []
    for s in range(case["seqs"]):
        count, u = int(st["counts"][s]), st["uniform"][s].tolist()
        x, row = st["tokens"][s].tolist(), []
        law = lambda z: torch.softmax(z.double() / temperature, 0) if temperature else torch.zeros_like(z, dtype=torch.float64).index_fill_(0, z.argmax(), 1.0)  # noqa: E731
        weight = None
        for i in range(count):
            p = law(st["target"][s, i])
            if not temperature or st["draft"] is None:
                q = torch.zeros_like(p)
                q[x[i]] = 1.0
            else:
                q = law(st["draft"][s, i])
            if not u[i] * float(q[x[i]]) < float(p[x[i]]):
                weight = (p - q).clamp(min=0)
                break
            row.append(x[i])
        if weight is None:
            weight = law(st["target"][s, count])
        sums = weight.cumsum(0)
        row.append(int((sums > u[d] * sums[-1]).to(torch.uint8).argmax()))
        accepted.append(len(row) - 1)
        tokens.append(row + [-1] * (d + 1 - len(row)))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)
