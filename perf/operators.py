"""Cases of the operators behind sampling several continuations of one prompt.

A prompt is computed once, forked into many sequences whose page tables share its full pages, and the sequences are
decoded together, one token at a time or several drafted tokens at a time:

* ``attn``: attention of one or a few query tokens a sequence over the paged cache, where the sequences of a group
  share the pages of a long prefix (``attn_shared``);
* ``copy``: the fork's data, pages of every layer copied to fresh pages (``kv_copy_pages``);
* ``compact``: live pages moved to the lowest page ids in every layer, with the rewritten tables (``kv_compact``);
* ``verify``: drafted tokens accepted or rejected against the target's probabilities, the token that follows, and the
  probabilities of what is emitted (``verify_sampled``).

Each case is run in a plain form of elementary torch operations in 32 bits (``own = False``) or through
``mod_b200.ops.native`` (``own = True``).  The cache layout is the engine's: K ``[pages, kv heads, 16, dim]`` and V
``[pages, kv heads, dim, 16]`` in bf16, tables and lengths in int32.
"""
import math
import random

import torch

own = False

PAGE = 16
DEV = "cuda"


def listed():
    return [
        # four samples of a short prompt on the 0.6B shape: launch latency is all that counts
        {"name": "attn tiny", "op": "attn", "heads": 16, "kv_heads": 8, "dim": 128, "groups": 1, "per": 4, "queries": 1,
         "prefix": 64, "tail": 9, "pad": 0},
        # one system prompt under a batch of 64 on the 30B-A3B shape, answers of up to 512 tokens
        {"name": "attn system prompt", "op": "attn", "heads": 32, "kv_heads": 4, "dim": 128, "groups": 1, "per": 64,
         "queries": 1, "prefix": 2048, "tail": 512, "pad": 0},
        # eight prompts of odd lengths with up to sixteen samples each on the 8B shape, and padded rows of a captured step
        {"name": "attn samples", "op": "attn", "heads": 32, "kv_heads": 8, "dim": 128, "groups": 8, "per": 16,
         "queries": 1, "prefix": 1501, "tail": 257, "pad": 3},
        # drafted tokens of four prompts' samples verified in one pass: up to five query tokens a sequence
        {"name": "attn drafts", "op": "attn", "heads": 32, "kv_heads": 8, "dim": 128, "groups": 4, "per": 8,
         "queries": 5, "prefix": 4001, "tail": 300, "pad": 0},
        # head dim 256 with two KV heads, as in the hybrid model's attention layers
        {"name": "attn dim 256", "op": "attn", "heads": 16, "kv_heads": 2, "dim": 256, "groups": 2, "per": 8,
         "queries": 1, "prefix": 1030, "tail": 333, "pad": 1},
        # a long document asked about 128 times on the 30B-A3B shape: the largest
        {"name": "attn long document", "op": "attn", "heads": 32, "kv_heads": 4, "dim": 128, "groups": 1, "per": 128,
         "queries": 1, "prefix": 32768, "tail": 1024, "pad": 0},
        # the fork of one prompt into four samples: one partial page in each of 28 layers, copied four times
        {"name": "fork four", "op": "copy", "layers": 28, "kv_heads": 8, "dim": 128, "pages": 64, "sources": 1,
         "copies": 4},
        # 24 prompts into eight samples each, 48 layers
        {"name": "fork batch", "op": "copy", "layers": 48, "kv_heads": 4, "dim": 128, "pages": 512, "sources": 24,
         "copies": 8},
        # a pool of 1500 pages of 36 layers, two thirds live, after requests of many lengths have come and gone
        {"name": "compact pool", "op": "compact", "layers": 36, "kv_heads": 8, "dim": 128, "pages": 1500, "rows": 96,
         "live": 1000, "moves": 333},
        # one sequence, four drafted tokens found by their n-gram: the latency of a single user's step
        {"name": "verify one", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 151936, "bits": 16, "ragged": False,
         "draft_probs": False, "heat": "warm"},
        # a batch with zero to four n-gram drafts each, greedy rows among sampled ones
        {"name": "verify batch", "op": "verify", "seqs": 64, "drafts": 4, "vocab": 151936, "bits": 16, "ragged": True,
         "draft_probs": False, "heat": "mixed"},
        # drafts of a draft model with its probabilities, 32-bit logits, an odd vocabulary
        {"name": "verify draft model", "op": "verify", "seqs": 24, "drafts": 6, "vocab": 151553, "bits": 32,
         "ragged": True, "draft_probs": True, "heat": "warm"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "copy", "compact", "verify", "verify"])
    if op == "attn":
        heads, kv_heads, dim = rng.choice([(16, 8, 128), (32, 4, 128), (32, 8, 128), (16, 4, 128), (16, 2, 256),
                                           (4, 2, 128), (12, 4, 128), (8, 8, 64)])
        seqs = _log(rng, 1, 128)
        groups = _log(rng, 1, min(seqs, 16))
        queries = rng.choice([1, 1, 1, rng.randint(2, 8)])
        case = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "groups": groups,
                "per": max(1, seqs // groups), "queries": queries, "prefix": _log(rng, 1, 32768),
                "tail": _log(rng, 1, 1024), "pad": rng.choice([0, 0, rng.randint(1, 7)])}
        # 32768 prefix tokens under 128 sequences of 32 heads is the most; a prefix of several groups is held once for each
        while (case["prefix"] * case["groups"] * case["per"] * queries * heads * dim > 32768 * 128 * 32 * 128
               or case["prefix"] * case["groups"] * kv_heads * dim > 32768 * 4 * 4 * 128):
            case["prefix"] //= 2
        return case
    if op in ("copy", "compact"):
        layers, kv_heads, dim = rng.choice([(28, 8, 128), (36, 8, 128), (48, 4, 128), (12, 2, 256), (2, 2, 128)])
        if op == "copy":
            sources = _log(rng, 1, 24)
            copies = _log(rng, 1, 8)
            return {"op": op, "layers": layers, "kv_heads": kv_heads, "dim": dim,
                    "pages": sources * (copies + 1) + _log(rng, 1, 200), "sources": sources, "copies": copies}
        pages = _log(rng, 16, 1500)
        live = rng.randint(pages // 4, 3 * pages // 4)
        return {"op": op, "layers": layers, "kv_heads": kv_heads, "dim": dim, "pages": pages,
                "rows": min(live, _log(rng, 1, 128)), "live": live, "moves": rng.randint(0, min(live, pages - live, 333))}
    probs = rng.random() < 0.4
    bits = rng.choice([16, 32])
    return {"op": op, "seqs": _log(rng, 1, 24 if probs or bits == 32 else 64), "drafts": rng.randint(1, 6 if probs else 4),
            "vocab": rng.choice([151936, 151552, 512, _log(rng, 1000, 151936)]), "bits": bits,
            "ragged": rng.random() < 0.7, "draft_probs": probs, "heat": rng.choice(["warm", "mixed"])}


# ------------------------------------------------------------------ sizes that follow from a case alone
def _sizes_of(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _attn_sizes(case):
    """Group sizes, shared lengths of the groups, context lengths and query counts of the sequences (padded rows last)."""
    r = _sizes_of(case)
    sizes, shared, ctx, nq = [], [], [], []
    for g in range(case["groups"]):
        n = case["per"] if case["groups"] == 1 else r.randint((case["per"] + 1) // 2, case["per"])
        p = case["prefix"] if case["groups"] == 1 else r.randint((case["prefix"] + 1) // 2, case["prefix"])
        sizes.append(n)
        shared.append(p)
        for _ in range(n):
            q = r.randint(1, case["queries"])
            nq.append(q)
            ctx.append(p + max(q, r.randint(1, case["tail"])))
    for _ in range(case["pad"]):  # rows of a captured step that hold no sequence: a group and an empty context each
        sizes.append(1)
        shared.append(0)
        ctx.append(0)
        nq.append(1)
    return sizes, shared, ctx, nq


def _compact_sizes(case):
    """Where each row's own pages begin in the list of live pages, the pages that it shares with the first row, and
    the tokens in its last page."""
    r = _sizes_of(case)
    R = case["rows"]
    cuts = [0] + (sorted(r.sample(range(1, case["live"]), R - 1)) if R > 1 else []) + [case["live"]]
    common = [0] + [r.randint(0, min(2, cuts[1])) for _ in range(R - 1)]
    return cuts, common, [r.randint(1, PAGE) for _ in range(R)]


def _verify_sizes(case):
    r = _sizes_of(case)
    n = [r.randint(0, case["drafts"]) if case["ragged"] else case["drafts"] for _ in range(case["seqs"])]
    heat = [r.choice([0.0, 0.7, 1.0, 1.3]) if case["heat"] == "mixed" else r.choice([0.6, 0.8, 1.0])
            for _ in range(case["seqs"])]
    return n, heat


def work(case):
    if case["op"] == "attn":
        sizes, shared, ctx, nq = _attn_sizes(case)
        H, K, D = case["heads"], case["kv_heads"], case["dim"]
        own_tokens = keys = s = 0
        for n, p in zip(sizes, shared):
            p16 = p // PAGE * PAGE
            own_tokens += p16
            for b in range(s, s + n):
                own_tokens += ctx[b] - p16 if ctx[b] else 0
                # query i of a sequence sees its context up to itself
                keys += sum(max(0, ctx[b] - nq[b] + i + 1) for i in range(nq[b]))
            s += n
        return {"bytes": 2 * own_tokens * K * D * 2 + 2 * sum(nq) * H * D * 2, "flops": 4 * keys * H * D}
    if case["op"] == "copy":
        page = 2 * case["layers"] * case["kv_heads"] * PAGE * case["dim"] * 2
        return {"bytes": page * case["sources"] * (1 + case["copies"]), "flops": 0}
    if case["op"] == "compact":
        page = 2 * case["layers"] * case["kv_heads"] * PAGE * case["dim"] * 2
        return {"bytes": 2 * page * case["moves"] + 4 * case["pages"] + 8 * 2 * case["live"], "flops": 0}
    n, _ = _verify_sizes(case)
    rows = sum(n) + len(n)
    # every logit once and one row of random numbers a sequence; a multiply, an exp and an add a logit
    return {"bytes": case["vocab"] * (rows * case["bits"] // 8 + 4 * len(n)), "flops": 3 * rows * case["vocab"]}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _ints(x):
    return torch.tensor(x, dtype=torch.int32).to(DEV)


def prepare(case, seed):
    return {"attn": _prepare_attn, "copy": _prepare_copy, "compact": _prepare_compact,
            "verify": _prepare_verify}[case["op"]](case, seed)


def _normal(g, *shape, scale=1.0):
    return torch.empty(*shape, dtype=torch.bfloat16, device=DEV).normal_(0.0, scale, generator=g)


def _prepare_attn(case, seed):
    g, r = _gen(seed), random.Random(seed)
    sizes, shared, ctx, nq = _attn_sizes(case)
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    need = [-(-c // PAGE) for c in ctx]
    total = sum(s // PAGE for s in shared) + sum(need) + 8
    pool = list(range(total))
    r.shuffle(pool)  # pages lie anywhere in the pool, as they do after some time of serving
    width = max(1, max(need)) + r.randint(0, 3)
    rows, b = [], 0
    for n, p in zip(sizes, shared):
        common = [pool.pop() for _ in range(p // PAGE)]
        for _ in range(n):
            row = common + [pool.pop() for _ in range(need[b] - len(common))] if need[b] else []
            rows.append(row + [0] * (width - len(row)))
            b += 1
    offs, cu = [0], [0]
    for n in sizes:
        offs.append(offs[-1] + n)
    for n in nq:
        cu.append(cu[-1] + n)
    q = _normal(g, cu[-1], H, D, scale=2.0)
    k = _normal(g, total, K, PAGE, D)
    v = _normal(g, total, K, D, PAGE)
    # the plain form's view of the same batch: which query row each group and each sequence holds, padded
    most = max(nq)
    gq = [[t for b in range(offs[i], offs[i + 1]) for t in range(cu[b], cu[b + 1])] for i in range(len(sizes))]
    wide = max(len(x) for x in gq)
    sq = [[cu[b] + min(i, nq[b] - 1) for i in range(most)] for b in range(len(ctx))]
    st = {"op": "attn", "q": q, "k": k, "v": v, "tables": _ints(rows), "ctx": _ints(ctx), "offs": _ints(offs),
          "shared": _ints(shared), "cu": _ints(cu), "scale": 1.0 / math.sqrt(D),
          "group_rows": torch.tensor([x + [0] * (wide - len(x)) for x in gq]).to(DEV),
          "seq_rows": torch.tensor(sq).to(DEV), "group_of": torch.tensor([i for i, n in enumerate(sizes) for _ in range(n)]).to(DEV),
          "place": torch.tensor([j for x in gq for j in range(len(x))]).to(DEV),
          "seq_of": torch.tensor([b for b, n in enumerate(nq) for _ in range(n)]).to(DEV),
          "most_prefix": max(shared) // PAGE, "most_tail": max(max(1, c - s // PAGE * PAGE) for c, s in
                                                               zip(ctx, [p for n, p in zip(sizes, shared) for _ in range(n)]))}
    if own:  # a decode step makes this schedule once from its lengths and uses it in every layer
        from mod_b200.ops import native as N

        st["plan"] = N.attn_shared_plan(st["tables"], st["ctx"], st["offs"], st["shared"], cu[-1], H, K, D,
                                        cu_q=st["cu"])
    return st


def _prepare_copy(case, seed):
    g, r = _gen(seed), random.Random(seed)
    L, K, D, NB = case["layers"], case["kv_heads"], case["dim"], case["pages"]
    ids = list(range(NB))
    r.shuffle(ids)
    src, dst = [], []
    for _ in range(case["sources"]):
        s = ids.pop()
        for _ in range(case["copies"]):
            src.append(s)
            dst.append(ids.pop())
    return {"op": "copy", "k": _normal(g, L, NB, K, PAGE, D), "v": _normal(g, L, NB, K, D, PAGE), "src": _ints(src),
            "dst": _ints(dst)}


def _prepare_compact(case, seed):
    g, r = _gen(seed), random.Random(seed)
    L, K, D, NB, live, moves = (case[x] for x in ("layers", "kv_heads", "dim", "pages", "live", "moves"))
    holes = set(r.sample(range(live), moves))
    pages = [i for i in range(live) if i not in holes] + r.sample(range(live, NB), moves)
    r.shuffle(pages)
    cuts, common, last = _compact_sizes(case)
    rows = [pages[:c] + pages[a:b] for c, a, b in zip(common, cuts, cuts[1:])]
    width = max(len(x) for x in rows) + 1
    lens = [PAGE * (len(x) - 1) + n for x, n in zip(rows, last)]
    return {"op": "compact", "k": _normal(g, L, NB, K, PAGE, D), "v": _normal(g, L, NB, K, D, PAGE),
            "tables": _ints([x + [0] * (width - len(x)) for x in rows]), "lens": _ints(lens)}


def _prepare_verify(case, seed):
    g, r = _gen(seed), random.Random(seed)
    n, heat = _verify_sizes(case)
    B, V, K = case["seqs"], case["vocab"], case["drafts"]
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x + 1)
    T = cu[-1]
    logits = torch.empty(T, V, device=DEV).normal_(0.0, 2.0, generator=g)
    likely = torch.randint(0, V, (T,), device=DEV, generator=g)
    logits[torch.arange(T, device=DEV), likely] = math.log(V) + 3.2  # a token of about three quarters of the probability
    drafts = torch.randint(0, V, (B, K), device=DEV, generator=g)
    at = torch.tensor([[min(cu[b] + j, T - 1) for j in range(K)] for b in range(B)]).to(DEV)
    hit = torch.rand(B, K, device=DEV, generator=g) < 0.85
    drafts = torch.where(hit, likely[at], drafts)
    st = {"op": "verify", "drafts": drafts, "cu": _ints(cu), "uniforms": torch.rand(B, K, device=DEV, generator=g),
          "noise": torch.empty(B, V, device=DEV).exponential_(generator=g).clamp_(min=1e-20),
          "temperature": torch.tensor(heat).to(DEV), "probs": None,
          "rows": torch.tensor([[min(cu[b] + j, cu[b + 1] - 1) for j in range(K + 1)] for b in range(B)]).to(DEV)}
    if case["draft_probs"]:  # the draft model's own distribution: the target's, disturbed
        q = logits[at.reshape(-1)] + torch.empty(B * K, V, device=DEV).normal_(0.0, 0.5, generator=g)
        st["probs"] = torch.softmax(q, -1).view(B, K, V)
    st["logits"] = logits.bfloat16() if case["bits"] == 16 else logits
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attn, "copy": _plain_copy, "compact": _plain_compact, "verify": _plain_verify}[state["op"]](state)


def _run_own(s):
    from mod_b200.ops import native as N

    if s["op"] == "attn":
        return N.attn_shared(s["q"], s["k"], s["v"], s["tables"], s["plan"])
    if s["op"] == "copy":
        N.kv_copy_pages(list(s["k"]), list(s["v"]), s["src"], s["dst"])
        return {"k": s["k"], "v": s["v"]}
    if s["op"] == "compact":
        tables, remap, live = N.kv_compact(list(s["k"]), list(s["v"]), s["tables"], s["lens"])
        return {"tables": tables, "remap": remap, "live": live, "k": s["k"], "v": s["v"]}
    accepted, token, probs = N.verify_sampled(s["logits"], s["cu"], s["drafts"], s["uniforms"], s["noise"],
                                              s["temperature"], draft_probs=s["probs"])
    return {"accepted": accepted, "token": token, "probs": probs}


def _part(q, k, v, seen, scale):
    """Unnormalised attention of q [N, Q, Hkv, G, D] over k, v [N, S, Hkv, D] where seen [N, Q, S]: the weighted sum
    of the values, the sum of the weights and the largest score of each row."""
    x = torch.einsum("nqhgd,nshd->nqhgs", q, k) * scale
    x = torch.where(seen[:, :, None, None, :], x, torch.full_like(x, -math.inf))
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(x - m)
    return torch.einsum("nqhgs,nshd->nqhgd", e, v), e.sum(-1, keepdim=True), m


def _plain_attn(s):
    T, H, D = s["q"].shape
    K = s["k"].shape[1]
    q = s["q"].float().view(T, K, H // K, D)
    first, width = s["offs"][:-1].long(), s["tables"].shape[1]
    lens = s["shared"] // PAGE * PAGE
    # every group's prefix, read once through its first sequence's table
    pages = s["tables"][first.clamp(max=s["tables"].shape[0] - 1), :max(1, s["most_prefix"])].long()
    G, P = pages.shape
    k = s["k"][pages].float().permute(0, 1, 3, 2, 4).reshape(G, P * PAGE, K, D)
    v = s["v"][pages].float().permute(0, 1, 4, 2, 3).reshape(G, P * PAGE, K, D)
    seen = (torch.arange(P * PAGE, device=q.device)[None, :] < lens[:, None])[:, None, :].expand(G, s["group_rows"].shape[1], -1)
    o1, l1, m1 = (x[s["group_of"][s["seq_of"]], s["place"]] for x in _part(q[s["group_rows"]], k, v, seen, s["scale"]))
    # every sequence's own tokens behind the prefix
    start = lens[s["group_of"]].long()
    S = -(-s["most_tail"] // PAGE)
    cols = start[:, None] // PAGE + torch.arange(S, device=q.device)[None, :]
    pages = torch.gather(s["tables"].long(), 1, cols.clamp(max=width - 1))
    B = pages.shape[0]
    k = s["k"][pages].float().permute(0, 1, 3, 2, 4).reshape(B, S * PAGE, K, D)
    v = s["v"][pages].float().permute(0, 1, 4, 2, 3).reshape(B, S * PAGE, K, D)
    rows = s["seq_rows"]
    limit = s["ctx"].long()[:, None] - (s["cu"][1:, None].long() - rows) + 1  # keys that each query token sees
    seen = (start[:, None] + torch.arange(S * PAGE, device=q.device)[None, :])[:, None, :] < limit[:, :, None]
    at = torch.arange(T, device=q.device) - s["cu"][s["seq_of"]]
    o2, l2, m2 = (x[s["seq_of"], at] for x in _part(q[rows], k, v, seen, s["scale"]))
    m = torch.maximum(torch.where(l1 > 0, m1, torch.full_like(m1, -math.inf)), torch.where(l2 > 0, m2, torch.full_like(m2, -math.inf)))
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    w1, w2 = torch.where(l1 > 0, torch.exp(m1 - m), 0.0), torch.where(l2 > 0, torch.exp(m2 - m), 0.0)
    l = l1 * w1 + l2 * w2
    o = torch.where(l > 0, (o1 * w1 + o2 * w2) / l, 0.0)
    return o.reshape(T, H, D).to(s["q"].dtype)


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return {"k": s["k"], "v": s["v"]}


def _plain_compact(s):
    tables, NB = s["tables"], s["k"].shape[1]
    used = torch.arange(tables.shape[1], device=tables.device)[None, :] < ((s["lens"] + PAGE - 1) // PAGE)[:, None]
    mark = torch.zeros(NB, dtype=torch.bool, device=tables.device)
    mark[tables[used].long()] = True
    live = mark.sum()
    ids = torch.arange(NB, device=tables.device)
    src = (mark & (ids >= live)).nonzero().flatten()   # live pages past the end of the compact pool, in order,
    dst = (~mark & (ids < live)).nonzero().flatten()   # take the holes below it, in order
    remap = torch.where(mark, ids, -1)
    remap[src] = dst
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    out = torch.where(used, remap[tables.long()], 0)
    return {"tables": out.int(), "remap": remap.int(), "live": live.int().view(1), "k": s["k"], "v": s["v"]}


def _plain_verify(s):
    B, K = s["drafts"].shape
    x = s["logits"][s["rows"]].float()                                          # [B, K + 1, V]
    V = x.shape[-1]
    n = s["cu"][1:] - s["cu"][:-1] - 1                                           # drafts of each sequence
    heat = s["temperature"][:, None, None]
    top = x.amax(-1, keepdim=True)
    first = x.argmax(-1)
    e = torch.exp((x - top) / torch.where(heat > 0, heat, 1.0))
    greedy = (torch.arange(V, device=x.device)[None, None, :] == first[:, :, None]).float()
    e = torch.where(heat > 0, e, greedy)
    p = e / e.sum(-1, keepdim=True)
    d = s["drafts"]
    pd = torch.gather(p[:, :K], 2, d[:, :, None])[:, :, 0]
    qd = torch.ones_like(pd) if s["probs"] is None else torch.gather(s["probs"], 2, d[:, :, None])[:, :, 0]
    ok = (s["uniforms"] * qd < pd) & (torch.arange(K, device=x.device)[None, :] < n[:, None])
    a = torch.cumprod(ok.int(), 1).sum(1)                                        # drafts accepted before the first refusal
    rows = torch.arange(B, device=x.device)
    pa, at = p[rows, a], a.clamp(max=K - 1)
    if s["probs"] is None:
        q = (torch.arange(V, device=x.device)[None, :] == d[rows, at][:, None]).float()
    else:
        q = s["probs"][rows, at]
    rest = (pa - q).clamp(min=0.0)
    rest = torch.where(((a < n) & (rest.sum(-1) > 0))[:, None], rest, pa)
    token = torch.where(rest > 0, rest / s["noise"], -1.0).argmax(-1)
    place = torch.arange(K + 1, device=x.device)[None, :]
    said = torch.where(place < a[:, None], torch.cat([d, token[:, None]], 1), token[:, None])   # what is emitted
    chance = torch.gather(p, 2, said[:, :, None])[:, :, 0]
    return {"accepted": a.int(), "token": token, "probs": torch.where(place <= a[:, None], chance, 0.0)}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    if case["op"] in ("copy",):
        return None  # pages are moved, not computed
    s = prepare(case, seed)
    if case["op"] == "attn":
        q, out = s["q"].double(), torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        ctx, cu, rep = s["ctx"].tolist(), s["cu"].tolist(), case["heads"] // case["kv_heads"]
        for b, c in enumerate(ctx):
            if not c:
                continue
            pages = s["tables"][b, :-(-c // PAGE)].long()
            k = s["k"][pages].double().transpose(1, 2).flatten(0, 1)[:c].repeat_interleave(rep, 1).permute(1, 2, 0)
            v = s["v"][pages].double().permute(0, 3, 1, 2).flatten(0, 1)[:c].repeat_interleave(rep, 1).transpose(0, 1)
            w = torch.bmm(q[cu[b]:cu[b + 1]].transpose(0, 1), k) * s["scale"]
            for i in range(cu[b + 1] - cu[b]):
                w[:, i, c - (cu[b + 1] - cu[b]) + i + 1:] = -math.inf
            out[cu[b]:cu[b + 1]] = torch.bmm(torch.softmax(w, -1), v).transpose(0, 1)
        return out
    if case["op"] == "compact":
        lens, tables = s["lens"].tolist(), s["tables"].tolist()
        used = [row[:-(-n // PAGE)] for row, n in zip(tables, lens)]
        pages = sorted({p for row in used for p in row})
        kept = {p for p in pages if p < len(pages)}
        to = dict(zip([p for p in pages if p >= len(pages)], [i for i in range(len(pages)) if i not in kept]))
        to.update((p, p) for p in kept)
        return {"tables": _ints([[to[p] for p in row] + [0] * (len(full) - len(row)) for row, full in zip(used, tables)]),
                "remap": _ints([to.get(i, -1) for i in range(case["pages"])]), "live": _ints([len(pages)]), "k": None, "v": None}
    accepted, token = [], []
    probs = torch.zeros(case["seqs"], case["drafts"] + 1, dtype=torch.float64, device=DEV)
    cu, heat = s["cu"].tolist(), s["temperature"].tolist()
    for b in range(case["seqs"]):
        def target(row):
            x = s["logits"][row].double()
            if heat[b] <= 0:
                return torch.zeros_like(x).index_fill_(0, x.argmax(), 1.0)
            return torch.softmax(x / s["temperature"][b].double(), 0)

        a, n = 0, cu[b + 1] - cu[b] - 1
        p = full = target(cu[b])
        while a < n:
            d = s["drafts"][b, a]
            q = torch.zeros_like(p).index_fill_(0, d, 1.0) if s["probs"] is None else s["probs"][b, a].double()
            if not float(s["uniforms"][b, a].double() * q[d]) < float(p[d]):
                rest = (p - q).clamp(min=0.0)
                p = rest if float(rest.sum()) > 0 else p
                break
            probs[b, a] = p[d]
            a += 1
            p = full = target(cu[b] + a)
        accepted.append(a)
        token.append(int((p / s["noise"][b].double()).argmax()))
        probs[b, a] = full[token[-1]]
    return {"accepted": _ints(accepted), "token": torch.tensor(token).to(DEV), "probs": probs}
