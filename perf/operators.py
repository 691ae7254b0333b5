"""Measured operators: one verification step of speculative decoding with a tree of drafted tokens, in its parts.

* ``tables``     positions, cache slots, block table, lengths and ancestor masks of a batch, from its requests' lengths and page lists.
* ``attention``  the drafted nodes' attention over the paged cache: a node sees the committed context, its ancestors and itself.
* ``draw``       one token a row from given uniform numbers, with the row's own temperature, top-k, top-p and min-p.
* ``commit``     the walk along the drafts that the drawn tokens confirm, and the move of their K / V rows behind the context, in every layer.

Lengths, trees and parameters come from the case alone; values from the seed.  Head shapes, layer counts and the vocabulary are those of
``models.config.PRESETS`` (and 64-wide heads as the models described layer by layer have them).
"""
import math
import random
import zlib

import torch

own = False

LOG2E = math.log2(math.e)
VOCAB = 151936


def listed():
    return [
        # a lone chat turn: a short chain of drafts
        dict(name="attention-one", op="attention", batch=1, nodes=5, ctx=1500, heads=32, kv_heads=8, dim=128, page=128, window=0),
        # a loaded server of a dense 8B model, ragged contexts
        dict(name="attention-batch", op="attention", batch=32, nodes=16, ctx=8192, heads=32, kv_heads=8, dim=128, page=128, window=0),
        # wide trees of a mixture model with eight query heads to a KV head
        dict(name="attention-wide", op="attention", batch=64, nodes=63, ctx=2048, heads=32, kv_heads=4, dim=128, page=128, window=0),
        # few long documents
        dict(name="attention-long", op="attention", batch=4, nodes=32, ctx=65536, heads=32, kv_heads=8, dim=128, page=128, window=0),
        # 64-wide heads, small pages, a sliding window, an odd group
        dict(name="attention-window", op="attention", batch=24, nodes=25, ctx=6000, heads=18, kv_heads=6, dim=64, page=16, window=1000),
        # one request's next token
        dict(name="draw-one", op="draw", rows=1, vocab=VOCAB, dtype="f32"),
        # every node of a batch of trees, each request with parameters of its own
        dict(name="draw-tree", op="draw", rows=512, vocab=VOCAB, dtype="f32"),
        # many rows over a smaller vocabulary of odd size, logits in 16 bits
        dict(name="draw-bf16", op="draw", rows=1500, vocab=32003, dtype="bf16"),
        # a decode-sized verify step
        dict(name="tables-step", op="tables", batch=32, nodes=16, ctx=4096, page=128, tree=True),
        # prompts of a loaded server with small pages
        dict(name="tables-large", op="tables", batch=768, nodes=60, ctx=16384, page=16, tree=True),
        # a small batch of a 0.6B model
        dict(name="commit-small", op="commit", batch=4, nodes=16, layers=28, kv_heads=8, dim=128, page=128),
        # wide trees of a loaded 8B server
        dict(name="commit-batch", op="commit", batch=64, nodes=64, layers=36, kv_heads=8, dim=128, page=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """A case of the listed ones' ranges that costs no more than the largest of its kind."""
    op = rng.choice(["attention", "attention", "draw", "tables", "commit"])
    while True:
        if op == "attention":
            kv = rng.choice([1, 2, 4, 6, 8])
            c = dict(op=op, batch=_log(rng, 1, 64), nodes=_log(rng, 1, 128), ctx=_log(rng, 1, 65536), heads=kv * rng.choice([1, 2, 3, 4, 7, 8]), kv_heads=kv,
                     dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), window=rng.choice([0, 0, 0, 100, 1000]))
            w, top = work(c), [work(x) for x in listed() if x["op"] == op]
            if c["batch"] * c["ctx"] > 32 * 8192 or c["batch"] * c["nodes"] * c["heads"] * c["ctx"] > 64 * 63 * 32 * 2048:      # (the plain form's scores)
                continue
            if any(w[k] > max(x[k] for x in top) for k in w):
                continue
            return c
        if op == "draw":
            v = _log(rng, 1000, 200000)
            return dict(op=op, rows=_log(rng, 1, max(1, 512 * VOCAB // v // 2)), vocab=v, dtype=rng.choice(["f32", "bf16"]))
        if op == "tables":
            return dict(op=op, batch=_log(rng, 1, 700), nodes=_log(rng, 1, 60), ctx=_log(rng, 1, 16000), page=rng.choice([16, 32, 64, 128]), tree=rng.random() < 0.7)
        return dict(op=op, batch=_log(rng, 1, 60), nodes=_log(rng, 1, 60), layers=rng.choice([8, 28, 36]), kv_heads=rng.choice([2, 4, 8]), dim=rng.choice([64, 128]),
                    page=rng.choice([16, 64, 128]))


# ------------------------------------------------------------------------------------------ shapes of a case
def _rng(case):
    return random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))


def _lengths(case):
    """Nodes and context of every sequence: the stated ones for the first, from a half (nodes) and a quarter (context) of that for the others."""
    r = _rng(case)
    n = [case["nodes"]] + [r.randint((case["nodes"] + 1) // 2, case["nodes"]) for _ in range(case["batch"] - 1)]
    c = [case["ctx"]] + [r.randint(case["ctx"] // 4, case["ctx"]) for _ in range(case["batch"] - 1)]
    return n, c, r


def _tree(n, r):
    """Parents of a tree in levels of equal width (at least as wide as it is deep); the root is node 0."""
    w = max(1, math.isqrt(max(0, n - 2)) + 1)
    level = lambda i: (i - 1) // w                                   # noqa: E731
    return [-1] + [0 if level(i) == 0 else r.randrange((level(i) - 1) * w + 1, level(i) * w + 1) for i in range(1, n)]


def _masks(parents, words):
    """Ancestors and self of every node as bits of ``words`` 64-bit integers."""
    sets = []
    for i, p in enumerate(parents):
        sets.append((sets[p] if p >= 0 else 0) | 1 << i)
    cut = lambda v: v - (1 << 64) if v >> 63 else v                  # noqa: E731
    return [[cut(s >> 64 * w & (1 << 64) - 1) for w in range(words)] for s in sets]


def _seen(case):
    """(keys that every head's rows look at, keys of the cache they read) summed over the batch."""
    n, c, _ = _lengths(case)
    w = case["window"]
    keys = [min(x, w) if w else x for x in c]
    return sum(a * (k + a / 4) for a, k in zip(n, keys)), sum(a + k for a, k in zip(n, keys))


def work(case):
    op = case["op"]
    if op == "attention":
        pairs, read = _seen(case)
        t = sum(_lengths(case)[0])
        return {"bytes": 4 * read * case["kv_heads"] * case["dim"] + 4 * t * case["heads"] * case["dim"], "flops": 4 * pairs * case["heads"] * case["dim"]}
    if op == "draw":
        return {"bytes": case["rows"] * (case["vocab"] * (4 if case["dtype"] == "f32" else 2) + 28), "flops": 4 * case["rows"] * case["vocab"]}
    n, c, _ = _lengths(dict(case, ctx=case.get("ctx", 100)))
    if op == "tables":
        pages = sum((a + b + case["page"] - 1) // case["page"] for a, b in zip(n, c))
        most = max((a + b + case["page"] - 1) // case["page"] for a, b in zip(n, c))
        return {"bytes": 4 * (5 * len(n) + pages + len(n) * most + sum(n) * (2 + 3 * case["tree"])), "flops": 8 * sum(n)}
    depth = lambda a: -(-(a - 1) // max(1, math.isqrt(max(0, a - 2)) + 1))     # noqa: E731
    moved = sum(depth(a) / 2 for a in n)
    return {"bytes": moved * 2 * case["layers"] * 2 * 2 * case["kv_heads"] * case["dim"] + 16 * sum(n), "flops": 2 * sum(n)}


# ------------------------------------------------------------------------------------------ inputs
def _pages(n, c, page, r):
    """Page lists (pointers and ids, shuffled over a pool that has some more)."""
    need = [(a + b + page - 1) // page for a, b in zip(n, c)]
    ids = list(range(sum(need) + 3))
    r.shuffle(ids)
    ptr = [0]
    for x in need:
        ptr.append(ptr[-1] + x)
    return ptr, ids[:ptr[-1]], len(ids)


def _table(ptr, ids):
    most = max(b - a for a, b in zip(ptr, ptr[1:]))
    return [ids[a:b] + [0] * (most - (b - a)) for a, b in zip(ptr, ptr[1:])]


def prepare(case, seed):
    i32 = dict(dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case=dict(case), op=op)
    if op == "draw":
        b, v = case["rows"], case["vocab"]
        x = torch.randn(b, v, generator=g, device="cuda") * 2.5
        peak = torch.randint(0, v, (b, 24), generator=g, device="cuda")
        x.scatter_add_(1, peak, 14 * torch.rand(b, 24, generator=g, device="cuda"))                 # the likely tokens
        x[torch.rand(b, 1, generator=g, device="cuda").expand(b, v) < 0.1] *= 0.2                    # some rows that hardly tell
        closed = (torch.rand(b, 1, generator=g, device="cuda") < 0.1) & (torch.rand(b, v, generator=g, device="cuda") < 0.9)
        x.masked_fill_(closed, float("-inf"))                                                       # rows under a grammar
        s["logits"] = x.to(torch.float32 if case["dtype"] == "f32" else torch.bfloat16)
        s["uniform"] = torch.rand(b, generator=g, device="cuda")
        r = _rng(case)
        rows = [(r.choice([0.6, 0.8, 1.0, 1.0, 1.3]), r.choice([0, 0, 20, 50, 1000]), r.choice([1.0, 0.8, 0.95, 0.95]), r.choice([0.0, 0.0, 0.05])) for _ in range(b)]
        rows[0] = (0.8, 40, 0.95, 0.0)
        if b > 4:
            rows[1:4] = [(0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0)]                 # greedy; the whole vocabulary; top-p alone
        f32 = dict(dtype=torch.float32, device="cuda")
        s["temperature"], s["top_p"], s["min_p"] = (torch.tensor([x[k] for x in rows], **f32) for k in (0, 2, 3))
        s["top_k"] = torch.tensor([x[1] for x in rows], **i32)
        return s
    n, c, r = _lengths(dict(case, ctx=case.get("ctx", 100)))
    trees = [_tree(a, r) for a in n]
    words = (max(n) + 63) // 64
    page = case["page"]
    if op == "tables":
        r = random.Random(seed)                                                                     # pages of another time: other places
    ptr, ids, pool = _pages(n, c, page, r)
    s.update(page=page, pool=pool, n_tokens=sum(n), max_nodes=max(n), max_pages=max(b - a for a, b in zip(ptr, ptr[1:])))
    if op == "tables":
        s.update(q_lens=torch.tensor(n, **i32), ctx_lens=torch.tensor(c, **i32), page_ptr=torch.tensor(ptr, **i32), pages=torch.tensor(ids, **i32),
                 parents=torch.tensor([p for t in trees for p in t], **i32) if case["tree"] else None)
        return s
    cu = [0]
    for a in n:
        cu.append(cu[-1] + a)
    s.update(cu_q=torch.tensor(cu, **i32), kv_len=torch.tensor([a + b for a, b in zip(n, c)], **i32), block_table=torch.tensor(_table(ptr, ids), **i32),
             mask=torch.tensor([m for t in trees for m in _masks(t, words)], dtype=torch.int64, device="cuda"))
    hkv, d = case["kv_heads"], case["dim"]
    if op == "attention":
        depth = [sum(bin(w & (1 << 64) - 1).count("1") for w in m) - 1 for t in trees for m in _masks(t, words)]
        first = [b for a, b in zip(n, c) for _ in range(a)]
        s["positions"] = torch.tensor([x + y for x, y in zip(depth, first)], **i32)
        s["q"] = (torch.randn(sum(n), case["heads"], d, generator=g, device="cuda") * (LOG2E / math.sqrt(d))).bfloat16()
        s["k_cache"], s["v_cache"] = (torch.empty(pool * page, hkv, d, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(2))
        return s
    # commit: drafted tokens (all different within a sequence), and drawn ones that confirm a path of any length
    s["caches"] = torch.empty(2 * case["layers"], pool * page, hkv, d, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    s["layers"] = list(s["caches"].unbind(0))
    s["parents"] = torch.tensor([p for t in trees for p in t], **i32)
    r = random.Random(seed)
    tokens, sampled = [], []
    for t in trees:
        at, a = r.randrange(VOCAB), len(t)
        mine = [(at + 7919 * i) % VOCAB for i in range(a)]
        drawn = [r.randrange(VOCAB) for _ in range(a)]
        tokens.extend(mine)
        w = max(1, math.isqrt(max(0, a - 2)) + 1)
        want, cur, length = r.randint(0, -(-(a - 1) // w)), 0, 0
        kids = [i for i in range(1, a) if t[i] == 0]
        kids = [i for i in kids if i == 1 or i > want]              # no accepted row lies where another one moves to: a second pass finds the same
        while length < want and kids:
            nxt = r.choice(kids)
            drawn[cur] = mine[nxt]
            cur, length = nxt, length + 1
            kids = [i for i in range(1, a) if t[i] == cur]
        drawn[cur] = (at + 7919 * a) % VOCAB
        sampled.extend(drawn)
    s["tokens"], s["sampled"] = torch.tensor(tokens, **i32), torch.tensor(sampled, **i32)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _calls(s)
    return {"tables": _tables, "attention": _attention, "draw": _draw, "commit": _commit}[s["op"]](s)


def _calls(s):
    op = s["op"]
    if op == "tables":
        from gemm_b200.ops import paging
        t = paging.batch_tables(s["q_lens"], s["ctx_lens"], s["page_ptr"], s["pages"], s["page"], s["n_tokens"], s["max_pages"], s["parents"], s["max_nodes"])
        out = dict(cu_q=t.cu_q, kv_len=t.kv_len, positions=t.positions, slots=t.slots, block_table=t.block_table)
        return dict(out, mask=t.mask) if s["parents"] is not None else out
    if op == "draw":
        from gemm_b200.ops import sampling
        token, logprob = sampling.draw(s["logits"], s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], want_logprob=True)
        return dict(token=token, logprob=logprob)
    from gemm_b200.ops import tree
    if op == "attention":
        return dict(out=tree.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["cu_q"], s["kv_len"], s["block_table"], s["page"], s["mask"], s["max_nodes"],
                                            window=s["case"]["window"], positions=s["positions"]))
    a = tree.tree_commit(s["layers"], s["tokens"], s["parents"], s["sampled"], s["cu_q"], s["kv_len"], s["block_table"], s["page"], s["max_nodes"])
    return dict(count=a.count, path=a.path, next_token=a.next_token, kv_len=a.kv_len, caches=s["caches"])


def _spread(cu, t):
    """Sequence of every token, and its place there."""
    at = torch.arange(t, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), at, right=True)
    return seq, at - cu.long()[seq]


def _tables(s):
    n, c, ps, t = s["q_lens"].long(), s["ctx_lens"].long(), s["page"], s["n_tokens"]
    ptr, pages = s["page_ptr"].long(), s["pages"]
    cu = torch.cat([n.new_zeros(1), n.cumsum(0)])
    seq, at = _spread(cu, t)
    place = c[seq] + at
    slots = pages[ptr[seq] + place // ps].long() * ps + place % ps
    col = torch.arange(s["max_pages"], device=n.device)
    have = ptr[1:] - ptr[:-1]
    at_page = (ptr[:-1, None] + col).clamp_max(max(0, pages.numel() - 1))
    table = torch.where(col < have[:, None], pages[at_page], 0)
    out = dict(cu_q=cu.int(), kv_len=(c + n).int(), positions=place.int(), slots=slots.int(), block_table=table)
    if s["parents"] is None:
        return out
    # ancestors: the closure of "parent of", by squaring
    b, m = n.numel(), s["max_nodes"]
    reach = torch.zeros(b, m, m, device=n.device)
    reach[seq, at, at] = 1
    p = s["parents"].long()
    reach[seq[p >= 0], at[p >= 0], p[p >= 0]] = 1
    for _ in range(max(1, m - 1).bit_length()):
        reach = (torch.bmm(reach, reach) > 0).float()
    anc = reach[seq, at] > 0                                         # [T, nodes]
    words = (m + 63) // 64
    anc = torch.nn.functional.pad(anc, (0, words * 64 - m)).view(t, words, 64)
    out["mask"] = (anc.long() << torch.arange(64, device=n.device)).sum(-1)
    out["positions"] = (c[seq] + anc.sum((1, 2)) - 1).int()
    return out


def _attention(s):
    q, cu, kv_len, mask = s["q"].float(), s["cu_q"].long(), s["kv_len"].long(), s["mask"]
    t, hq, d = q.shape
    hkv, b, m = s["k_cache"].shape[1], kv_len.numel(), s["max_nodes"]
    n = cu[1:] - cu[:-1]
    most = s["block_table"].shape[1] * s["page"]
    key = torch.arange(most, device=q.device)
    slot = s["block_table"].long()[:, key // s["page"]] * s["page"] + key % s["page"]
    k, v = s["k_cache"][slot].float(), s["v_cache"][slot].float()    # [B, keys, Hkv, D]
    row = torch.arange(m, device=q.device)
    live = row < n[:, None]
    at = torch.where(live, cu[:-1, None] + row, 0)
    off = key - (kv_len - n)[:, None]                                # place in the tree; negative: context
    bits = mask[at].gather(2, (off >> 6).clamp(0, mask.shape[1] - 1)[:, None].expand(b, m, most)) >> (off & 63)[:, None]
    see = (off < 0)[:, None] | (bits & 1).bool()
    see &= (key < kv_len[:, None])[:, None] & live[:, :, None]
    if s["case"]["window"]:
        see &= (off >= 0)[:, None] | (key > s["positions"].long()[at][:, :, None] - s["case"]["window"])
    sc = torch.einsum("bnhgd,bkhd->bhgnk", q[at].view(b, m, hkv, hq // hkv, d), k)
    sc.masked_fill_(~see[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp2(sc - top)
    o = torch.einsum("bhgnk,bkhd->bnhgd", p, v) / p.sum(-1).clamp_min(1e-30).permute(0, 3, 1, 2)[..., None]
    return dict(out=o.reshape(b, m, hq, d)[live].bfloat16())


def _draw(s):
    x = s["logits"].float()
    x = torch.where(x.isnan(), float("-inf"), x)
    val, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    t, k = s["temperature"].double()[:, None], s["top_k"].long()[:, None]
    rank = torch.arange(x.shape[1], device=x.device)
    k = torch.where(t <= 0, 1, torch.where(k > 0, k, x.shape[1]))
    val = val.double()
    w = torch.exp((val - val[:, :1]) / torch.where(t <= 0, 1.0, t)) * (rank < k)
    cum = w.cumsum(-1)
    front = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], 1)
    top_p = s["top_p"].double()[:, None]
    keep = ((front < top_p * cum[:, -1:]) | (top_p >= 1)) & (w >= s["min_p"].double()[:, None]) & (rank < k)
    w = torch.zeros_like(w).scatter_(1, ids, w * keep)
    cdf = w.cumsum(-1)
    pick = (cdf <= s["uniform"].double()[:, None] * cdf[:, -1:]).sum(-1, keepdim=True)
    return dict(token=pick[:, 0].int(), logprob=(w.gather(1, pick) / cdf[:, -1:]).log()[:, 0].float())


def _commit(s):
    cu, tokens, parents, sampled, mask = s["cu_q"].long(), s["tokens"], s["parents"].long(), s["sampled"], s["mask"]
    t, b, m, ps = tokens.numel(), cu.numel() - 1, s["max_nodes"], s["page"]
    seq, at = _spread(cu, t)
    up = cu[seq] + parents.clamp_min(0)
    fits = (parents < 0) | (tokens == sampled[up])                   # (the tokens of a sequence's nodes differ)
    word = at >> 6
    have = torch.zeros(b, mask.shape[1], dtype=torch.int64, device=cu.device)
    have.index_put_((seq, word), fits.long() << (at & 63), accumulate=True)
    taken = ((mask & ~have[seq]) == 0).all(1)                        # the node and all its ancestors fit
    count = torch.zeros(b, dtype=torch.int64, device=cu.device).index_add_(0, seq, taken.long())
    which, order = seq[taken], torch.cumsum(taken.long(), 0)[taken] - 1
    order = order - torch.cat([count.new_zeros(1), count.cumsum(0)[:-1]])[which]
    path = torch.full((b, m), -1, dtype=torch.int64, device=cu.device)
    path[which, order] = at[taken]
    last = path.gather(1, (count - 1)[:, None])[:, 0]
    ctx = s["kv_len"].long() - (cu[1:] - cu[:-1])
    slot = lambda sq, p: s["block_table"].long()[sq, p // ps] * ps + p % ps      # noqa: E731
    src, dst = slot(which, ctx[which] + at[taken]), slot(which, ctx[which] + order)
    s["caches"][:, dst] = s["caches"][:, src]
    return dict(count=count.int(), path=path.int(), next_token=sampled[cu[:-1] + last], kv_len=(ctx + count).int(), caches=s["caches"])


# ------------------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "attention":
        return _exact_attention(s)
    if op == "draw":
        return _exact_draw(s)
    if op == "tables":
        n, c, ptr, ids, ps = (s[k].tolist() if k != "page" else s[k] for k in ("q_lens", "ctx_lens", "page_ptr", "pages", "page"))
        cu, pos, slots, masks = [0], [], [], []
        words = (s["max_nodes"] + 63) // 64
        par = s["parents"].tolist() if case["tree"] else None
        for i, (a, b) in enumerate(zip(n, c)):
            place = [b + j for j in range(a)]
            slots += [ids[ptr[i] + p // ps] * ps + p % ps for p in place]
            if par is not None:
                mine = _masks(par[cu[-1]:cu[-1] + a], words)
                masks += mine
                place = [b + sum(bin(w & (1 << 64) - 1).count("1") for w in x) - 1 for x in mine]
            pos += place
            cu.append(cu[-1] + a)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32)              # noqa: E731
        out = dict(cu_q=i32(cu), kv_len=i32([a + b for a, b in zip(n, c)]), positions=i32(pos), slots=i32(slots), block_table=i32(_table(ptr, ids)))
        return dict(out, mask=torch.tensor(masks, dtype=torch.int64)) if par is not None else out
    cu, tok, par, smp, kvl, bt = (s[k].tolist() for k in ("cu_q", "tokens", "parents", "sampled", "kv_len", "block_table"))
    ps, caches = s["page"], s["caches"].clone()
    counts, paths, nxt, lens = [], [], [], []
    for i in range(len(cu) - 1):
        o, a = cu[i], cu[i + 1] - cu[i]
        path = [0]
        while True:
            kids = [j for j in range(1, a) if par[o + j] == path[-1] and tok[o + j] == smp[o + path[-1]]]
            if not kids:
                break
            path.append(kids[0])
        ctx = kvl[i] - a
        at = lambda p: bt[i][p // ps] * ps + p % ps                     # noqa: E731,B023
        for j, node in enumerate(path):
            caches[:, at(ctx + j)] = s["caches"][:, at(ctx + node)]
        counts.append(len(path)), nxt.append(smp[o + path[-1]]), lens.append(ctx + len(path))
        paths.append(path + [-1] * (s["max_nodes"] - len(path)))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)                  # noqa: E731
    return dict(count=i32(counts), path=i32(paths), next_token=i32(nxt), kv_len=i32(lens), caches=caches)


def _exact_attention(s):
    q, cu, kvl = s["q"].double(), s["cu_q"].tolist(), s["kv_len"].tolist()
    hq, hkv, win = q.shape[1], s["k_cache"].shape[1], s["case"]["window"]
    out = torch.zeros_like(q)
    for i, length in enumerate(kvl):
        a, z = cu[i], cu[i + 1]
        ctx = length - (z - a)
        places = torch.arange(length, device=q.device)
        slot = s["block_table"][i].long()[places // s["page"]] * s["page"] + places % s["page"]
        see = torch.ones(z - a, length, dtype=torch.bool, device=q.device)
        if win:
            see[:, :ctx] = s["positions"][a:z, None] - places[None, :ctx] < win
        for j in range(z - a):
            see[:, ctx + j] = (s["mask"][a:z, j // 64] >> (j % 64)) % 2 == 1
        for h in range(hkv):
            k, v = s["k_cache"][slot, h].double(), s["v_cache"][slot, h].double()
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                e = (q[a:z, g] @ k.t() * math.log(2.0)).masked_fill(~see, float("-inf"))
                out[a:z, g] = torch.softmax(e, -1) @ v
    return dict(out=out)


def _exact_draw(s):
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    if x.size > 80_000_000:
        return None
    u, temp, tk, tp, mp = (s[k].double().cpu().numpy() for k in ("uniform", "temperature", "top_k", "top_p", "min_p"))
    token, logprob = [], []
    for i, row in enumerate(x):
        order = np.argsort(-row, kind="stable")
        if temp[i] <= 0:
            token.append(int(order[0])), logprob.append(0.0)
            continue
        order = order[: int(tk[i])] if tk[i] > 0 else order
        w = np.exp((row[order] - row[order[0]]) / temp[i])
        n = len(w)
        if tp[i] < 1:
            n = int(np.searchsorted(np.cumsum(w), tp[i] * w.sum())) + 1
        n = max(1, min(n, int(np.sum(w >= mp[i]))))
        keep = np.sort(order[:n])
        w = np.exp((row[keep] - row[order[0]]) / temp[i])
        cdf = np.cumsum(w)
        j = int(np.searchsorted(cdf, u[i] * cdf[-1], side="right"))
        token.append(int(keep[j])), logprob.append(math.log(w[j] / cdf[-1]))
    return dict(token=torch.tensor(token, dtype=torch.int32), logprob=torch.tensor(logprob, dtype=torch.float64))
