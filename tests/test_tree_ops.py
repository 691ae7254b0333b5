"""Operators of tree-speculative decoding: batch tables, attention of tree nodes, draws with per-row parameters, acceptance and cache move.  The plain forms are
checked on the CPU against independent statements of the definitions; the kernels against the plain forms in 64 bits."""
import math
import random

import pytest
import torch

from gemm_b200 import _native
from gemm_b200.ops import paging, sampling, tree

gpu = pytest.mark.gpu
LOG2E = math.log2(math.e)


def random_tree(n, r, wide=False):
    return [-1] + [0 if wide else r.randrange(i) for i in range(1, n)]


def masks_of(parents, words):
    sets = []
    for i, p in enumerate(parents):
        sets.append((sets[p] if p >= 0 else set()) | {i})
    out = torch.zeros(len(parents), words, dtype=torch.int64)
    for i, s in enumerate(sets):
        for j in s:
            out[i, j // 64] |= (1 << (j % 64)) - ((1 << 64) if j % 64 == 63 else 0)
    return out, [len(s) - 1 for s in sets]


def paged(nodes, ctx, page, r, spare=2):
    need = [(a + b + page - 1) // page for a, b in zip(nodes, ctx)]
    ids = list(range(sum(need) + spare))
    r.shuffle(ids)
    ptr = [0]
    for x in need:
        ptr.append(ptr[-1] + x)
    table = torch.zeros(len(nodes), max(need + [1]), dtype=torch.int32)
    for s in range(len(nodes)):
        table[s, :need[s]] = torch.tensor(ids[ptr[s]:ptr[s + 1]], dtype=torch.int32)
    return ptr, ids, table, len(ids)


# ------------------------------------------------------------------------------------------ tables
TABLES = [([1], [0], 16, None), ([1, 1, 1], [5, 16, 31], 16, None), ([0, 7, 0, 33, 0], [3, 0, 0, 95, 0], 32, None), ([200, 1, 513], [0, 4000, 129], 128, None),
          ([5, 0, 64, 1], [10, 3, 127, 0], 16, "tree"), ([129, 256, 65], [0, 1000, 31], 64, "tree"), ([0, 0], [4, 5], 16, None), ([], [], 16, None),
          ([3] * 1500, [17] * 1500, 8, "tree")]


def table_inputs(q, ctx, page, kind, pad=0):
    r = random.Random(len(q) * 1000 + sum(q))
    ptr, ids, table, _ = paged(q, ctx, page, r)
    par = [p for n in q for p in (random_tree(n, r) if n else [])] + [-1] * pad if kind else None
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)                     # noqa: E731
    return (i32(q), i32(ctx), i32(ptr), i32(ids), page, sum(q) + pad, table.shape[1], i32(par) if par is not None else None, max(q, default=0) if kind else 0), table


@pytest.mark.parametrize("q,ctx,page,kind", TABLES)
def test_tables_plain(q, ctx, page, kind):
    args, table = table_inputs(q, ctx, page, kind, pad=3)
    got = paging.batch_tables(*args)
    at = 0
    for s, (n, c) in enumerate(zip(q, ctx)):
        assert got.cu_q[s] == at and got.kv_len[s] == n + c
        par = args[7][at:at + n].tolist() if kind else None
        for i in range(n):
            assert got.slots[at + i] == int(table[s, (c + i) // page]) * page + (c + i) % page
            chain = [i]
            while par is not None and par[chain[-1]] >= 0:
                chain.append(par[chain[-1]])
            assert got.positions[at + i] == c + (len(chain) - 1 if kind else i)
            if kind:
                assert [j for j in range(got.mask.shape[1] * 64) if got.mask[at + i, j // 64] >> (j % 64) & 1] == sorted(chain)
        at += n
    assert got.cu_q[len(q)] == at and got.block_table.shape == (len(q), args[6])
    if len(q):
        assert torch.equal(got.block_table, table[:, :args[6]])
    assert got.slots[at:].tolist() == [-1] * 3 and got.positions[at:].tolist() == [0] * 3


@gpu
@pytest.mark.parametrize("pad", [0, 700])
@pytest.mark.parametrize("q,ctx,page,kind", TABLES)
def test_tables_kernel(q, ctx, page, kind, pad):
    args, _ = table_inputs(q, ctx, page, kind, pad)
    want = paging.batch_tables(*args)
    got = paging.batch_tables(*[a.cuda() if torch.is_tensor(a) else a for a in args])
    for name, a, b in zip(want._fields, got, want):
        assert (a is None) == (b is None) and (a is None or torch.equal(a.cpu(), b)), name


@gpu
def test_tables_kernel_odd_inputs():
    """Negative lengths, more tokens than rows, pages that are missing, parents that are none: defined answers, the plain form's."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)                     # noqa: E731
    args = (i32([4, -3, 6, 9]), i32([14, 2, 0, 1]), i32([0, 1, 2, 2, 4]), i32([7, 3, 5, 1]), 16, 15, 3, i32([-1, 5, 0, 2] + [-1, 0, 1, 3, 2, 9] + [-1, -5, 1, 0, 3]), 9)
    want = paging.batch_tables(*args)
    got = paging.batch_tables(*[a.cuda() if torch.is_tensor(a) else a for a in args])
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    assert want.slots[2:4].tolist() == [-1, -1] and want.slots[4:10].tolist() == [-1] * 6 and want.cu_q.tolist() == [0, 4, 4, 10, 15]


def test_tables_refusals():
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)                     # noqa: E731
    ok = dict(q_lens=i32([2]), ctx_lens=i32([3]), page_ptr=i32([0, 1]), pages=i32([0]), page_size=8, total_tokens=2, max_pages=1)
    paging.batch_tables(**ok)
    for bad in (dict(q_lens=torch.tensor([2])), dict(ctx_lens=i32([3, 4])), dict(page_ptr=i32([0])), dict(page_size=0), dict(total_tokens=-1), dict(max_pages=-1),
                dict(parents=i32([-1])), dict(parents=i32([-1, 0]), max_nodes=0), dict(parents=i32([-1, 0]), max_nodes=257), dict(pages=i32([[0, 1], [2, 3]])[:, 0])):
        with pytest.raises(ValueError):
            paging.batch_tables(**{**ok, **bad})


# ------------------------------------------------------------------------------------------ attention
def attention_inputs(nodes, ctx, hq, hkv, dk, dv, page, dtype=torch.bfloat16, seed=0, full_mask=False):
    r = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    ptr, ids, table, pool = paged(nodes, ctx, page, r)
    words = paging.mask_words(max(nodes + [1]))
    masks, depth = [torch.zeros(0, words, dtype=torch.int64)], []
    for n in nodes:
        m, d = masks_of(random_tree(n, r), words) if n else (torch.zeros(0, words, dtype=torch.int64), [])
        masks.append(m)
        depth.append(d)
    cu = torch.tensor([0] + list(torch.tensor(nodes).cumsum(0)), dtype=torch.int32)
    pos = torch.tensor([c + x for c, d in zip(ctx, depth) for x in d], dtype=torch.int32)
    t = sum(nodes)
    # a cache whose unused places hold what must not count
    k, v = (torch.full((pool * page, hkv, d), float("nan")) for d in (dk, dv))
    for s, (n, c) in enumerate(zip(nodes, ctx)):
        place = torch.arange(n + c)
        slot = table[s].long()[place // page] * page + place % page
        k[slot], v[slot] = torch.randn(n + c, hkv, dk, generator=g), torch.randn(n + c, hkv, dv, generator=g)
    q = torch.randn(t, hq, dk, generator=g) * (LOG2E / math.sqrt(dk))
    return dict(q=q.to(dtype), k_cache=k.to(dtype), v_cache=v.to(dtype), cu_q=cu, kv_len=torch.tensor([a + b for a, b in zip(nodes, ctx)], dtype=torch.int32),
                block_table=table, page_size=page, mask=torch.cat(masks), max_nodes=max(nodes + [1]), positions=pos)


def wide(s):
    return {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}


def on_gpu(s):
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in s.items()}


# The weights are rounded to bf16 for the second product (at most 2^-8 of each, independent: far less of their sum), the output to bf16 (2^-8 of each).  The
# scores' error is that of sums of products of bf16 in f32: below 1e-5.  Together, relative to the largest value a row's output is made of: 2 * 2^-8 and a little.
def close(got, s, out_of=None):
    want = tree.tree_attention_ref(**{k: v for k, v in wide(s).items() if k not in ("max_nodes", "out")})
    got = got.double().cpu()
    if s["q"].dtype == torch.float32:
        # sums of a few thousand f32 products, weights that add up to one
        assert torch.allclose(got, want, rtol=0, atol=2e-5), float((got - want).abs().max())
        return
    big = torch.nan_to_num(s["v_cache"].double()).abs().max()
    err = (got - want).abs()
    assert bool((err <= 2 ** -8 * want.abs() + 2 ** -8 * big).all()), float(err.max())
    rel = float((got - want).norm() / want.norm().clamp_min(1e-30))
    assert rel < 2 ** -7, rel


def test_attention_plain_is_the_definition():
    s = attention_inputs([3, 0, 6], [5, 2, 0], 4, 2, 8, 6, 4, torch.float32)
    s["window"] = 4
    got = tree.tree_attention(**s)
    for seq in range(3):
        for i in range(int(s["cu_q"][seq]), int(s["cu_q"][seq + 1])):
            ctx = int(s["kv_len"][seq]) - int(s["cu_q"][seq + 1] - s["cu_q"][seq])
            seen = [j for j in range(ctx) if int(s["positions"][i]) - j < 4]
            seen += [ctx + j for j in range(64) if int(s["mask"][i, 0]) >> j & 1]
            for h in range(4):
                slot = [int(s["block_table"][seq, j // 4]) * 4 + j % 4 for j in seen]
                w = [math.exp(float(s["q"][i, h].double() @ s["k_cache"][x, h // 2].double()) / LOG2E) for x in slot]
                want = sum(a * s["v_cache"][x, h // 2].double() for a, x in zip(w, slot)) / sum(w)
                assert torch.allclose(got[i, h].double(), want, atol=1e-5)


def test_attention_plain_masked_values():
    """A value that is not finite reaches the rows that see it, and no others; a row that sees nothing is zero."""
    s = attention_inputs([3], [2], 2, 1, 4, 4, 4, torch.float32)
    s["mask"] = torch.tensor([[0b001], [0b010], [0b100]])
    place = lambda j: int(s["block_table"][0, j // 4]) * 4 + j % 4         # noqa: E731
    s["v_cache"][place(3)] = float("inf")
    got = tree.tree_attention(**s)
    assert torch.isfinite(got[0]).all() and torch.isinf(got[1]).all() and torch.isfinite(got[2]).all()
    s = attention_inputs([2], [0], 2, 1, 4, 4, 4, torch.float32)
    s["mask"] = torch.tensor([[0], [0b10]])
    got = tree.tree_attention(**s)
    assert (got[0] == 0).all() and (got[1] != 0).all()


def test_attention_refusals():
    s = attention_inputs([3, 2], [5, 2], 4, 2, 8, 8, 4, torch.float32)
    tree.tree_attention(**s)
    bad = [dict(q=s["q"].transpose(0, 1).contiguous().transpose(0, 1)), dict(q=s["q"].half()), dict(q=s["q"].bfloat16()), dict(k_cache=s["k_cache"][:, :1]),
           dict(v_cache=s["v_cache"].transpose(1, 2)), dict(cu_q=s["cu_q"].long()), dict(cu_q=s["cu_q"][:2]), dict(block_table=s["block_table"][:1]), dict(page_size=0),
           dict(mask=s["mask"].int()), dict(mask=s["mask"][:3]), dict(max_nodes=0), dict(max_nodes=300), dict(max_nodes=65), dict(window=-1), dict(window=3, positions=None),
           dict(positions=s["positions"][:2]), dict(out=torch.empty(5, 4, 7)), dict(q=torch.zeros(5, 3, 8))]
    for b in bad:
        with pytest.raises(ValueError):
            tree.tree_attention(**{**s, **b})


ATTENTION = [
    # nodes, ctx, hq, hkv, dk, dv, page, window
    ([1], [0], 4, 4, 128, 128, 128, 0),
    ([1, 1], [700, 1], 8, 1, 128, 128, 16, 0),
    ([5], [1500], 32, 8, 128, 128, 128, 0),
    ([3, 0, 17, 8], [127, 50, 128, 0], 8, 2, 128, 128, 64, 0),
    ([16, 9], [1000, 4097], 16, 4, 128, 128, 32, 0),
    ([64, 33], [63, 300], 8, 2, 128, 128, 16, 0),
    ([40, 63, 2], [2000, 129, 5000], 32, 4, 128, 128, 128, 0),
    ([130, 256], [500, 77], 4, 1, 128, 128, 8, 0),
    ([25, 13], [900, 6000], 18, 6, 64, 64, 16, 1000),
    ([12, 7], [400, 130], 6, 6, 64, 128, 32, 100),
    ([30], [513], 14, 2, 128, 64, 64, 1),
    ([20, 4], [100, 200], 28, 4, 64, 64, 8, 130),
    ([9], [50], 96, 1, 128, 128, 16, 0),
    ([6, 3], [40, 9], 6, 3, 80, 72, 16, 0),
    ([4], [33], 2, 1, 192, 256, 128, 20),
    ([7, 2], [100, 3], 5, 5, 33, 17, 48, 0),
    ([2], [20], 130, 1, 64, 64, 16, 0),
]


@gpu
@pytest.mark.parametrize("nodes,ctx,hq,hkv,dk,dv,page,window", ATTENTION)
def test_attention_kernel(nodes, ctx, hq, hkv, dk, dv, page, window):
    s = attention_inputs(nodes, ctx, hq, hkv, dk, dv, page, seed=sum(ctx))
    s["window"] = window
    got = tree.tree_attention(**on_gpu(s))
    _native.assert_status_ok()
    close(got, s)


@gpu
@pytest.mark.parametrize("nodes,ctx,hq,hkv,dk,dv,page,window", [ATTENTION[0], ATTENTION[3], ATTENTION[8], ATTENTION[15]])
def test_attention_kernel_f32(nodes, ctx, hq, hkv, dk, dv, page, window):
    s = attention_inputs(nodes, ctx, hq, hkv, dk, dv, page, torch.float32)
    s["window"] = window
    close(tree.tree_attention(**on_gpu(s)), s)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nodes,ctx,hq,hkv,dk,dv,page,window", [
    ([7, 2], [100, 3], 6, 2, 320, 300, 16, 0), ([5, 0, 9, 1, 2, 1, 1], [70, 3, 0, 500, 31, 32, 33], 9, 3, 40, 256, 8, 0), ([1] * 40, list(range(40)), 3, 3, 256, 80, 12, 9),
    ([256, 3], [10, 700], 5, 1, 16, 24, 32, 300)])
def test_attention_kernel_other_heads(nodes, ctx, hq, hkv, dk, dv, page, window, dtype):
    """Tiles of rows that span sequences and tokens, heads wider than a tile's, pages of any size."""
    s = attention_inputs(nodes, ctx, hq, hkv, dk, dv, page, dtype, seed=dk)
    s["window"] = window
    close(tree.tree_attention(**on_gpu(s)), s)


@gpu
@pytest.mark.parametrize("hq,hkv,n,d", [(4, 2, 3, 128), (16, 2, 70, 128), (8, 8, 12, 64), (2, 1, 5, 96)])
def test_attention_kernel_masked_places(hq, hkv, n, d):
    """Arbitrary masks, empty rows among them; keys and values that are not finite at nodes that some rows do not see; the lowest value of the type."""
    s = attention_inputs([n, n], [0, 130], hq, hkv, d, d, 16, seed=n)
    g = torch.Generator().manual_seed(1)
    words = s["mask"].shape[1]
    s["mask"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (2 * n, words), generator=g)
    s["mask"][0] = 0                                                        # sees nothing: its sequence has no context
    s["mask"][n] = 0                                                        # sees the context alone
    for word in range(words):
        s["mask"][:, word] &= ~(1 << 1) if word == 0 else -1                # node 1 is seen by nobody
    for seq in range(2):
        j = [0, 130][seq] + 1
        slot = int(s["block_table"][seq, j // 16]) * 16 + j % 16
        s["v_cache"][slot] = float("inf") if seq else float("nan")
        s["k_cache"][slot] = float("nan") if seq else torch.finfo(torch.bfloat16).min
    got = tree.tree_attention(**on_gpu(s))
    assert (got[0] == 0).all() and torch.isfinite(got).all()
    close(got, s)
    # node 2 of the second sequence has an infinite feature that only some rows see
    slot = int(s["block_table"][1, 132 // 16]) * 16 + 132 % 16
    s["v_cache"][slot, :, 3] = float("inf")
    got = tree.tree_attention(**on_gpu(s)).cpu()
    sees = (s["mask"][n:, 0] >> 2 & 1).bool()
    assert torch.equal(torch.isinf(got[n:, :, 3]).all(1), sees) and torch.isfinite(got[n:][~sees]).all()
    assert torch.isfinite(got[n:, :, 4:]).all()


def window_inputs(hq, hkv, n, d, window, ctx):
    """Keys and values that are not finite in front of every row's window, and one infinite feature at a place that only the root of each tree sees."""
    s = attention_inputs([n, 1, n], [ctx, ctx, ctx + 61], hq, hkv, d, d, 16, seed=n)
    s["window"] = window
    odd = s["v_cache"].clone()
    for seq, c in enumerate((ctx, ctx, ctx + 61)):
        place = torch.arange(max(0, c - window + 1))
        slot = s["block_table"][seq].long()[place // 16] * 16 + place % 16
        for cache in (s["k_cache"], s["v_cache"], odd):
            cache[slot] = float("nan")
        j = c - window + 1
        odd[int(s["block_table"][seq, j // 16]) * 16 + j % 16, :, 3] = float("inf")
    depth0 = torch.zeros(2 * n + 1, dtype=torch.bool)
    depth0[[0, n, n + 1]] = True
    return s, odd, depth0


WINDOWS = [(4, 2, 3, 128, 50, 300), (16, 2, 70, 128, 130, 700), (8, 8, 12, 64, 100, 260), (32, 8, 20, 128, 257, 3000), (4, 1, 30, 64, 7, 130), (2, 1, 5, 96, 40, 130)]


def check_window(run, hq, hkv, n, d, window, ctx):
    s, odd, depth0 = window_inputs(hq, hkv, n, d, window, ctx)
    got = run(s).cpu()
    assert torch.isfinite(got).all()
    close(got, s)
    got = run({**s, "v_cache": odd}).cpu()
    # What sees the infinite value is not finite: infinite, or NaN, since a row may be held as several sums over its places, and in those that leave the place out it
    # is multiplied by a weight of zero (0 * inf = NaN) where all of the sequence's rows see it.
    assert not torch.isfinite(got[depth0][:, :, 3]).any() and torch.isfinite(got[~depth0]).all() and torch.isfinite(got[:, :, 4:]).all()


@pytest.mark.parametrize("hq,hkv,n,d,window,ctx", WINDOWS)
def test_attention_plain_window(hq, hkv, n, d, window, ctx):
    check_window(lambda s: tree.tree_attention(**s), hq, hkv, n, d, window, ctx)


@gpu
@pytest.mark.parametrize("hq,hkv,n,d,window,ctx", WINDOWS)
def test_attention_kernel_window(hq, hkv, n, d, window, ctx):
    check_window(lambda s: tree.tree_attention(**on_gpu(s)), hq, hkv, n, d, window, ctx)


def deep_inputs(n, hq, hkv, dk, dv, page, window, dtype=torch.bfloat16):
    """Trees deeper than the window: a chain, a tree whose branches reach past the window at several depths, and a wide one that does not."""
    s = attention_inputs([n, n, n], [0, 200, 3], hq, hkv, dk, dv, page, dtype, seed=n + window)
    r = random.Random(n)
    masks, pos = [], []
    for ctx, par in ((0, list(range(-1, n - 1))), (200, [-1] + [max(0, i - r.randint(1, 3)) for i in range(1, n)]), (3, random_tree(n, r, wide=True))):
        m, d = masks_of(par, s["mask"].shape[1])
        masks.append(m)
        pos += [ctx + x for x in d]
    s.update(mask=torch.cat(masks), positions=torch.tensor(pos, dtype=torch.int32), window=window)
    return s


def by_definition(s):
    """A node sees the places of the context and the nodes of its mask that are less than ``window`` in front of it, one after the other, in 64 bits."""
    q, k, v = (s[x].double() for x in ("q", "k_cache", "v_cache"))
    g, page, out = q.shape[1] // k.shape[1], s["page_size"], torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64)
    for seq in range(s["kv_len"].numel()):
        a, z = int(s["cu_q"][seq]), int(s["cu_q"][seq + 1])
        ctx, pos = int(s["kv_len"][seq]) - (z - a), s["positions"].tolist()
        for i in range(a, z):
            seen = [j for j in range(ctx) if pos[i] - j < s["window"]]
            seen += [ctx + j for j in range(z - a) if int(s["mask"][i, j // 64]) >> (j % 64) & 1 and pos[i] - pos[a + j] < s["window"]]
            slot = torch.tensor([int(s["block_table"][seq, j // page]) * page + j % page for j in seen], dtype=torch.long)
            for h in range(q.shape[1]):
                w = torch.softmax(k[slot, h // g] @ q[i, h] * math.log(2.0), 0)
                out[i, h] = w @ v[slot, h // g]
    return out


DEEP = [(9, 4, 2, 128, 128, 16, 4), (30, 8, 2, 64, 64, 16, 10), (100, 4, 1, 128, 64, 32, 70), (140, 2, 2, 64, 128, 64, 33), (12, 6, 3, 80, 72, 16, 1), (70, 2, 1, 320, 300, 48, 20)]


@pytest.mark.parametrize("n,hq,hkv,dk,dv,page,window", DEEP)
def test_attention_plain_window_inside_the_tree(n, hq, hkv, dk, dv, page, window):
    s = deep_inputs(n, hq, hkv, dk, dv, page, window, torch.float32)
    assert torch.allclose(tree.tree_attention(**s).double(), by_definition(s), rtol=0, atol=2e-5)      # (sums of a few hundred f32 products, weights that add up to one)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hkv,dk,dv,page,window", DEEP)
def test_attention_kernel_window_inside_the_tree(n, hq, hkv, dk, dv, page, window, dtype):
    """Ancestors out of the window count no more than the context out of it: neither finite ones nor those that are no numbers."""
    s = deep_inputs(n, hq, hkv, dk, dv, page, window, dtype)
    got = tree.tree_attention(**on_gpu(s))
    _native.assert_status_ok()
    close(got, s)
    # the chain's root: its infinite feature reaches the nodes less than a window behind it, and no others
    slot = int(s["block_table"][0, 0]) * page
    s["v_cache"][slot, :, 3] = float("inf")
    got = tree.tree_attention(**on_gpu(s)).cpu()
    assert not torch.isfinite(got[:window, :, 3]).any() and torch.isfinite(got[window:]).all() and torch.isfinite(got[:, :, 4:]).all()


def stray_positions(dk, dtype):
    """Positions in front of the context and behind the last node's, and the same as the operator takes them: the nearest that a node can have."""
    n, ctx, window = 40, (0, 300, 1000), 20
    s = attention_inputs([n, n, n], list(ctx), 4, 2, dk, dk, 16, dtype, seed=3)
    g = torch.Generator().manual_seed(4)
    s["window"] = window
    s["positions"] = s["positions"] + torch.randint(-200, 200, (3 * n,), generator=g, dtype=torch.int32)
    s["positions"][::7], s["positions"][1::7] = -2 ** 31, 2 ** 31 - 1
    first = torch.tensor(ctx).repeat_interleave(n)
    return s, {**s, "positions": s["positions"].long().clamp(first, first + n - 1).int()}


def test_attention_plain_stray_positions():
    s, taken = stray_positions(64, torch.float32)
    got = tree.tree_attention(**s)
    assert torch.equal(got, tree.tree_attention(**taken)) and torch.allclose(got.double(), by_definition(taken), rtol=0, atol=2e-5)


@gpu
@pytest.mark.parametrize("dk,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32), (320, torch.float32)])
def test_attention_kernel_stray_positions(dk, dtype):
    """Both kernels answer alike, and what no row sees stays out, even where it is no number."""
    s, taken = stray_positions(dk, dtype)
    for seq, ctx in enumerate((0, 300, 1000)):
        place = torch.arange(max(0, ctx - 20 + 1))                         # in front of every window
        slot = s["block_table"][seq].long()[place // 16] * 16 + place % 16
        for x in ("k_cache", "v_cache"):
            s[x][slot] = float("nan")
    got = tree.tree_attention(**on_gpu(s))
    _native.assert_status_ok()
    close(got, taken)


@gpu
@pytest.mark.parametrize("seqs,hkv", [(24, 6), (25, 6), (37, 4), (38, 8)])
def test_attention_kernel_windows_around_a_round(seqs, hkv):
    """As many windowed items as there are SMs, some fewer and some more: left whole, or cut."""
    r = random.Random(seqs)
    s = attention_inputs([r.randint(1, 9) for _ in range(seqs)], [r.randint(0, 900) for _ in range(seqs)], 2 * hkv, hkv, 64, 64, 16, seed=seqs)
    s["window"] = 600
    close(tree.tree_attention(**on_gpu(s)), s)
    _native.assert_status_ok()


@gpu
def test_attention_kernel_single_rows():
    """The strides of dimensions of size one do not matter."""
    for nodes, hq, hkv in (([1], 4, 2), ([3], 1, 1)):
        s = attention_inputs(nodes, [40], hq, hkv, 64, 64, 16)
        c = on_gpu(s)
        c["q"] = c["q"].as_strided(c["q"].shape, (8, 64, 1) if nodes == [1] else (64, 8, 1))
        close(tree.tree_attention(**c), s)


@gpu
@pytest.mark.parametrize("nodes,hkv,ctx", [(8, 4, 4000), (40, 2, 1500)])
def test_attention_kernel_long_pieces(nodes, hkv, ctx):
    """Many items to a block, with last blocks in all states of filling: every run gives the same, right answer."""
    r = random.Random(nodes)
    n, c = ([r.randint(1, top) for _ in range(48)] for top in (nodes, ctx))
    s = attention_inputs(n, c, 4 * hkv, hkv, 128, 128, 128, seed=1)
    dev = on_gpu(s)
    cold = torch.empty(64 << 20, device="cuda")
    got = []
    for i in range(6):
        cold.fill_(i)                                                       # the cache comes from HBM again
        got.append(tree.tree_attention(**dev))
    close(got[0], s)
    assert all(torch.equal(g, got[0]) for g in got)


@gpu
def test_attention_kernel_rows_and_strides():
    """Query rows cut out of a wider projection; rows behind the last sequence keep what they hold; an empty batch."""
    s = attention_inputs([4, 9], [200, 33], 8, 2, 128, 128, 16)
    t = s["q"].shape[0]
    wide_q = torch.randn(t + 3, 8 * 128 + 512).bfloat16()
    wide_q[:t, :1024] = s["q"].reshape(t, -1)
    mask = torch.cat([s["mask"], torch.full((3, s["mask"].shape[1]), -1)])
    c = on_gpu({**s, "mask": mask, "positions": None})
    c["q"] = wide_q.cuda()[:, :1024].unflatten(1, (8, 128))
    c["out"] = torch.full((t + 3, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = tree.tree_attention(**c)
    assert got.data_ptr() == c["out"].data_ptr() and (got[t:] == 7).all()
    close(got[:t], s)
    e = on_gpu(attention_inputs([0, 0], [3, 4], 4, 2, 128, 128, 16))
    assert tree.tree_attention(**e).shape == (0, 4, 128)


@gpu
def test_attention_kernel_replays_with_other_lengths():
    """A captured call reads its lengths, tables and masks from the device: a replay with other ones answers for those."""
    a, b = (attention_inputs(n, c, 16, 4, 128, 128, 32, seed=5) for n, c in (([6, 14], [900, 40]), ([14, 6], [3, 1600])))
    pool, cols = max(x["k_cache"].shape[0] for x in (a, b)), max(x["block_table"].shape[1] for x in (a, b))
    static = None
    for s in (a, b):
        s["k_cache"], s["v_cache"] = (torch.cat([x, torch.zeros(pool - x.shape[0], *x.shape[1:], dtype=x.dtype)]) for x in (s["k_cache"], s["v_cache"]))
        s["block_table"] = torch.nn.functional.pad(s["block_table"], (0, cols - s["block_table"].shape[1]))
        s["max_nodes"] = 14
    static = on_gpu(a)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        tree.tree_attention(**static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tree.tree_attention(**static)
    for s in (b, a):
        for k, v in s.items():
            if torch.is_tensor(v):
                static[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        close(out, s)


@gpu
def test_attention_kernel_two_streams():
    """Calls on two streams at once do not share anything."""
    sets = [attention_inputs([20, 30], [3000, 2000], 16, 4, 128, 128, 64, seed=i) for i in range(2)]
    dev = [on_gpu(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(tree.tree_attention(**dev[i]))
    torch.cuda.synchronize()
    for i in range(2):
        close(got[i][0], sets[i])
        assert all(torch.equal(g, got[i][0]) for g in got[i])


# ------------------------------------------------------------------------------------------ draws
def draw_oracle(row, u, t, k, p, m):
    """The definition, one step after the other, in Python floats."""
    row = [float("-inf") if x != x else x for x in row]
    order = sorted(range(len(row)), key=lambda i: (-row[i], i))
    if row[order[0]] == float("-inf"):
        return 0, float("-inf")
    if not t > 0:
        return order[0], 0.0
    if k > 0:
        order = order[:k]
    top = row[order[0]]
    w = [1.0 if row[i] == top else math.exp((row[i] - top) / t) for i in order]
    w = [x if x > 2.0 ** -45 else 0.0 for x in w]
    total, front, kept = math.fsum(w), 0.0, []
    for i, x in zip(order, w):
        if kept and p < 1 and not front < p * total:
            break
        if x >= m:
            kept.append((i, x))
        front += x
    kept.sort()
    total = math.fsum(x for _, x in kept)
    at = 0.0
    for i, x in kept:
        at += x
        if x > 0 and at > u * total:
            break
    return i, math.log(x / total)


def draw_rows(b, v, dtype, seed, kind):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, v, generator=g) * 2.5
    if kind == "flat":
        x = torch.randn(b, v, generator=g) * 0.05
    if kind == "equal":
        x = torch.full((b, v), 3.25)
    if kind == "ties":
        x = torch.randint(-6, 3, (b, v), generator=g).float()
    if kind == "masked":
        x[torch.rand(b, v, generator=g) < 0.97] = float("-inf")
        x[torch.rand(b, v, generator=g) < 0.01] = float("nan")
        x[torch.rand(b, v, generator=g) < 0.3] = torch.finfo(dtype).min
    if kind == "far":
        x = x * 1000
    if kind == "infinite":
        x[:, v // 3] = float("inf")
        x[::2, v // 2] = float("inf")
    if kind == "none":
        x[:] = float("-inf")
        x[::2, 0] = float("nan")
    r = random.Random(seed)
    pick = lambda *vs: [r.choice(vs) for _ in range(b)]                    # noqa: E731
    f = lambda vs: torch.tensor(vs, dtype=torch.float32)                   # noqa: E731
    return dict(logits=x.to(dtype), uniform=torch.rand(b, generator=g), temperature=f(pick(0.0, 0.3, 0.8, 1.0, 1.7, 50.0)),
                top_k=torch.tensor(pick(0, 0, 1, 2, 7, 50, v // 2, v, v + 9, -4), dtype=torch.int32), top_p=f(pick(1.0, 1.0, 0.9, 0.5, 0.999, 0.05, 0.0, 1.5)),
                min_p=f(pick(0.0, 0.0, 0.05, 0.5, 1.0, 2.0)))


def same_draws(got, s):
    want, lp = sampling.draw_ref(**s)
    tok, lq = (x.cpu() for x in got)
    assert torch.equal(tok, want), [(i, int(a), int(b), *(float(s[k][i]) for k in ("uniform", "temperature", "top_k", "top_p", "min_p")))
                                    for i, (a, b) in enumerate(zip(tok, want)) if a != b][:5]
    # a logarithm of up to -31 in f32 (2^-24 of it), a mass that is off by 2^-45 an id: below 1e-8 of itself
    assert torch.equal(torch.isinf(lq), torch.isinf(lp)) and torch.allclose(lq, lp, rtol=2 ** -22, atol=2e-7)


KINDS = ["normal", "flat", "equal", "ties", "masked", "far", "infinite", "none"]


@pytest.mark.parametrize("kind", KINDS)
def test_draw_plain_is_the_definition(kind):
    s = draw_rows(60, 41, torch.float32, 3, kind)
    s["min_p"].clamp_(max=1.0)
    tok, lp = sampling.draw(**s, want_logprob=True)
    for i in range(60):
        t, want = draw_oracle(s["logits"][i].tolist(), *(x[i].item() for x in (s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])))
        assert int(tok[i]) == t and (float(lp[i]) == want or abs(float(lp[i]) - want) < 1e-5), (i, int(tok[i]), t)


def test_draw_scalars_and_refusals():
    s = draw_rows(4, 100, torch.float32, 1, "normal")
    x, u = s["logits"], s["uniform"]
    a = sampling.draw(x, u, 0.7, 20, 0.9, 0.01)
    b = sampling.draw(x, u, *(torch.full((4,), v, dtype=d) for v, d in ((0.7, torch.float32), (20, torch.int32), (0.9, torch.float32), (0.01, torch.float32))))
    assert torch.equal(a, b) and torch.equal(sampling.draw(x, u, 0.0), x.argmax(1).int())
    for bad in (dict(logits=x.half()), dict(logits=x[0]), dict(logits=x.t()), dict(uniform=u.double()), dict(uniform=u[:3]), dict(temperature=torch.ones(3)),
                dict(top_k=torch.ones(4)), dict(top_p=torch.ones(4, 1)), dict(min_p=torch.ones(4, dtype=torch.float64))):
        with pytest.raises(ValueError):
            sampling.draw(**{**s, **bad})


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 2, 37, 4096, 4099, 50257, 151936])
@pytest.mark.parametrize("kind", KINDS)
def test_draw_kernel(kind, v, dtype):
    s = draw_rows(97 if v < 50000 else 40, v, dtype, v, kind)
    got = sampling.draw(**on_gpu(s), want_logprob=True)
    _native.assert_status_ok()
    same_draws(got, s)
    assert torch.equal(got[0], sampling.draw(**on_gpu(s)))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 37, 1009, 2048])
@pytest.mark.parametrize("kind", KINDS)
def test_draw_kernel_many_short_rows(kind, v, dtype):
    s = draw_rows(700, v, dtype, v, kind)
    got = sampling.draw(**on_gpu(s), want_logprob=True)
    _native.assert_status_ok()
    same_draws(got, s)


@gpu
def test_draw_kernel_borders_and_strides():
    """Numbers of 0 and 1 and beyond; rows that begin at odd places; one row; no rows; the largest vocabulary."""
    s = draw_rows(50, 5001, torch.bfloat16, 9, "normal")
    s["uniform"][:8] = torch.tensor([0.0, 1.0, 2.0, -1.0, float("nan"), 1 - 2 ** -24, 2 ** -30, 0.5])
    same_draws(sampling.draw(**on_gpu(s), want_logprob=True), s)
    c = on_gpu(s)
    c["logits"] = torch.cat([torch.full((50, 3), 99.0, dtype=torch.bfloat16), s["logits"], torch.full((50, 2), 99.0, dtype=torch.bfloat16)], 1).cuda()[:, 3:-2]
    same_draws(sampling.draw(**c, want_logprob=True), s)
    one = {k: x[:1] for k, x in s.items()}
    same_draws(sampling.draw(**on_gpu(one), want_logprob=True), one)
    assert sampling.draw(**on_gpu({k: x[:0] for k, x in s.items()})).shape == (0,)
    s = draw_rows(6, 400_000, torch.float32, 2, "normal")
    same_draws(sampling.draw(**on_gpu(s), want_logprob=True), s)
    with pytest.raises(RuntimeError, match="vocabulary"):
        sampling.draw(torch.zeros(1, 420_000, device="cuda"), torch.zeros(1, device="cuda"))


@gpu
def test_draw_kernel_largest_masses():
    """Rows of as many ids as there is room for, all or nearly all equal: masses beyond 2^63."""
    v = 800_000
    r = random.Random(0)
    x = torch.full((12, v), 1.5)
    x[6:, torch.randint(0, v, (1000,), generator=torch.Generator().manual_seed(1))] = 1.0
    f = lambda vs: torch.tensor(vs, dtype=torch.float32)                   # noqa: E731
    s = dict(logits=x.bfloat16(), uniform=f([r.random() for _ in range(12)]), temperature=f([1.0] * 6 + [0.7, 1e9] * 3), top_k=torch.tensor([0, 0, 0, 700_000, 799_999, 0] * 2, dtype=torch.int32),
             top_p=f([1.0, 0.9, 0.99999, 1.0, 0.95, 0.3] * 2), min_p=f([0.0, 0.0, 0.5, 0.0, 0.0, 1.0] * 2))
    s["uniform"][0] = 1 - 2 ** -24
    got = sampling.draw(**on_gpu(s), want_logprob=True)
    _native.assert_status_ok()
    same_draws(got, s)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [3, 60])
def test_draw_kernel_likely_tokens_side_by_side(rows, dtype):
    """The likely tokens at neighbouring ids: one block of a row's cluster holds all candidates, more than its share of the places."""
    s = draw_rows(rows, 151936, dtype, rows, "normal")
    r = random.Random(rows)
    for row in s["logits"]:
        at = r.choice([0, 70_000, 150_000])
        row[at:at + 1500] += 12
    s["top_k"] = torch.tensor([r.choice([0, 200, 300, 700, 1000, 1400]) for _ in range(rows)], dtype=torch.int32)
    s["temperature"].fill_(1.1)
    got = sampling.draw(**on_gpu(s), want_logprob=True)
    _native.assert_status_ok()
    same_draws(got, s)


@gpu
def test_draw_kernel_frequencies():
    """Evenly spaced numbers meet every kept id as often as its probability says, to one number."""
    g = torch.Generator().manual_seed(0)
    row, n = torch.randn(1000, generator=g) * 2, 20000
    u = ((torch.arange(n) + 0.5) / n).float()
    tok = sampling.draw(row.cuda().expand(n, 1000).contiguous(), u.cuda(), 0.9, 200, 0.95).cpu().long()
    p = torch.softmax(row.double() / float(torch.tensor(0.9)), 0)
    top = torch.sort(p, descending=True)
    keep = torch.zeros(1000, dtype=torch.bool)
    q = top.values[:200] / top.values[:200].sum()
    keep[top.indices[:200][(q.cumsum(0) - q) < float(torch.tensor(0.95))]] = True
    want = torch.where(keep, p, 0.0) / p[keep].sum() * n
    assert (torch.bincount(tok, minlength=1000) - want).abs().max() <= 1.0 + 20000 * 2 ** -23


# ------------------------------------------------------------------------------------------ commit
def commit_inputs(nodes, ctx, page, shapes, seed=0, accept=0.8, vocab=5):
    """Trees over a tiny vocabulary (siblings with equal tokens among them); the drawn token of a node is often one of its children's."""
    r = random.Random(seed)
    ptr, ids, table, pool = paged(nodes, ctx, page, r)
    tok, par, drawn = [], [], []
    for n in nodes:
        p = random_tree(n, r) if n else []
        t = [r.randrange(vocab) for _ in p]
        kids = [[i for i in range(n) if p[i] == j] for j in range(n)]
        tok += t
        par += p
        drawn += [t[r.choice(k)] if k and r.random() < accept else r.randrange(vocab + 2) for k in kids]
    g = torch.Generator().manual_seed(seed)
    caches = [torch.randint(-100, 100, (pool * page, *sh), generator=g).to(dt) for sh, dt in shapes]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)                     # noqa: E731
    return dict(caches=caches, tokens=i32(tok), parents=i32(par), sampled=i32(drawn), cu_q=i32([0] + list(torch.tensor(nodes).cumsum(0))),
                kv_len=i32([a + b for a, b in zip(nodes, ctx)]), block_table=table, page_size=page, max_nodes=max(nodes + [1]))


COMMIT = [([1], [0], 16, [((2, 8), torch.bfloat16)]), ([6, 0, 20], [15, 4, 100], 16, [((2, 128), torch.bfloat16)] * 4),
          ([64, 33, 2, 1], [7, 0, 31, 400], 8, [((8, 128), torch.bfloat16), ((8, 128), torch.int8), ((8,), torch.float32), ((3,), torch.int8), ((5, 3), torch.bfloat16)]),
          ([256, 130], [1000, 3], 64, [((1, 64), torch.float32)] * 2), ([12] * 5, [9] * 5, 4, [((2, 8), torch.bfloat16)] * 300), ([5, 5], [3, 3], 16, [])]


@pytest.mark.parametrize("nodes,ctx,page,shapes", COMMIT)
def test_commit_plain_is_the_definition(nodes, ctx, page, shapes):
    s = commit_inputs(nodes, ctx, page, shapes)
    old = [c.clone() for c in s["caches"]]
    got = tree.tree_commit(**s)
    for q, (n, c) in enumerate(zip(nodes, ctx)):
        k, path = int(got.count[q]), got.path[q].tolist()
        a = int(s["cu_q"][q])
        assert (k > 0) == (n > 0) and path[k:] == [-1] * (len(path) - k) and int(got.kv_len[q]) == c + k
        for x, y in zip(path[:k], path[1:k]):
            kids = [i for i in range(n) if s["parents"][a + i] == x and s["tokens"][a + i] == s["sampled"][a + x]]
            assert kids[0] == y
        if n:
            assert path[0] == 0 and int(got.next_token[q]) == int(s["sampled"][a + path[k - 1]])
            assert not [i for i in range(n) if s["parents"][a + i] == path[k - 1] and s["tokens"][a + i] == s["sampled"][a + path[k - 1]]]
        slot = lambda p: int(s["block_table"][q, p // page]) * page + p % page       # noqa: E731,B023
        for new, was in zip(s["caches"], old):
            for j, x in enumerate(path[:k]):
                assert torch.equal(new[slot(c + j)], was[slot(c + x)])
            for p in list(range(c)) + list(range(c + k, c + n)):
                assert torch.equal(new[slot(p)], was[slot(p)])


@gpu
@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("nodes,ctx,page,shapes", COMMIT)
def test_commit_kernel(nodes, ctx, page, shapes, seed):
    s = commit_inputs(nodes, ctx, page, shapes, seed, accept=[0.8, 0.97, 0.2][seed], vocab=[5, 40, 3][seed])
    d = on_gpu({**s, "caches": None})
    d["caches"] = [c.cuda() for c in s["caches"]]
    got, want = tree.tree_commit(**d), tree.tree_commit(**s)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    for a, b in zip(d["caches"], s["caches"]):
        assert torch.equal(a.cpu(), b)


@gpu
def test_commit_kernel_missing_places():
    """A block table that is too short for the tree, and entries outside the cache: those rows stay, and nothing else is touched."""
    s = commit_inputs([40, 40], [60, 0], 16, [((2, 64), torch.bfloat16)], 1, accept=1.0, vocab=100)
    s["block_table"] = s["block_table"][:, :5].contiguous()
    s["block_table"][1, 1] = 10 ** 6
    s["block_table"][1, 2] = -3
    d = on_gpu({**s, "caches": None})
    d["caches"] = [c.cuda() for c in s["caches"]]
    got, want = tree.tree_commit(**d), tree.tree_commit(**s)
    for a, b in zip(list(got) + d["caches"], list(want) + s["caches"]):
        assert torch.equal(a.cpu(), b)


def test_commit_refusals():
    s = commit_inputs([4, 2], [3, 0], 8, [((2, 8), torch.bfloat16)] * 2)
    tree.tree_commit(**s)
    for bad in (dict(tokens=s["tokens"].long()), dict(parents=s["parents"][:3]), dict(sampled=s["sampled"][:1]), dict(cu_q=s["cu_q"][:2]), dict(max_nodes=0), dict(max_nodes=257),
                dict(page_size=0), dict(block_table=s["block_table"][0]), dict(caches=[s["caches"][0], s["caches"][1][:3]]), dict(caches=[s["caches"][0].transpose(1, 2)])):
        with pytest.raises(ValueError):
            tree.tree_commit(**{**s, **bad})


def test_commit_refuses_caches_that_overlap():
    """A row moved twice would be read after it was written."""
    s = commit_inputs([4, 2], [3, 0], 8, [((2, 8), torch.bfloat16)] * 2)
    for caches in ([s["caches"][0]] * 2, [s["caches"][0], s["caches"][0].flatten()[: -8 * s["caches"][0].shape[0]].view(-1, 8)]):
        with pytest.raises(ValueError, match="overlap"):
            tree.tree_commit(**{**s, "caches": caches})


@gpu
def test_commit_kernel_refuses_caches_that_overlap():
    s = commit_inputs([4, 2], [3, 0], 8, [((2, 8), torch.bfloat16)] * 2)
    d = on_gpu({**s, "caches": None})
    with pytest.raises(RuntimeError, match="overlap"):
        tree.tree_commit(**{**d, "caches": [s["caches"][0].cuda()] * 2})
    flat = s["caches"][0].cuda().flatten()                                     # neighbours in one buffer
    half = flat.numel() // 2
    want = tree.tree_commit(**{**s, "caches": [flat[:half].cpu().view(-1, 8), flat[half:].cpu().view(-1, 8)]})
    for a, b in zip(tree.tree_commit(**{**d, "caches": [flat[:half].view(-1, 8), flat[half:].view(-1, 8)]}), want):
        assert torch.equal(a.cpu(), b)


# ------------------------------------------------------------------------------------------ a step
def step_of(s):
    """A verification step in its parts, from tensors alone."""
    t = paging.batch_tables(s["q"], s["ctx"], s["ptr"], s["pages"], 16, s["parents"].numel(), 40, s["parents"], 12)
    o = tree.tree_attention(s["rows"], s["k"], s["v"], t.cu_q, t.kv_len, t.block_table, 16, t.mask, 12, window=64, positions=t.positions, out=torch.zeros_like(s["rows"]))
    logits = o.flatten(1)[:, :50] * 8
    tok, lp = sampling.draw(logits, s["u"], s["temp"], 5, s["top_p"], 0.02, want_logprob=True)
    return [t.slots, o, tok, lp] + list(tree.tree_commit([s["k"], s["v"]], s["tokens"], s["parents"], tok, t.cu_q, t.kv_len, t.block_table, 16, 12)) + [s["k"], s["v"]]


def step_inputs(seed):
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    q, ctx = [r.randint(0, 12) for _ in range(7)], [r.randint(0, 600) for _ in range(7)]
    pages = list(range(7 * 40))
    r.shuffle(pages)
    par = [p for n in q for p in (random_tree(n, r) if n else [])]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)                     # noqa: E731
    cut = lambda v: (v + [-1] * 84)[:84]                                    # noqa: E731
    need = [(a + b + 15) // 16 for a, b in zip(q, ctx)]
    ptr = [0] + [int(x) for x in torch.tensor(need).cumsum(0)]
    rnd = lambda *sh: torch.randn(*sh, generator=g).bfloat16()             # noqa: E731
    return dict(q=i32(q), ctx=i32(ctx), ptr=i32(ptr), pages=i32(pages), parents=i32(cut(par)), tokens=i32([r.randrange(4) for _ in range(84)]), rows=rnd(84, 8, 64) / 4,
                k=rnd(7 * 640, 2, 64), v=rnd(7 * 640, 2, 64), u=torch.rand(84, generator=g), temp=torch.rand(84, generator=g) * 2,
                top_p=torch.rand(84, generator=g))


@gpu
def test_captured_steps():
    """Two captured steps, replayed in turn with other lengths, trees and numbers, and one beside the other on two streams: what the eager calls answer, bit for bit."""
    cases = [{k: x.cuda() for k, x in step_inputs(i).items()} for i in range(4)]
    copy = lambda s: {k: x.clone() for k, x in s.items()}                   # noqa: E731
    want = [[x.clone() for x in step_of(copy(s))] for s in cases]
    static, graphs, outs = [copy(cases[0]), copy(cases[0])], [torch.cuda.CUDAGraph() for _ in range(2)], []
    torch.cuda.synchronize()
    for s, graph in zip(static, graphs):
        with torch.cuda.graph(graph):
            outs.append(step_of(s))
    for first, second in ((1, 2), (3, 0), (2, 2)):
        for s, i in zip(static, (first, second)):
            for k, x in s.items():
                x.copy_(cases[i][k])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got, i in zip(outs, (first, second)):
            for a, b in zip(got, want[i]):
                assert torch.equal(a, b)
    _native.assert_status_ok()
