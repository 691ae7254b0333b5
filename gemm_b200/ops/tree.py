"""Trees of drafted tokens over a paged KV cache: the attention of their nodes (csrc/kernels/tree_attn.cu, tree_any.cu) and, once the target model's tokens are
drawn, the acceptance of a path and the move of its K / V rows (csrc/kernels/tree_commit.cu).

A sequence with ``ctx`` committed tokens brings a tree of ``n`` nodes: node 0 is its last certain token, every other node a draft that continues its
parent, which has a lower index.  Node i is cached at place ``ctx + i`` of the sequence (``kv_len = ctx + n``) and has the position ``ctx + depth``
(``ops.paging.batch_tables`` makes these tables and the masks).
"""
from __future__ import annotations

import math
from array import array
from operator import attrgetter
from typing import NamedTuple, Optional, Sequence

import torch

from .. import _native
from .paging import MAX_NODES, check_int32

_TILE, _PAGES = (64, 128), (8, 16, 32, 64, 128)
_nbytes, _shape = attrgetter("nbytes"), attrgetter("shape")


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cu_q: torch.Tensor, kv_len: torch.Tensor, block_table: torch.Tensor,
                   page_size: int, mask: torch.Tensor, max_nodes: int, window: int = 0, positions: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention output ``[T, Hq, dv]`` of the nodes ``q [T, Hq, dk]`` (multiplied by scale * log2(e); rows may lie further apart than Hq * dk) over
    ``k_cache [slots, Hkv, dk]`` / ``v_cache [slots, Hkv, dv]``.  Sequence s has the nodes ``cu_q[s] .. cu_q[s + 1]`` (at most ``max_nodes`` <= 256), cached at
    its last places.  A node sees the places in front of the tree and the nodes whose bits are set in its row of ``mask`` (int64 ``[T, words]``, its own bit among
    them as a rule); with ``window`` > 0, of both those that are less than ``window`` in front of its ``positions`` entry (a place of the context by its number, a
    node by its own entry; ``ctx + depth`` as ``ops.paging.batch_tables`` makes them: an entry outside ``ctx .. ctx + nodes - 1`` counts as the nearest of these).  A node that sees nothing gets zeros; rows behind the last sequence stay as they were in ``out``.  Keys that a node does not see never count, even if their rows are not
    finite; a value that is not finite makes that feature of the nodes that see it not finite."""
    t, hq, dk = q.shape
    slots, hkv, dv = v_cache.shape
    dev, dtype = q.device, q.dtype
    b = kv_len.numel()
    q_ts, q_hs, q_es = q.stride()
    if t <= 1:
        q_ts = hq * dk
    if q_es != 1 or (hq > 1 and q_hs != dk) or q_ts < hq * dk:
        raise ValueError("q: the heads of a token lie one after the other")
    if k_cache.shape != (slots, hkv, dk) or not (k_cache.is_contiguous() and v_cache.is_contiguous()) or v_cache.dtype is not dtype or k_cache.dtype is not dtype:
        raise ValueError("contiguous caches of the same slots, heads and type as the queries are needed")
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise ValueError(f"tree_attention takes bf16 or f32, not {dtype}")
    if hkv < 1 or hq % hkv:
        raise ValueError(f"{hq} query heads do not share {hkv} KV heads evenly")
    check_int32(dev, "cu_q kv_len block_table", cu_q, kv_len, block_table)
    if cu_q.numel() != b + 1 or block_table.dim() != 2 or block_table.shape[0] != b or page_size < 1:
        raise ValueError("cu_q, kv_len and block_table name different numbers of sequences")
    if mask.dtype is not torch.int64 or mask.dim() != 2 or not mask.is_contiguous() or mask.device != dev or k_cache.device != dev or v_cache.device != dev:
        raise ValueError("mask: a contiguous int64 tensor [T, words] beside the queries is needed")
    rows, words = mask.shape
    if rows != t or not 1 <= max_nodes <= MAX_NODES or words * 64 < max_nodes or words > MAX_NODES // 64:
        raise ValueError(f"trees of 1 to {MAX_NODES} nodes with a mask bit each, not {max_nodes} in a mask [{rows}, {words}]")
    if window < 0 or (window > 0 and positions is None):
        raise ValueError("a window needs the nodes' positions")
    if positions is not None:
        check_int32(dev, "positions", positions)
        if positions.numel() != t:
            raise ValueError("positions: one for each node")
    if out is None:
        out = q.new_empty(t, hq, dv)
    elif out.shape != (t, hq, dv) or out.dtype is not dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out: a contiguous tensor [{t}, {hq}, {dv}] of the queries' type is needed")
    elif out.data_ptr() % 16:
        raise ValueError("out: a 16-byte boundary is needed")
    if dev.type != "cuda":
        return tree_attention_ref(q, k_cache, v_cache, cu_q, kv_len, block_table, page_size, mask, window, positions, out)
    if t == 0 or b == 0:
        return out
    if slots == 0:
        raise ValueError("an empty cache")
    cols = block_table.shape[1]
    qp, kp, vp = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    pos = positions.data_ptr() if positions is not None else None
    with _native.on_device(dev):
        # the tcgen05 kernel's forms: its tiles hold 64 or 128 columns, 128 rows and whole pages, and TMA wants 16-byte boundaries
        n = 0
        if dtype is torch.bfloat16 and dk in _TILE and dv in _TILE and page_size in _PAGES and hq // hkv <= 128 and not (q_ts & 7 or (qp | kp | vp) & 15):
            n = _native.entry("gb_tree_attn_workspace", "iiiiiiii")(b, cols, page_size, max_nodes, hq, hkv, dv, window)
        if n > 0:
            work = q.new_empty(n, dtype=torch.float32)
            rc = _native.entry("gb_tree_attn", "plpppppppiipipiliiiiiiipp")(
                qp, q_ts, kp, vp, out.data_ptr(), work.data_ptr(), cu_q.data_ptr(), kv_len.data_ptr(), block_table.data_ptr(), cols, page_size, mask.data_ptr(), words, pos,
                b, slots, t, max_nodes, hq, hkv, dk, dv, window, _native.status_ptr(), _native.stream())
            _native.check(rc, "gb_tree_attn", n=1 if n <= 4 else 2)
        else:
            rc = _native.entry("gb_tree_any", "plpppippp" + "iipipiliiiiiip")(
                qp, q_ts, kp, vp, out.data_ptr(), int(dtype is torch.float32), cu_q.data_ptr(), kv_len.data_ptr(), block_table.data_ptr(), cols, page_size,
                mask.data_ptr(), words, pos, b, slots, t, hq, hkv, dk, dv, window, _native.stream())
            _native.check(rc, "gb_tree_any")
    return out


def tree_attention_ref(q, k_cache, v_cache, cu_q, kv_len, block_table, page_size, mask, window=0, positions=None, out=None) -> torch.Tensor:
    """``tree_attention`` in plain f32 (f64 for f64 tensors)."""
    t, hq, _ = q.shape
    g = hq // k_cache.shape[1]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    if out is None:
        out = torch.zeros(t, hq, v_cache.shape[2], dtype=q.dtype, device=q.device)
    cu = cu_q.tolist()
    for s in range(len(cu) - 1):
        a, z, length = cu[s], cu[s + 1], int(kv_len[s])
        if z <= a:
            continue
        ctx = max(0, length - (z - a))
        place = torch.arange(min(length, block_table.shape[1] * page_size), device=q.device)
        slot = block_table[s].long()[place // page_size] * page_size + place % page_size
        off = place - ctx
        bits = mask[a:z][:, (off >> 6).clamp(0, mask.shape[1] - 1)] >> (off & 63) & 1
        see = (off < 0) | ((bits == 1) & (off < 64 * mask.shape[1]))
        if window > 0:
            pos = positions[a:z].long().clamp(ctx, ctx + z - a - 1)
            see &= torch.where(off < 0, place, pos[off.clamp(0, z - a - 1)]) > pos[:, None] - window
        k = k_cache[slot].to(wide).repeat_interleave(g, dim=1)
        v = v_cache[slot].to(wide).repeat_interleave(g, dim=1)
        sc = (torch.einsum("qhd,khd->hqk", q[a:z].to(wide), k) * math.log(2.0)).masked_fill(~see, float("-inf"))
        p = torch.softmax(sc, dim=-1).masked_fill(~see, 0.0)              # (a row that sees nothing is all NaN in front of the fill)
        fine = torch.isfinite(v)
        o = torch.einsum("hqk,khd->qhd", p, torch.where(fine, v, 0.0))
        for key in (~fine).flatten(1).any(1).nonzero()[:, 0].tolist():     # values that are not finite reach the rows that see them, and no others
            o += torch.where(see[:, key, None, None] & ~fine[key], v[key], 0.0)
        out[a:z] = o.to(out.dtype)
    return out


class Accepted(NamedTuple):
    count: torch.Tensor                     # int32 [B] nodes on the accepted path, the root among them (0: a sequence without nodes)
    path: torch.Tensor                      # int32 [B, max_nodes] their indices, then -1
    next_token: torch.Tensor                # int32 [B] the token drawn at the path's last node (-1: no nodes)
    kv_len: torch.Tensor                    # int32 [B] committed length: ctx + count


def tree_commit(caches: Sequence[torch.Tensor], tokens: torch.Tensor, parents: torch.Tensor, sampled: torch.Tensor, cu_q: torch.Tensor, kv_len: torch.Tensor,
                block_table: torch.Tensor, page_size: int, max_nodes: int) -> Accepted:
    """Accepts, from the root of every tree, the first child whose token (``tokens``) is the one drawn at its parent (``sampled``), as long as there is one, and
    moves the accepted nodes' rows of all ``caches`` (``[slots, ...]`` contiguous, any type, e.g. every layer's K and V) from the places ``ctx + node`` to
    ``ctx, ctx + 1, ...``, in place.  ``tokens`` / ``parents`` / ``sampled``: int32 ``[T]``; the lengths and tables are those of the verifying pass (``kv_len``
    includes the tree).  The caches do not overlap.  No caches: the walk alone."""
    dev, t, b = tokens.device, tokens.numel(), kv_len.numel()
    check_int32(dev, "tokens parents sampled cu_q kv_len block_table", tokens, parents, sampled, cu_q, kv_len, block_table)
    if parents.numel() != t or sampled.numel() != t:
        raise ValueError("tokens, parents and sampled name different numbers of nodes")
    if cu_q.numel() != b + 1 or block_table.dim() != 2 or block_table.shape[0] != b or page_size < 1 or b > 65535:
        raise ValueError("cu_q, kv_len and block_table name different numbers of sequences")
    if not 1 <= max_nodes <= MAX_NODES:
        raise ValueError(f"trees of 1 to {MAX_NODES} nodes, not {max_nodes}")
    # (two caches a layer: by maps over the list, a loop of Python steps took 45 us of 56)
    shapes = set(map(_shape, caches))
    slots = next((s[0] for s in shapes if s), 0)
    on = dev.index if dev.type == "cuda" else -1
    if not all(map(torch.Tensor.is_contiguous, caches)) or set(map(torch.Tensor.get_device, caches)) - {on} or any(not s or s[0] != slots for s in shapes):
        raise ValueError("contiguous caches of equal numbers of slots beside the tokens are needed")
    if dev.type != "cuda":
        spans = sorted((c.data_ptr(), c.nbytes) for c in caches if c.nbytes)
        if any(a + n > z for (a, n), (z, _) in zip(spans, spans[1:])):
            raise ValueError("tree_commit: caches that overlap")
        return tree_commit_ref(caches, tokens, parents, sampled, cu_q, kv_len, block_table, page_size, max_nodes)
    with _native.on_device(dev):
        count, nxt, new, path = kv_len.new_empty(b * (3 + max_nodes)).split_with_sizes((b, b, b, b * max_nodes))
        ptrs = array("Q", map(torch.Tensor.data_ptr, caches))
        alike = len(shapes) == 1 and len(set(map(torch.Tensor.element_size, caches))) == 1
        sizes = array("q", (caches[0].nbytes,)) * len(ptrs) if alike else array("q", map(_nbytes, caches))
        rc = _native.entry("gb_tree_commit", "ppilppppppiiiiippppp")(
            ptrs.buffer_info()[0], sizes.buffer_info()[0], len(ptrs), slots, tokens.data_ptr(), parents.data_ptr(), sampled.data_ptr(), cu_q.data_ptr(),
            kv_len.data_ptr(), block_table.data_ptr(), block_table.shape[1], page_size, b, t, max_nodes, count.data_ptr(), path.data_ptr(), nxt.data_ptr(),
            new.data_ptr(), _native.stream())
        _native.check(rc, "gb_tree_commit", n=max(1, (len(ptrs) + 223) // 224) if b else 0)
    return Accepted(count, path.view(b, max_nodes), nxt, new)


def tree_commit_ref(caches, tokens, parents, sampled, cu_q, kv_len, block_table, page_size, max_nodes) -> Accepted:
    """``tree_commit`` in plain Python."""
    cu, tok, par, drawn = cu_q.tolist(), tokens.tolist(), parents.tolist(), sampled.tolist()
    count, paths, nxt, new = [], [], [], []
    for s in range(len(cu) - 1):
        a, n = cu[s], min(max(cu[s + 1] - cu[s], 0), max_nodes)
        ctx = int(kv_len[s]) - max(cu[s + 1] - cu[s], 0)
        path = [0] if n else []
        while path:
            kid = next((i for i in range(path[-1] + 1, n) if par[a + i] == path[-1] and tok[a + i] == drawn[a + path[-1]]), None)
            if kid is None:
                break
            path.append(kid)
        for j, node in enumerate(path):
            src, dst = ((ctx + x) for x in (node, j))
            if node != j and dst >= 0 and src // page_size < block_table.shape[1]:
                src, dst = (int(block_table[s, x // page_size]) * page_size + x % page_size for x in (src, dst))
                for c in caches:
                    if c.numel() and 0 <= src < c.shape[0] and 0 <= dst < c.shape[0]:
                        c[dst] = c[src]
        count.append(len(path))
        paths.append(path + [-1] * (max_nodes - len(path)))
        nxt.append(drawn[a + path[-1]] if path else -1)
        new.append(ctx + len(path))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=tokens.device)          # noqa: E731
    return Accepted(i32(count), i32(paths).reshape(len(count), max_nodes), i32(nxt), i32(new))
