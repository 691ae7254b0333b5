"""Tables of a forward pass over a paged KV cache, built on the GPU from the lengths of its requests (csrc/kernels/paging.cu)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _native

MAX_SEQS = 8192
MAX_NODES = 256                   # nodes of a tree of drafted tokens: four 64-bit words of mask


def check_int32(device, names: str, *tensors) -> None:
    """Raise ``ValueError`` unless every tensor is a contiguous int32 one on ``device``."""
    for i, t in enumerate(tensors):
        if t.dtype is not torch.int32 or t.device != device or not t.is_contiguous():
            raise ValueError(f"{names.split()[i]}: a contiguous int32 tensor on {device} is needed, not {t.dtype} on {t.device}")


class BatchTables(NamedTuple):
    cu_q: torch.Tensor                      # int32 [B + 1]
    kv_len: torch.Tensor                    # int32 [B] length including the step's tokens
    positions: torch.Tensor                 # int32 [T]
    slots: torch.Tensor                     # int32 [T] (-1: no place in the cache)
    block_table: torch.Tensor               # int32 [B, max_pages]
    mask: Optional[torch.Tensor] = None     # int64 [T, words]: trees only


def mask_words(max_nodes: int) -> int:
    """64-bit words of a node's mask."""
    return (max_nodes + 63) // 64


def batch_tables(q_lens: torch.Tensor, ctx_lens: torch.Tensor, page_ptr: torch.Tensor, pages: torch.Tensor, page_size: int, total_tokens: int,
                 max_pages: int, parents: Optional[torch.Tensor] = None, max_nodes: int = 0) -> BatchTables:
    """Sequence s brings ``q_lens[s]`` tokens on top of ``ctx_lens[s]`` cached ones; its pages are ``pages[page_ptr[s] : page_ptr[s + 1]]`` (all int32).  Tokens are
    packed in sequence order into ``total_tokens`` rows; rows behind the last token get slot -1 and position 0 (tokens beyond ``total_tokens`` are dropped).
    ``block_table`` has ``max_pages`` columns, zero where a sequence has no page.  A token whose page a sequence does not have gets slot -1.

    ``parents`` (int32 ``[total_tokens]``; trees of drafted tokens, at most ``max_nodes`` <= 256 a sequence): the index within its sequence of every token's parent,
    which comes in front of it; -1 at a root.  The slot of a node still goes by its index, its position is ``ctx + depth``, and ``mask`` has a bit for
    each of its ancestors and for itself: what ``ops.tree.tree_attention`` takes."""
    b, dev = q_lens.numel(), q_lens.device
    check_int32(dev, "q_lens ctx_lens page_ptr pages", q_lens, ctx_lens, page_ptr, pages)
    if ctx_lens.numel() != b or page_ptr.numel() != b + 1:
        raise ValueError(f"{b} lengths go with as many context lengths and one more page pointer, not {ctx_lens.numel()} and {page_ptr.numel()}")
    if b > MAX_SEQS or page_size < 1 or total_tokens < 0 or max_pages < 0:
        raise ValueError(f"batch_tables: at most {MAX_SEQS} sequences, pages of at least one token, no negative sizes")
    words = 0
    if parents is not None:
        check_int32(dev, "parents", parents)
        if parents.numel() != total_tokens or not 1 <= max_nodes <= MAX_NODES:
            raise ValueError(f"a parent for each of the {total_tokens} tokens is needed, and trees of 1 to {MAX_NODES} nodes")
        words = mask_words(max_nodes)
    if dev.type != "cuda":
        return batch_tables_ref(q_lens, ctx_lens, page_ptr, pages, page_size, total_tokens, max_pages, parents, max_nodes)
    with _native.on_device(dev):
        # one buffer for all that is int32, every table on a 16-byte boundary
        gap, rows = -total_tokens & 3, b * max_pages
        x1, x2 = -(b + 1) & 3, -b & 3
        cu, _, kv, _, pos, _, slots, _, table = q_lens.new_empty(2 * (b + total_tokens + gap) + 1 + x1 + x2 + rows).split_with_sizes(
            (b + 1, x1, b, x2, total_tokens, gap, total_tokens, gap, rows))
        mask = q_lens.new_empty(total_tokens, words, dtype=torch.int64) if words else None
        rc = _native.entry("gb_batch_tables", "ppppiiiiipippppppp")(
            q_lens.data_ptr(), ctx_lens.data_ptr(), page_ptr.data_ptr(), pages.data_ptr(), pages.numel(), b, page_size, total_tokens, max_pages,
            parents.data_ptr() if words else None, max_nodes, cu.data_ptr(), kv.data_ptr(), pos.data_ptr(), slots.data_ptr(), table.data_ptr(),
            mask.data_ptr() if words else None, _native.stream())
        _native.check(rc, "gb_batch_tables")
    return BatchTables(cu, kv, pos, slots, table.view(b, max_pages), mask)


def batch_tables_ref(q_lens, ctx_lens, page_ptr, pages, page_size, total_tokens, max_pages, parents=None, max_nodes=0) -> BatchTables:
    """``batch_tables`` in plain Python."""
    ptr, ids = page_ptr.tolist(), pages.tolist()
    par = parents.tolist() if parents is not None else None
    words = mask_words(max_nodes) if par is not None else 0
    cu, kv, pos, slots, table, masks = [0], [], [0] * total_tokens, [-1] * total_tokens, [], [[0] * words for _ in range(total_tokens)]
    for s, (q, ctx) in enumerate(zip(q_lens.tolist(), ctx_lens.tolist())):
        mine = ids[max(ptr[s], 0): max(0, ptr[s + 1])]
        begin = cu[-1]
        q = min(max(q, 0), total_tokens - begin)
        table.append((mine + [0] * max_pages)[:max_pages])
        for i in range(q):
            place = ctx + i
            if place >= 0 and place // page_size < len(mine):
                slots[begin + i] = mine[place // page_size] * page_size + place % page_size
            depth = 0
            if par is not None:
                x, bits = i, 0
                while True:
                    bits |= 1 << x
                    p = par[begin + x]
                    if p < 0 or p >= x:
                        break
                    x, depth = p, depth + 1
                for w in range(words):
                    v = bits >> (64 * w) & (1 << 64) - 1
                    masks[begin + i][w] = v - (1 << 64) if v >> 63 else v
            pos[begin + i] = place if par is None else ctx + depth
        kv.append(ctx + q)
        cu.append(begin + q)
    dev = q_lens.device
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)         # noqa: E731
    return BatchTables(t(cu), t(kv), t(pos), t(slots), t(table).reshape(len(kv), max_pages),
                       torch.tensor(masks, dtype=torch.int64, device=dev).reshape(total_tokens, words) if par is not None else None)
