"""Attention of drafted token trees over the paged cache (libkvc
`kvc_tree_attention`) and the move that keeps an accepted path
(`kvc_commit_rows`).

A step of tree speculation: the drafted tokens' keys and values are appended
at the positions after the context, tree_attention gives every drafted token
the context and its own path, the accepted root-to-leaf path's rows are moved
to the context's end by commit_tree_path (in every layer at once), and the
context grows by the path's length.  The engine drafts nothing; there is no
reference counterpart.
"""
from __future__ import annotations

import torch

from .. import _native as nat
from .scored import _int32, check_pool, check_queries, check_scores


def tree_mask_from_parents(parents, device=None) -> torch.Tensor:
    """The mask of drafted trees from their parents: `parents` is one list per
    sequence, parents[i][t] the index of token t's parent in its own tree (-1
    for a root), which comes before it.  Returns int64 [tokens, words], the
    path from the root to each token, the token included, as bits."""
    rows, widest = [], 0
    for tree in parents:
        bits = []
        for t, parent in enumerate(tree):
            if not -1 <= parent < t:
                raise ValueError(f"token {t}'s parent {parent} does not come before it")
            bits.append((bits[parent] if parent >= 0 else 0) | (1 << t))
        rows += bits
        widest = max(widest, len(tree))
    words = max(1, (widest + 63) // 64)
    full = (1 << 64) - 1
    table = [[b >> (64 * w) & full for w in range(words)] for b in rows]
    table = [[x - (1 << 64) if x >> 63 else x for x in row] for row in table]
    return torch.tensor(table, dtype=torch.int64, device=device).view(len(rows), words)


def tree_attention(q, k_cache, v_cache, block_tables, context_lens, tree_mask, scale, *,
                   cu_seqlens_q=None, max_seqlen_q=None, softcap=0.0, alibi_slopes=None, window=0):
    """q: [T, H, 128] bf16, the drafted tokens of all sequences; sequence i's
    are rows cu_seqlens_q[i] .. cu_seqlens_q[i + 1] - 1 (int32 on the device),
    at most max_seqlen_q of them; without cu_seqlens_q every sequence has
    T / batch.  Their keys are in the pool at positions context_lens[i] + t.
    Token t sees every context key and the tree keys of its mask (tree_mask
    int64 [T, words], bit u % 64 of word u / 64).  softcap, alibi_slopes and
    window as in scored_attention, with the token's depth (bits in its mask,
    less one) for its distance from the context.  Returns out [T, H, 128]; a
    token that sees no key gives 0, rows of no tree are not written."""
    if nat.is_current(q):
        done = nat.host().tree(q, k_cache, v_cache, block_tables, context_lens, tree_mask, scale,
                               cu_seqlens_q, max_seqlen_q, softcap, alibi_slopes, window,
                               nat.stream_of(q))
        if done is not None:
            return done
    q = check_queries(q, k_cache.size(2), "tree attention")
    T, num_heads, head_dim = q.shape
    block_tables = check_pool(q, k_cache, v_cache, block_tables)
    softcap, alibi_slopes, window = check_scores(scale, softcap, alibi_slopes, window, num_heads,
                                                 q.device)
    batch = block_tables.size(0)
    context_lens = _int32(context_lens, batch, "context_lens", q.device)
    if cu_seqlens_q is None:
        if batch == 0 or T % batch:
            raise ValueError(f"{T} drafted tokens do not divide over {batch} sequences")
        max_seqlen_q = T // batch
    else:
        cu_seqlens_q = _int32(cu_seqlens_q, batch + 1, "cu_seqlens_q", q.device)
        if max_seqlen_q is None:
            raise ValueError("cu_seqlens_q needs max_seqlen_q, the longest tree")
    if tree_mask.dtype != torch.int64 or tree_mask.ndim != 2 or tree_mask.size(0) != T:
        raise ValueError("tree_mask must be int64 [tokens, words]")
    if tree_mask.size(1) * 64 < max_seqlen_q:
        raise ValueError(f"tree_mask has {tree_mask.size(1)} words for trees of {max_seqlen_q}")
    if tree_mask.device != q.device:
        raise ValueError("tree_mask must be on q's device")
    tree_mask = tree_mask.contiguous()
    nat.require_device(q)
    out = torch.empty((T, num_heads, head_dim), dtype=q.dtype, device=q.device)
    if T == 0:
        return out
    kvh = k_cache.size(2)
    need = nat.query("kvc_tree_workspace_bytes", T, num_heads, kvh, batch, max_seqlen_q)
    ws = nat.workspace(need, q.device)
    nat.call_on(
        q, "kvc_tree_attention", q.data_ptr(), q.stride(0), q.stride(1), T, num_heads,
        k_cache.data_ptr(), v_cache.data_ptr(), k_cache.size(0), k_cache.size(1), kvh, head_dim,
        block_tables.data_ptr(), block_tables.stride(0), block_tables.size(1), batch,
        context_lens.data_ptr(), nat.ptr(cu_seqlens_q), max_seqlen_q, tree_mask.data_ptr(),
        tree_mask.size(1), nat.ptr(alibi_slopes), softcap, window, float(scale), out.data_ptr(),
        out.stride(0), out.stride(1), nat.ptr(ws), need, nat.stream_of(q))
    return out


def commit_tree_path(kv_cache, block_tables, context_lens, paths, path_lens):
    """Keeps the accepted path of every sequence's tree, in place: for each
    sequence b and j < path_lens[b], the token row at position
    context_lens[b] + paths[b, j] of the pool goes to position
    context_lens[b] + j, in every layer, K and V, as one simultaneous move
    (the context then grows by path_lens[b]).  kv_cache is the whole pool
    [2, L, blocks, page, ...], or a companion of an int8 pool of that shape
    (scales, side rows); paths int32 [batch, most], a path strictly
    increasing (tree tokens come after their parents): it ends at the first
    entry that is not.  No two sequences may share the pages behind their
    contexts."""
    if nat.is_current(kv_cache) and nat.host().commit(kv_cache, block_tables, context_lens, paths,
                                                      path_lens, nat.stream_of(kv_cache)):
        return
    if kv_cache.dim() < 4:
        raise ValueError("pool must be [2, layers, blocks, page, ...]")
    if not kv_cache.is_contiguous():
        raise AssertionError("the KV pool must be contiguous")
    if block_tables.ndim != 2 or paths.ndim != 2 or paths.size(0) != block_tables.size(0):
        raise ValueError("expected block_tables=[batch,pages] and paths=[batch,most]")
    dev = kv_cache.device
    if not (block_tables.device == paths.device == dev):
        raise ValueError("the pool, block_tables and paths must be on one device")
    batch = block_tables.size(0)
    context_lens = _int32(context_lens, batch, "context_lens", dev)
    path_lens = _int32(path_lens, batch, "path_lens", dev)
    if block_tables.dtype != torch.int32 or block_tables.stride(1) != 1:
        block_tables = block_tables.to(torch.int32).contiguous()
    if paths.dtype != torch.int32 or paths.stride(1) != 1:
        paths = paths.to(torch.int32).contiguous()
    nat.require_device(kv_cache)
    if kv_cache.numel() == 0 or batch == 0:
        return
    blocks, page = kv_cache.size(2), kv_cache.size(3)
    plane = kv_cache[0, 0].numel() * kv_cache.element_size()
    nat.call_on(
        kv_cache, "kvc_commit_rows", kv_cache.data_ptr(), kv_cache.size(0) * kv_cache.size(1),
        plane, blocks, page, plane // (blocks * page), block_tables.data_ptr(),
        block_tables.stride(0), block_tables.size(1), context_lens.data_ptr(), paths.data_ptr(),
        paths.stride(0), paths.size(1), path_lens.data_ptr(), batch, nat.stream_of(kv_cache))
