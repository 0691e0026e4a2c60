"""Attention with shaped scores over the paged cache (libkvc
`kvc_scored_attention`): scores capped by a tanh, a bias by distance (one
slope per query head), a sliding window and a two-way prefix, for the same
rows as `varlen_attention` (decode rows first, then prefill chunks).

The engine's own models need none of these (nanovllm/layers/attention.py:
130-279 is causal and unshaped); this is the entry point for models that do.
The lengths are read on the device, so a call whose arguments stay in place
can be captured into a graph.
"""
from __future__ import annotations

import torch

from .. import _native as nat


def _rows_ok(t: torch.Tensor) -> bool:
    """Rows that the kernels read 16 bytes at a time."""
    return (t.stride(-1) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0
            and t.data_ptr() % 16 == 0)


def check_scores(scale, softcap, alibi_slopes, window, num_heads, device):
    """The score arguments shared by scored_attention and tree_attention,
    checked; returns (softcap, slopes, window) in the launch's form."""
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale must be finite and > 0 (got {scale})")
    softcap = float(softcap or 0.0)
    if not 0.0 <= softcap < float("inf"):
        raise ValueError(f"softcap must be finite and >= 0 (got {softcap})")
    window = int(window or 0)
    if not 0 <= window < 1 << 30:
        raise ValueError(f"window must be >= 0 (got {window})")
    if alibi_slopes is not None:
        if alibi_slopes.numel() != num_heads:
            raise ValueError(f"alibi_slopes must hold {num_heads} slopes, one per query head")
        if alibi_slopes.device != device:
            raise ValueError("alibi_slopes must be on q's device")
        alibi_slopes = alibi_slopes.to(torch.float32).contiguous()
    return softcap, alibi_slopes, window


def check_pool(q, k_cache, v_cache, block_tables):
    """The paged pool's arguments, checked; returns int32 block tables."""
    if k_cache.ndim != 4 or v_cache.shape != k_cache.shape or k_cache.size(3) != q.size(2):
        raise ValueError("expected kv=[pages,page,kv_heads,dim]")
    if k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise ValueError(f"KV pool dtype {k_cache.dtype} is not supported (bf16)")
    if k_cache.size(1) % 32:
        raise ValueError("page_size must be a multiple of 32")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise AssertionError("KV pools must be contiguous [pages, page, kv_heads, dim]")
    if not (q.device == k_cache.device == v_cache.device == block_tables.device):
        raise ValueError("q, the pools and block_tables must be on one device")
    if block_tables.ndim != 2:
        raise ValueError("block_tables must be [rows, pages]")
    if block_tables.dtype != torch.int32:
        block_tables = block_tables.to(torch.int32)
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    return block_tables


def check_queries(q, num_kv_heads, what):
    if q.ndim != 3 or q.size(2) != 128:
        raise ValueError(f"{what} requires q=[tokens,heads,128]")
    if q.dtype != torch.bfloat16:
        raise ValueError(f"q must be bf16 (got {q.dtype})")
    if num_kv_heads == 0 or q.size(1) % num_kv_heads:
        raise ValueError("num_heads must be a multiple of num_kv_heads")
    return q if _rows_ok(q) else q.contiguous()


def _int32(t, n, what, device):
    if t is None or t.numel() != n:
        raise ValueError(f"{what} must hold {n} values")
    if t.device != device:
        raise ValueError(f"{what} must be on q's device")
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def scored_attention(q, k_cache, v_cache, *, scale, block_tables=None, num_decode_rows=0,
                     decode_context_lens=None, cu_seqlens_q=None, cu_seqlens_k=None,
                     cu_seqlens_q_list=None, cu_seqlens_k_list=None, k=None, v=None,
                     softcap=0.0, alibi_slopes=None, window=0, prefix_lens=None, out=None):
    """q: [T, H, 128] bf16 with T = num_decode_rows + prefill tokens, rows and
    keys as in varlen_attention (a bf16 pool through block_tables, or the
    step's fresh k / v when block_tables is None; cu_seqlens_q starts at 0,
    the first row after the decode rows).  A query at place p sees
    key j when j <= p or j < prefix_lens[i] (int32, one per prefill chunk),
    and, with a window, p - j < window; its score is scale q.k, then
    softcap * tanh(score / softcap) if softcap > 0, then minus
    alibi_slopes[h] * |p - j| (fp32 [H]) if given.  Returns out [T, H, 128]
    bf16 (the given one, or a new one); a query that sees no key gives 0."""
    if out is None and nat.is_current(q):
        done = nat.host().scored(q, k_cache, v_cache, block_tables, num_decode_rows,
                                 decode_context_lens, cu_seqlens_q, cu_seqlens_k,
                                 cu_seqlens_q_list, cu_seqlens_k_list, k, v, softcap,
                                 alibi_slopes, window, prefix_lens, scale, nat.stream_of(q))
        if done is not None:
            return done
    fresh = block_tables is None
    if fresh and (k is None or v is None):
        raise ValueError("without block_tables the keys come from k/v")
    q = check_queries(q, k.size(1) if fresh else k_cache.size(2), "scored attention")
    T, num_heads, head_dim = q.shape
    softcap, alibi_slopes, window = check_scores(scale, softcap, alibi_slopes, window, num_heads,
                                                 q.device)
    num_prefill, max_q, keys = 0, 0, 0
    if cu_seqlens_q_list is not None or cu_seqlens_q is not None:
        cu_q = cu_seqlens_q_list if cu_seqlens_q_list is not None else cu_seqlens_q.tolist()
        cu_k = cu_seqlens_k_list if cu_seqlens_k_list is not None else cu_seqlens_k.tolist()
        num_prefill = len(cu_q) - 1
        if len(cu_k) != len(cu_q) or not cu_q:
            raise ValueError("cu_seqlens_q and cu_seqlens_k differ in length or are empty")
        if cu_q[0] != 0 or cu_k[0] < 0:
            raise ValueError("cu_seqlens_q must start at 0, cu_seqlens_k at 0 or later (got "
                             f"{cu_q[0]}, {cu_k[0]})")
        for i in range(num_prefill):
            n, m = cu_q[i + 1] - cu_q[i], cu_k[i + 1] - cu_k[i]
            if n < 0 or m < 0 or (n > 0 and m < n):
                raise ValueError("a prefill chunk has fewer keys than queries")
            max_q = max(max_q, n)
        keys = cu_k[-1]
        tokens = cu_q[-1]
    else:
        tokens = 0
    if num_decode_rows + tokens != T:
        raise ValueError(f"{T} query rows but {num_decode_rows} decode rows + "
                         f"{tokens} prefill tokens")
    if num_prefill:
        if cu_seqlens_q is None or cu_seqlens_q.device != q.device:
            cu_seqlens_q = torch.tensor(cu_q, dtype=torch.int32, device=q.device)
        if cu_seqlens_k is None or cu_seqlens_k.device != q.device:
            cu_seqlens_k = torch.tensor(cu_k, dtype=torch.int32, device=q.device)
        cu_seqlens_q = _int32(cu_seqlens_q, num_prefill + 1, "cu_seqlens_q", q.device)
        cu_seqlens_k = _int32(cu_seqlens_k, num_prefill + 1, "cu_seqlens_k", q.device)
    if num_decode_rows:
        decode_context_lens = _int32(decode_context_lens, num_decode_rows, "decode_context_lens",
                                     q.device)
    if prefix_lens is not None:
        prefix_lens = _int32(prefix_lens, num_prefill, "prefix_lens", q.device)
    if fresh:
        if num_decode_rows:
            raise ValueError("decode rows need a paged pool and block_tables")
        if k.ndim != 3 or v.shape != k.shape or k.size(2) != head_dim or k.size(0) < keys:
            raise ValueError("expected k/v=[keys,kv_heads,128]")
        if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
            raise ValueError("k and v must be bf16")
        if k.device != q.device or v.device != q.device:
            raise ValueError("k and v must be on q's device")
        k, v = (t if _rows_ok(t) else t.contiguous() for t in (k, v))
        kvh, page, blocks, max_blocks = k.size(1), 0, 0, 0
        ks, vs = k.stride(), v.stride()
        pool = (None, None, 0, 0, kvh, head_dim, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0],
                vs[1], k.size(0), None, 0, 0)
    else:
        block_tables = check_pool(q, k_cache, v_cache, block_tables)
        if block_tables.size(0) < num_decode_rows + num_prefill:
            raise ValueError("block_tables has fewer rows than the call has sequences")
        blocks, page, kvh = k_cache.size(0), k_cache.size(1), k_cache.size(2)
        max_blocks = block_tables.size(1)
        pool = (k_cache.data_ptr(), v_cache.data_ptr(), blocks, page, kvh, head_dim, None, 0, 0,
                None, 0, 0, 0, block_tables.data_ptr(), block_tables.stride(0), max_blocks)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype
                            or out.device != q.device or not _rows_ok(out)):
        raise ValueError("out must be bf16 [tokens,heads,128] on q's device, its rows 16-byte "
                         "aligned")
    nat.require_device(q)
    if out is None:
        out = torch.empty((T, num_heads, head_dim), dtype=q.dtype, device=q.device)
    if T == 0:
        return out
    need = nat.query("kvc_scored_workspace_bytes", T, num_heads, kvh, num_decode_rows, num_prefill,
                     max_q)
    ws = nat.workspace(need, q.device)
    nat.call_on(
        q, "kvc_scored_attention", q.data_ptr(), q.stride(0), q.stride(1), T, num_heads, *pool,
        num_decode_rows, decode_context_lens.data_ptr() if num_decode_rows else None, num_prefill,
        cu_seqlens_q.data_ptr() if num_prefill else None,
        cu_seqlens_k.data_ptr() if num_prefill else None, max_q, nat.ptr(prefix_lens),
        nat.ptr(alibi_slopes), softcap, window, float(scale), out.data_ptr(), out.stride(0),
        out.stride(1), nat.ptr(ws), need, nat.stream_of(q))
    return out
