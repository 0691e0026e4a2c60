"""KV cache in 4-bit floats: quantise on append, dequantise on read, paged decode
(libkvc `kvc_*_fp4`; the engine has no counterpart).

The pool holds codes uint8 [blocks, page, KVH, 64] (two dims a byte, the even one
in the low half: bit 3 the sign, 0 .. 7 = 0, 0.5, 1, 1.5, 2, 3, 4, 6) and scales
uint8 [blocks, page, KVH, 4]: byte g is the exponent + 127 of the power of two
that scales dims 32 g .. 32 g + 31, the smallest that brings the run's largest
magnitude to 6 or less (2^-126 at least, 2^125 at most).  Values round to the
nearest code, ties to the even mantissa; a run that holds an infinity or a NaN
is NaN (scale 255).  68 bytes a row of 128, 3.8 times fewer than bf16.

Where an int8 pool's entry points take k_scale / v_scale, those of a 4-bit pool
take these: paged_decode_attention, varlen_attention and gather_kv go by the
pool's dtype.
"""
from __future__ import annotations

import torch

from .. import _native as nat
from .kv_int8 import _check_rows, _slots

ROW_BYTES = 64
POWERS = 4


def check_fp4_pool(k_cache, v_cache, k_scale, v_scale):
    """A 4-bit pool's four tensors, checked."""
    if k_scale is None or v_scale is None:
        raise ValueError("a 4-bit KV pool needs k_scale/v_scale")
    if k_cache.ndim != 4 or k_cache.size(3) != ROW_BYTES or v_cache.shape != k_cache.shape:
        raise ValueError("expected 4-bit kv=[pages,page,kv_heads,64]")
    if any(t.dtype != torch.uint8 for t in (k_cache, v_cache, k_scale, v_scale)):
        raise ValueError("a 4-bit pool's codes and scales are uint8")
    want = k_cache.shape[:3] + (POWERS,)
    if k_scale.shape != want or v_scale.shape != want:
        raise ValueError(f"4-bit scales must be {list(want)}")
    if not all(t.is_contiguous() for t in (k_cache, v_cache, k_scale, v_scale)):
        raise AssertionError("KV pools and their scales must be contiguous")
    if len({t.device for t in (k_cache, v_cache, k_scale, v_scale)}) != 1:
        raise ValueError("a pool's codes and scales must be on one device")


def _one_device(pool, **tensors):
    for name, t in tensors.items():
        if t.device != pool.device:
            raise ValueError(f"{name} must be on the pool's device")


def _append_rows(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping):
    """An append's arguments, checked: its slots and their bytes."""
    check_fp4_pool(k_cache, v_cache, k_scale, v_scale)
    if key.ndim != 3 or value.shape != key.shape or key.shape[1:] != (k_cache.size(2), 128):
        raise ValueError("expected key/value=[tokens,kv_heads,128]")
    _check_rows(key, value)
    assert slot_mapping.numel() == key.size(0)
    _one_device(k_cache, key=key, value=value, slot_mapping=slot_mapping)
    nat.require_device(k_cache)
    return _slots(slot_mapping)


def store_kvcache_fp4(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping):
    """store_kvcache into a 4-bit pool: key / value [N, KVH, 128] bf16 rows
    quantised at slot_mapping (int32 or int64 [N]; a negative slot counts from
    the pool's end, one outside the pool is skipped).  One launch, capturable.
    Two tokens of a call at one slot leave a mixture of both there."""
    if nat.is_current(key) and nat.host().fp4_store(key, value, k_cache, v_cache, k_scale,
                                                    v_scale, slot_mapping, nat.stream_of(key)):
        return
    slots, sb = _append_rows(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
    nat.call_on(
        k_cache, "kvc_store_fp4", key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(),
        value.stride(0), value.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
        k_scale.data_ptr(), v_scale.data_ptr(), k_cache.size(0) * k_cache.size(1),
        slots.data_ptr(), sb, key.size(0), key.size(1), 128, nat.stream_of(k_cache))


def dequant_fp4(codes, scale):
    """codes [..., 64] and scale [..., 4] uint8 -> bf16 [..., 128]."""
    if codes.dtype != torch.uint8 or scale.dtype != torch.uint8 or codes.ndim < 1 \
            or codes.size(-1) != ROW_BYTES or scale.shape != codes.shape[:-1] + (POWERS,):
        raise ValueError("expected codes=[...,64] and scale=[...,4] uint8")
    if scale.device != codes.device:
        raise ValueError("codes and scale must be on one device")
    nat.require_device(codes)
    codes, scale = codes.contiguous(), scale.contiguous()
    if codes.data_ptr() % 4:
        codes = codes.clone()
    out = torch.empty(codes.shape[:-1] + (128,), dtype=torch.bfloat16, device=codes.device)
    if out.numel():
        nat.call_on(codes, "kvc_dequant_fp4", codes.data_ptr(), scale.data_ptr(),
                    out.numel() // 128, 128, out.data_ptr(), nat.stream_of(codes))
    return out


def gather_kv_fp4(k_cache, v_cache, k_scale, v_scale, block_tables, cu_seqlens_k,
                  cu_seqlens_k_list, row0=0):
    """gather_kv over a 4-bit pool."""
    num_prefill, total = len(cu_seqlens_k_list) - 1, cu_seqlens_k_list[-1]
    if nat.is_current(k_cache):
        done = nat.host().fp4_gather(k_cache, v_cache, k_scale, v_scale, block_tables,
                                     cu_seqlens_k, row0, num_prefill, total,
                                     nat.stream_of(k_cache))
        if done is not None:
            return done
    check_fp4_pool(k_cache, v_cache, k_scale, v_scale)
    _one_device(k_cache, block_tables=block_tables, cu_seqlens_k=cu_seqlens_k)
    if block_tables.size(0) < row0 + num_prefill:
        raise ValueError("block_tables has fewer rows than the call has sequences")
    if cu_seqlens_k.numel() < num_prefill + 1:
        raise ValueError("cu_seqlens_k has fewer entries than its list")
    nat.require_device(k_cache)
    block_tables = block_tables.to(torch.int32)
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    cu_seqlens_k = cu_seqlens_k.to(torch.int32).contiguous()
    out_k = torch.empty((total, k_cache.size(2), 128), dtype=torch.bfloat16,
                        device=k_cache.device)
    out_v = torch.empty_like(out_k)
    if total:
        nat.call_on(
            k_cache, "kvc_gather_kv_fp4", k_cache.data_ptr(), v_cache.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), k_cache.size(0), k_cache.size(1),
            k_cache.size(2), 128, block_tables.data_ptr(), block_tables.stride(0),
            block_tables.size(1), row0, num_prefill, cu_seqlens_k.data_ptr(), total,
            out_k.data_ptr(), out_v.data_ptr(), nat.stream_of(k_cache))
    return out_k, out_v


def _rows16(t):
    return (t.stride(2) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0
            and t.data_ptr() % 16 == 0)


def _decode_rows(q, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, out):
    """A decode call's arguments, checked and in the library's form: q, block_tables,
    context_lens, out, the bytes of its workspace."""
    check_fp4_pool(k_cache, v_cache, k_scale, v_scale)
    if q.ndim != 3:
        raise ValueError("expected q=[batch,heads,dim], kv=[pages,page,kv_heads,64]")
    batch, num_heads, head_dim = q.shape
    page_size, num_kv_heads = k_cache.size(1), k_cache.size(2)
    if head_dim != 128 or page_size % 32 or page_size == 0 or num_kv_heads == 0 \
            or num_heads % num_kv_heads:
        raise ValueError(
            "paged decode requires head_dim=128, page_size a multiple of 32 and "
            "GQA-divisible heads")
    if q.dtype != torch.bfloat16:
        raise ValueError(f"q must be bf16 (got {q.dtype})")
    _one_device(k_cache, q=q, block_tables=block_tables, context_lens=context_lens)
    if block_tables.ndim != 2 or block_tables.size(0) < batch or context_lens.numel() != batch:
        raise ValueError("expected block_tables=[batch,pages] and context_lens=[batch]")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype
                            or out.device != q.device or not _rows16(out)):
        raise ValueError("out must be bf16 [batch,heads,128] on q's device, its rows 16-byte "
                         "aligned")
    nat.require_device(k_cache)
    if not _rows16(q):
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
    if block_tables.dtype != torch.int32:
        block_tables = block_tables.to(torch.int32)
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    if context_lens.dtype != torch.int32 or not context_lens.is_contiguous():
        context_lens = context_lens.to(torch.int32).contiguous()
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    need = nat.query("kvc_paged_decode_fp4_workspace_bytes", batch, num_heads, num_kv_heads,
                     page_size, block_tables.size(1))
    return q, block_tables, context_lens, out, need


def paged_decode_fp4(q, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, scale,
                     out=None):
    """paged_decode_attention over a 4-bit pool, written to `out` if given.  A
    row with context_lens[b] <= 0 gives zeros."""
    if nat.is_current(q):
        done = nat.host().fp4_rows(out, q, k_cache, v_cache, k_scale, v_scale, block_tables,
                                   q.size(0) if q.ndim else 0, context_lens, None, None, None,
                                   None, scale, nat.stream_of(q), None, None, None)
        if done is not None:
            return done
    q, block_tables, context_lens, out, need = _decode_rows(
        q, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, out)
    if q.size(0) == 0:
        return out
    ws = nat.workspace(need, q.device)
    nat.call_on(
        k_cache, "kvc_paged_decode_fp4", q.data_ptr(), q.stride(0), q.stride(1),
        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
        k_cache.size(0), k_cache.size(1), k_cache.size(2), 128, block_tables.data_ptr(),
        block_tables.stride(0), block_tables.size(1), context_lens.data_ptr(), q.size(0),
        q.size(1), float(scale), out.data_ptr(), out.stride(0), out.stride(1), nat.ptr(ws), need,
        nat.stream_of(q))
    return out


def varlen_fp4(q, k_cache, v_cache, k_scale, v_scale, block_tables, num_decode_rows,
               decode_context_lens, chunk_blocks, cu_seqlens_q, cu_seqlens_k, scale, out,
               num_prefill=None):
    """varlen_attention's rows over a 4-bit pool read as it is
    (kvc_varlen_fp4), into out; arguments as varlen_attention checked and
    converted them, int32 offsets on q's device.  num_prefill: the chunks, whose
    offsets come first in tensors that may be longer (by default all of
    cu_seqlens_q)."""
    if num_prefill is None:
        num_prefill = cu_seqlens_q.numel() - 1
    if min(cu_seqlens_q.numel(), cu_seqlens_k.numel()) < num_prefill + 1:
        raise ValueError("cu_seqlens_q / cu_seqlens_k have fewer entries than the call has chunks")
    if num_decode_rows and decode_context_lens.numel() < num_decode_rows:
        raise ValueError("decode_context_lens has fewer entries than the call has decode rows")
    _one_device(k_cache, q=q, block_tables=block_tables, cu_seqlens_q=cu_seqlens_q,
                cu_seqlens_k=cu_seqlens_k)
    if num_decode_rows:
        _one_device(k_cache, decode_context_lens=decode_context_lens)
    if block_tables.size(0) < num_decode_rows + num_prefill:
        raise ValueError("block_tables has fewer rows than the call has sequences")
    if not _rows16(q):
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
    tokens, num_heads, _ = q.shape
    page_size, kvh, max_blocks = k_cache.size(1), k_cache.size(2), block_tables.size(1)
    need = nat.query("kvc_varlen_fp4_workspace_bytes", tokens, num_heads, kvh, page_size,
                     max_blocks, num_decode_rows, num_prefill, chunk_blocks)
    ws = nat.workspace(need, q.device)
    nat.call_on(
        k_cache, "kvc_varlen_fp4", q.data_ptr(), q.stride(0), q.stride(1), tokens, num_heads,
        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
        k_cache.size(0), page_size, kvh, 128, block_tables.data_ptr(), block_tables.stride(0),
        max_blocks, num_decode_rows,
        decode_context_lens.data_ptr() if num_decode_rows else None, num_prefill, chunk_blocks,
        cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), float(scale), out.data_ptr(),
        out.stride(0), out.stride(1), nat.ptr(ws), need, nat.stream_of(q))
    return out


def paged_decode_append_fp4(q, key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping,
                            block_tables, context_lens, scale, out=None):
    """The decode step over a 4-bit pool: store_kvcache_fp4 of the new tokens,
    then paged_decode_fp4 over context_lens (which count them).  A call that is
    refused stores nothing."""
    if nat.is_current(q):
        done = nat.host().fp4_rows(out, q, k_cache, v_cache, k_scale, v_scale, block_tables,
                                   q.size(0) if q.ndim else 0, context_lens, None, None, None,
                                   None, scale, nat.stream_of(q), key, value, slot_mapping)
        if done is not None:
            return done
    q, block_tables, context_lens, out, need = _decode_rows(
        q, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, out)
    slots, sb = _append_rows(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
    ws = nat.workspace(need, q.device)
    nat.call_on(
        k_cache, "kvc_paged_decode_append_fp4", q.data_ptr(), q.stride(0), q.stride(1),
        key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0),
        value.stride(1), slots.data_ptr(), sb, key.size(0), k_cache.data_ptr(),
        v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k_cache.size(0),
        k_cache.size(1), k_cache.size(2), 128, block_tables.data_ptr(), block_tables.stride(0),
        block_tables.size(1), context_lens.data_ptr(), q.size(0), q.size(1), float(scale),
        out.data_ptr(), out.stride(0), out.stride(1), nat.ptr(ws), need, nat.stream_of(q))
    return out
