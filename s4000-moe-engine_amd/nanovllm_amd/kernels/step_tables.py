"""A serving step's tables from its requests' lengths, built on the GPU (libkvc
`kvc_step_tables`).

The engine builds slots, positions, offsets and block tables on the host, token
by token, from its block manager's lists (nanovllm/engine/model_runner.py:
579-699), and uploads them.  That is what a step needs whose lengths the host
knows.  Where they are known on the device alone (how much of a drafted tree was
accepted, a step captured in a graph that goes on without the host), one call
here allocates the pages and writes the tables there, with no host read.
engine/device_tables.py holds the state between steps.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _native as nat

NO_SLOT = 2 ** 31 - 1  # outside every pool: an append skips it


@dataclass(slots=True)
class StepTables:
    """What a step's kernels read, all on the device.  Fields as in Context where
    they meet one: context_lens of a decode step is seq_lens here."""
    slot_mapping: torch.Tensor   # int32 [max_tokens]
    positions: torch.Tensor      # int64 [max_tokens]
    query_lens: torch.Tensor     # int32 [batch]: tokens granted
    seq_lens: torch.Tensor       # int32 [batch]: keys the step attends, 0 for a waiting row
    context_lens: torch.Tensor   # int32 [batch]: tokens held after the step
    cu_seqlens_q: torch.Tensor   # int32 [batch + 1]
    cu_seqlens_k: torch.Tensor   # int32 [batch + 1]
    num_blocks: torch.Tensor     # int32 [batch]: pages held
    num_free: torch.Tensor       # int32 [1]


def _vector(t, n, what, device):
    if t.dtype != torch.int32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be int32 [{n}], contiguous")
    if t.device != device:
        raise ValueError(f"{what} must be on the tables' device")


def new_step_tables(batch, max_tokens, device) -> StepTables:
    """Outputs for build_step_tables(out=), for steps that keep their places."""
    def i32(n):
        return torch.empty(n, dtype=torch.int32, device=device)

    return StepTables(i32(max_tokens), torch.empty(max_tokens, dtype=torch.int64, device=device),
                      i32(batch), i32(batch), i32(batch), i32(batch + 1), i32(batch + 1),
                      i32(batch), i32(1))


def build_step_tables(context_lens, query_lens, block_tables, num_blocks, free_blocks, num_free,
                      page_size, max_tokens, *, tokens_per_row=0, finished=None,
                      pad_slot=NO_SLOT, out=None, clear_ended=False) -> StepTables:
    """Row b of block_tables (int32 [batch, width], changed in place) holds
    num_blocks[b] pages for context_lens[b] tokens and asks for query_lens[b]
    new ones; free_blocks (int32, changed in place) is a stack of num_free[0]
    free pages.  All int32 on one device, read there.

    Rows with finished[b] (bool or uint8) first give their pages back and are
    empty from then on: a request that ended, or whose row a new one takes.
    Then the rows are served in order: one gets its tokens if its table row is
    wide enough, if the pages needed up to it are there (or it needs none), and
    if the tokens wanted up to it fit into max_tokens.  Others wait: no tokens,
    no pages, their state as it was.  Pages come from the top of the stack.

    Tokens are packed in row order (with cu_seqlens_q), or, with tokens_per_row,
    row b's begin at b * tokens_per_row (max_tokens is then batch *
    tokens_per_row); entries without a token hold pad_slot and position 0.  out:
    a StepTables to write; its num_blocks, num_free, context_lens and query_lens
    may be the given ones.

    clear_ended: set the given context_lens of finished rows to 0 (for lengths that
    are kept while out.context_lens is another tensor; refused where it is the same)."""
    if out is None and not clear_ended and nat.is_current(block_tables):
        done = nat.host().step_tables(context_lens, query_lens, block_tables, num_blocks,
                                      free_blocks, num_free, page_size, max_tokens,
                                      tokens_per_row, finished, pad_slot,
                                      nat.stream_of(block_tables))
        if done is not None:
            return StepTables(*done)
    if block_tables.ndim != 2 or block_tables.dtype != torch.int32 \
            or (block_tables.size(1) > 1 and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be int32 [batch, pages] with dense rows")
    batch, width = block_tables.shape
    if batch > 1 and width > 0 and block_tables.stride(0) < width:
        raise ValueError("block_tables has overlapping rows")
    dev = block_tables.device
    page_size, max_tokens, tokens_per_row = int(page_size), int(max_tokens), int(tokens_per_row)
    if page_size <= 0:
        raise ValueError(f"page_size must be > 0 (got {page_size})")
    if max_tokens < 0 or tokens_per_row < 0:
        raise ValueError("max_tokens and tokens_per_row must be >= 0")
    if tokens_per_row and max_tokens != batch * tokens_per_row:
        raise ValueError(f"max_tokens must be batch x tokens_per_row ({batch} x {tokens_per_row})")
    if not -2 ** 31 <= pad_slot < 2 ** 31:
        raise ValueError("pad_slot must be an int32")
    _vector(context_lens, batch, "context_lens", dev)
    _vector(query_lens, batch, "query_lens", dev)
    _vector(num_blocks, batch, "num_blocks", dev)
    _vector(num_free, 1, "num_free", dev)
    _vector(free_blocks, free_blocks.numel(), "free_blocks", dev)
    if finished is not None and (finished.dtype not in (torch.bool, torch.uint8)
                                 or finished.numel() != batch or not finished.is_contiguous()
                                 or finished.device != dev):
        raise ValueError(f"finished must be bool [{batch}] on the tables' device")
    if out is not None:
        if out.positions.dtype != torch.int64 or out.positions.numel() != max_tokens \
                or not out.positions.is_contiguous() or out.positions.device != dev:
            raise ValueError(f"out.positions must be int64 [{max_tokens}]")
        for name, n in (("slot_mapping", max_tokens), ("query_lens", batch), ("seq_lens", batch),
                        ("context_lens", batch), ("cu_seqlens_q", batch + 1),
                        ("cu_seqlens_k", batch + 1), ("num_blocks", batch), ("num_free", 1)):
            _vector(getattr(out, name), n, f"out.{name}", dev)
    nat.require_device(block_tables)
    if out is None:
        out = new_step_tables(batch, max_tokens, dev)
    nat.call_on(
        block_tables, "kvc_step_tables_ended", context_lens.data_ptr(), query_lens.data_ptr(),
        nat.ptr(finished), context_lens.data_ptr() if clear_ended else None,
        block_tables.data_ptr(), block_tables.stride(0), width, batch, num_blocks.data_ptr(),
        free_blocks.data_ptr(), free_blocks.numel(), num_free.data_ptr(), page_size, max_tokens,
        tokens_per_row, pad_slot, out.slot_mapping.data_ptr(),
        out.positions.data_ptr(), out.query_lens.data_ptr(), out.seq_lens.data_ptr(),
        out.context_lens.data_ptr(), out.num_blocks.data_ptr(), out.num_free.data_ptr(),
        out.cu_seqlens_q.data_ptr(), out.cu_seqlens_k.data_ptr(), nat.stream_of(block_tables))
    return out
