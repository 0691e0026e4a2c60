"""Block tables, lengths and free pages of a set of requests, held on the GPU.

The engine keeps them on the host (nanovllm/engine/block_manager.py, mirrored in
engine/block_manager.py here) and uploads a step's slots and tables
(model_runner.py:579-699).  DeviceBlockTables is for steps whose lengths are known
on the device alone, or that go on without the host (a captured step replayed with
advancing lengths): `step` hands out pages and writes the step's metadata in one
call (kernels/step_tables.py).  It knows neither shared prefixes nor host offload;
its pages are its own, none that a BlockManager hands out too.
"""
from __future__ import annotations

import torch

from ..kernels.step_tables import NO_SLOT, StepTables, build_step_tables, new_step_tables


class DeviceBlockTables:
    """max_rows rows of up to max_blocks_per_seq pages of page_size tokens, handed
    out from `blocks` (a count, or the block ids themselves, the last on top of
    the stack).  State, all on the device: block_tables [rows, pages],
    context_lens (tokens that a row holds: the caller may lower it, after drafts
    were not accepted, but not while a step reads it), num_blocks (pages held),
    free_blocks and num_free.  pad_slot: where the appends of entries without a
    token go (by default nowhere)."""

    def __init__(self, max_rows: int, max_blocks_per_seq: int, page_size: int, blocks,
                 device="cuda", pad_slot: int = NO_SLOT):
        if max_rows <= 0 or max_blocks_per_seq <= 0 or page_size <= 0:
            raise ValueError("max_rows, max_blocks_per_seq and page_size must be > 0")
        ids = list(range(blocks)) if isinstance(blocks, int) else [int(b) for b in blocks]
        if len(set(ids)) != len(ids) or (ids and min(ids) < 0):
            raise ValueError("blocks must be distinct block ids")
        if ids and (max(ids) + 1) * page_size >= 2 ** 31:
            raise ValueError("slots of these blocks do not fit into int32")
        self.max_rows, self.page_size, self.pad_slot = max_rows, page_size, pad_slot
        self.block_tables = torch.full((max_rows, max_blocks_per_seq), -1, dtype=torch.int32,
                                       device=device)
        self.context_lens = torch.zeros(max_rows, dtype=torch.int32, device=device)
        self.num_blocks = torch.zeros_like(self.context_lens)
        self.free_blocks = torch.tensor(ids, dtype=torch.int32, device=device)
        self.num_free = torch.tensor([len(ids)], dtype=torch.int32, device=device)

    @property
    def device(self) -> torch.device:
        return self.block_tables.device

    def outputs(self, max_tokens: int, advance: bool = True) -> StepTables:
        """Tensors for step(out=): places that a captured step keeps.  The pages
        held and free are the state itself, and so are the lengths with advance;
        without, out.context_lens is a tensor of its own and the state keeps the
        lengths from before the step, 0 for rows that ended (drafted tokens, of
        which the caller adds the accepted ones to context_lens)."""
        out = new_step_tables(self.max_rows, max_tokens, self.device)
        out.num_blocks, out.num_free = self.num_blocks, self.num_free
        if advance:
            out.context_lens = self.context_lens
        return out

    def step(self, query_lens: torch.Tensor, max_tokens: int, *, tokens_per_row: int = 0,
             finished: torch.Tensor | None = None, advance: bool = True,
             out: StepTables | None = None) -> StepTables:
        """One step: rows that `finished` marks give their pages back and start
        empty, then every row takes pages for its query_lens new tokens if they
        are there (build_step_tables has the rules).  out: from outputs(), with
        the same max_tokens and advance."""
        if out is None:
            out = self.outputs(max_tokens, advance)
        elif (out.num_blocks is not self.num_blocks or out.num_free is not self.num_free
              or (out.context_lens is self.context_lens) != advance):
            raise ValueError("out must come from this object's outputs(), with the same advance")
        return build_step_tables(
            self.context_lens, query_lens, self.block_tables, self.num_blocks, self.free_blocks,
            self.num_free, self.page_size, max_tokens, tokens_per_row=tokens_per_row,
            finished=finished, pad_slot=self.pad_slot, out=out,
            clear_ended=finished is not None and not advance)
