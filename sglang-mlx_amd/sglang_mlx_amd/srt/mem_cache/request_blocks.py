"""Block tables of the open requests, kept on the device.

BlockTable (paged_pool.py) builds slots and tables on the host and copies them
whole each step.  RequestBlocks keeps every request's block ids in one device
table; a step copies its request rows, lengths and new block ids (a few words a
sequence, one copy) and ``kernels.build_step_tables`` makes the step's block
tables, slots and positions from them.  The host keeps what it needs to allocate
and free: each request's blocks and token count.

A request only grows: the tokens of a step stay in its context until it is
closed.  Drafted tokens that a verification refuses cannot be taken back here; a
caller that drafts keeps its own tables (``kernels.build_step_tables`` takes any
lengths).
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from .paged_pool import BlockAllocator


@dataclass
class StepTables:
    """One step's tables, as ``kernels`` takes them (int32 device tensors), and
    its longest context and most new tokens of a sequence (at least 1 each)."""

    block_tables: torch.Tensor
    context_lens: torch.Tensor
    query_start_loc: torch.Tensor
    slot_mapping: torch.Tensor
    positions: torch.Tensor
    max_seq_len: int
    max_query_len: int


class RequestBlocks:
    """Up to ``max_requests`` open requests of up to ``max_blocks`` blocks each,
    from ``allocator``."""

    def __init__(self, max_requests: int, max_blocks: int, block_size: int, allocator: BlockAllocator, device):
        if max_requests <= 0 or max_blocks <= 0 or block_size <= 0:
            raise ValueError("max_requests, max_blocks and block_size must be positive")
        self.block_size, self.max_blocks, self.allocator = block_size, max_blocks, allocator
        self.table = torch.full((max_requests, max_blocks), -1, dtype=torch.int32, device=device)
        self._free_rows = list(range(max_requests - 1, -1, -1))
        self._blocks: dict[int, list[int]] = {}
        self._tokens: dict[int, int] = {}

    def open(self, prefix_blocks=()) -> int:
        """A new request's row.  ``prefix_blocks`` (whole blocks that hold its
        first tokens, as BlockRadixCache.match_prefix returns them) are shared."""
        prefix = [int(b) for b in prefix_blocks]
        if len(prefix) > self.max_blocks:
            raise ValueError(f"{len(prefix)} prefix blocks exceed max_blocks={self.max_blocks}")
        if not self._free_rows:
            raise MemoryError("Cannot open another request: every row is in use")
        self.allocator.share(prefix)
        row = self._free_rows.pop()
        self._blocks[row], self._tokens[row] = prefix, len(prefix) * self.block_size
        if prefix:
            self.table[row, :len(prefix)] = torch.tensor(prefix, dtype=torch.int32).to(self.table.device)
        return row

    def close(self, row: int) -> None:
        """Ends a request: its blocks lose its reference, the row is free again."""
        if row not in self._tokens:
            raise ValueError(f"row {row} is not open")
        self.allocator.free(self._blocks.pop(row))
        del self._tokens[row]
        self._free_rows.append(row)

    def blocks(self, row: int) -> list[int]:
        return list(self._blocks[row])

    def num_tokens(self, row: int) -> int:
        return self._tokens[row]

    def step(self, rows, new_tokens, num_seqs: int | None = None, num_tokens: int | None = None) -> StepTables:
        """Adds ``new_tokens[i]`` tokens to request ``rows[i]`` and returns the
        step's tables, the new tokens of all requests end to end.  num_seqs and
        num_tokens pad the batch to fixed sizes (a captured graph's): sequences
        without tokens, slots of -1.  MemoryError (nothing changed) when the
        allocator has too few blocks."""
        from ... import kernels

        rows = [int(r) for r in rows]
        new = [int(n) for n in new_tokens]
        if len(rows) != len(new):
            raise ValueError("rows and new_tokens must have the same length")
        if len(set(rows)) != len(rows):
            raise ValueError("a request can be in a step once")
        for r, n in zip(rows, new):
            if r not in self._tokens:
                raise ValueError(f"row {r} is not open")
            if n < 0:
                raise ValueError("new_tokens must be non-negative")
        bs = self.block_size
        ctx = [self._tokens[r] + n for r, n in zip(rows, new)]
        if any(-(-c // bs) > self.max_blocks for c in ctx):
            raise ValueError(f"a request's context exceeds max_blocks={self.max_blocks}")
        total = sum(new)
        seqs = len(rows) if num_seqs is None else int(num_seqs)
        tokens = total if num_tokens is None else int(num_tokens)
        if seqs < len(rows) or tokens < total:
            raise ValueError("num_seqs and num_tokens must hold the step")
        need = [-(-c // bs) - len(self._blocks[r]) for r, c in zip(rows, ctx)]
        taken = self.allocator.alloc(sum(need))
        try:
            pad = seqs - len(rows)
            words = np.array(rows + [-1] * pad + ctx + [0] * pad + new + [0] * pad + taken, dtype=np.int32)
            dev = torch.from_numpy(words).to(self.table.device)
            lens = dev[seqs:2 * seqs]
            out = kernels.build_step_tables(self.table, dev[:seqs], lens, dev[2 * seqs:3 * seqs], dev[3 * seqs:], bs,
                                            tokens)
        except BaseException:
            self.allocator.free(taken)
            raise
        at = 0
        for r, c, k in zip(rows, ctx, need):
            self._blocks[r].extend(taken[at:at + k])
            self._tokens[r] = c
            at += k
        return StepTables(out[0], lens, out[3], out[1], out[2], max(ctx + [1]), max(new + [1]))
