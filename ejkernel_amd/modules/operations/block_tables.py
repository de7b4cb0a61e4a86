"""Block tables and slot maps of a paged cache, built on the device from request lengths.

One call is one step of the bookkeeping that a serving loop does before the model runs: it gives the
new tokens of every request the pages they need, says where each token's key and value go, and takes
back the pages of requests that have ended.  Nothing is read on the host, so the step can stand in a
HIP graph in front of ``quantized_cache_update`` and the paged attention operations, which take its
results as they are.  No counterpart in the reference, whose callers build these arrays on the host.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ... import _native
from .quantized_cache import _call, _check_index_arrays, _on_device

__all__ = ["BlockTables", "BuildBlockTables", "build_block_tables"]


class BlockTables(NamedTuple):
    """Results of ``build_block_tables``, int32 tensors on the device of its arguments."""

    query_start_loc: torch.Tensor  #: ``[max_num_seqs + 1]`` prefix sums of the query lengths
    context_lens: torch.Tensor     #: ``[max_num_seqs]`` cached + new tokens; 0 for refused and ended requests
    slot_mapping: torch.Tensor     #: ``[total_tokens]`` ``page * page_size + offset``, -1 for rows without a token that runs
    positions: torch.Tensor        #: ``[total_tokens]`` position in the sequence, -1 as above
    admitted: torch.Tensor         #: ``[max_num_seqs]`` 1 where the request's tokens run (or it idles), 0 where it is refused or has ended
    cached_lens: torch.Tensor      #: ``[max_num_seqs]`` the next step's ``cached_lens``
    free_state: torch.Tensor       #: ``[2]`` the next step's ``free_state``


class BuildBlockTables:
    """Kernel object of ``build_block_tables``."""

    op_id = "build_block_tables"

    _entry = _native.Entry("rpa_block_tables_launch", _native.RpaBlockTablesParams)

    def run(self, query_lens, cached_lens, block_tables, free_pages, free_state, num_seqs, *, page_size: int, total_tokens: int):
        if block_tables.dim() != 2 or 0 in block_tables.shape:
            raise ValueError(f"block_tables must be [max_num_seqs, pages_per_seq], got {tuple(block_tables.shape)}")
        n, pages_per_seq = block_tables.shape
        if not isinstance(num_seqs, torch.Tensor):
            num_seqs = torch.tensor([int(num_seqs)], dtype=torch.int32, device=block_tables.device)
        _check_index_arrays(("query_lens", query_lens, n), ("cached_lens", cached_lens, n), ("free_state", free_state, 2), ("num_seqs", num_seqs, 1))
        if free_pages.dim() != 1 or free_pages.shape[0] == 0:
            raise ValueError(f"free_pages must be a ring of one page at least, got {tuple(free_pages.shape)}")
        if block_tables.dtype != torch.int32 or free_pages.dtype != torch.int32:
            raise ValueError(f"block_tables.dtype={block_tables.dtype} and free_pages.dtype={free_pages.dtype} must be int32")
        if not block_tables.is_contiguous() or not free_pages.is_contiguous():
            raise ValueError("block_tables and free_pages must be contiguous: they are updated in place")
        if not 0 < page_size < 2**31:
            raise ValueError(f"page_size={page_size} must be positive and below 2**31")
        if not 0 <= total_tokens <= 2**30:
            raise ValueError(f"total_tokens={total_tokens} must be from 0 to 2**30")
        index = _on_device("build_block_tables", ("block_tables", block_tables), ("query_lens", query_lens), ("cached_lens", cached_lens),
                           ("free_pages", free_pages), ("free_state", free_state), ("num_seqs", num_seqs))
        query_lens, cached_lens, free_state = query_lens.contiguous(), cached_lens.contiguous(), free_state.contiguous()

        # one allocation: the kernels' scratch, at the allocator's alignment, and a view for each result
        sizes = (4 * n + 4, n + 1, n, total_tokens, total_tokens, n, n, 2)
        memory = torch.empty(sum(sizes), dtype=torch.int32, device=block_tables.device)
        results = torch.unsafe_split_with_sizes(memory, sizes)[1:]  # nothing here is differentiated
        at, places = memory.data_ptr(), []
        for size in sizes:
            places.append(at)
            at += 4 * size
        _call(self._entry, index, query_lens.data_ptr(), cached_lens.data_ptr(), block_tables.data_ptr(), free_pages.data_ptr(), free_state.data_ptr(),
              num_seqs.data_ptr(), *places[1:], places[0], n, pages_per_seq, free_pages.shape[0], page_size, total_tokens, 0)
        return BlockTables._make(results)


_build = BuildBlockTables()


def build_block_tables(query_lens, cached_lens, block_tables, free_pages, free_state, num_seqs, /, *, page_size: int,
                       total_tokens: int) -> BlockTables:
    """One step of a paged cache's bookkeeping, for requests ``s < num_seqs`` in order.

    ``query_lens[s] > 0``: the request has that many new tokens and gets the pages they need beyond the
    ``ceil(cached_lens[s] / page_size)`` it holds, from the front of the ring of free pages.  It is refused
    (nothing taken, slots -1, context 0, ``cached_lens`` as before) if its context would pass
    ``pages_per_seq`` pages, if its tokens end behind ``total_tokens``, or if it needs a page and the needs
    of the requests up to it exceed the free pages; requests that need none run all the same.
    ``query_lens[s] == 0``: the request idles.  ``query_lens[s] < 0``: it has ended, and its pages go back
    to the end of the ring, in the order of its table (pages that requests share are not counted here).

    Args:
        query_lens: ``[max_num_seqs]`` int32.
        cached_lens: ``[max_num_seqs]`` int32, tokens in the cache before this step.
        block_tables: ``[max_num_seqs, pages_per_seq]`` int32, updated in place; entries behind a request's pages
            keep what they hold.
        free_pages: ``[num_free_slots]`` int32, the ring, updated in place; as many places as the pool has pages.
        free_state: ``[2]`` int32, the ring's first free place and how many pages are free.
        num_seqs: ``[1]`` int32 tensor (or int), requests present.
        page_size: tokens per page.
        total_tokens: rows of the flat batch (static; rows behind the last token get slot -1).

    Returns:
        :class:`BlockTables`; ``cached_lens`` and ``free_state`` are new tensors, to be passed to the next step.
    """
    return _build.run(query_lens, cached_lens, block_tables, free_pages, free_state, num_seqs, page_size=page_size,
                      total_tokens=total_tokens)
