"""Pages of the key/value cache handed out on the device.

A ``KVPool`` keeps what a scheduler keeps on the host otherwise: the block table
and lengths of a fixed number of sequences and who holds which page.  A step's
new tokens get their pages (``kv_assign``), rejected or ended ones give theirs back
(``kv_trim``), a beam search's sequences go on from their parents (``kv_reorder``)
and share their pages until they are written (``kv_copy``), and the rows of a batch get
their positions and slots (``kv_slots``).  Nothing is read back, so all of it can
stand in a captured step.  No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass, field

import torch

from .. import _native
from .kv_cache import MAX_LENGTH, PAGE_SIZES, KVBatch, KVCache, _device_ints


@dataclass(frozen=True)
class KVPool:
    """The pages of any number of caches that have as many and as large ones (a
    model's layers), and the sequences that hold them.

    ``table``: int32 ``[sequences, width]``, each sequence's pages, -1 past them;
    ``lengths``: int32 ``[sequences]``; ``refs``: int32 ``[blocks]``, how many sequences
    hold a page; ``free``: uint8, 1 for a page that nobody holds.  Calls on a pool
    change it in their order, so they belong on one stream (or behind its events).  Autograd
    is not told of these changes, nor of a step's: what it is to keep is cloned first."""

    table: torch.Tensor
    lengths: torch.Tensor
    refs: torch.Tensor
    free: torch.Tensor
    blocks: int
    block_size: int
    sequences: int
    width: int
    device: torch.device
    _scratch: torch.Tensor = field(repr=False, compare=False, default=None)
    _struct: object = field(repr=False, compare=False, default=None)
    _ref: int = field(repr=False, compare=False, default=0)


@dataclass(frozen=True)
class KVStep:
    """What ``kv_assign`` writes and the calls of a step read: ``batch`` (its
    lengths are ``lengths``, zero for a sequence without new tokens), ``copies``
    int32 ``[sequences, 3]`` (page, the page it is copied to, tokens; -1, -1, 0: none)
    and ``missing`` int32 ``[1]``: 0, the pages that the pool lacked, -1 where a
    sequence would have passed its row of the table or ``max_length``, -2 where the
    new tokens were more than ``rows``."""

    batch: KVBatch
    lengths: torch.Tensor
    starts: torch.Tensor | None
    copies: torch.Tensor
    missing: torch.Tensor
    pool: KVPool = field(repr=False, compare=False)
    _struct: object = field(repr=False, compare=False, default=None)
    _ref: int = field(repr=False, compare=False, default=0)


class KVPoolOps:
    """The pool's entry points, part of ``HipRNSBackend``."""

    def create_kv_pool(self, *, device: torch.device, blocks: int, block_size: int, sequences: int, width: int) -> KVPool:
        """An empty pool of ``blocks`` pages of ``block_size`` tokens (16, 32, 64 or
        128) for ``sequences`` sequences of up to ``width`` pages."""
        if block_size not in PAGE_SIZES:
            raise ValueError(f"block_size must be one of {PAGE_SIZES}")
        blocks, sequences, width = int(blocks), int(sequences), int(width)
        if blocks < 1 or sequences < 1 or width < 1:
            raise ValueError("a pool has at least one page, one sequence and one column")
        if blocks > 2 ** 31 - 1 or sequences > 2 ** 31 - 1 or width * block_size > MAX_LENGTH:
            raise ValueError(f"a pool has less than 2**31 pages and sequences, of up to {MAX_LENGTH} tokens")
        table = torch.full((sequences, width), -1, dtype=torch.int32, device=device)
        lengths = torch.zeros((sequences,), dtype=torch.int32, device=device)
        refs = torch.zeros((blocks,), dtype=torch.int32, device=device)
        free = torch.ones((-(-blocks // 16) * 16,), dtype=torch.uint8, device=device)
        free[blocks:] = 0
        scratch = torch.zeros((int(self._lib.rnsmx_kv_pool_scratch_words(blocks, sequences, width)),), dtype=torch.int32,
                              device=device)
        scratch[blocks:2 * blocks] = 2 ** 31 - 1
        struct = _native.KVPoolStruct(table.data_ptr(), lengths.data_ptr(), refs.data_ptr(), free.data_ptr(), scratch.data_ptr(),
                                      blocks, int(block_size), sequences, width)
        return KVPool(table, lengths, refs, free, blocks, int(block_size), sequences, width, refs.device, scratch, struct,
                      ctypes.addressof(struct))

    def kv_step(self, pool: KVPool, *, rows: int | None = None, max_query: int | None = None,
                max_length: int | None = None) -> KVStep:
        """The buffers of a step, for any number of steps.  ``rows``: most new
        tokens of all sequences, ``max_query``: most of one (default: ``rows``); their
        rows lie one sequence behind the other.  Without ``rows`` every sequence
        has a row of its own, for at most one new token.  ``max_length`` as in ``kv_batch``."""
        lengths = torch.zeros((pool.sequences,), dtype=torch.int32, device=pool.device)
        copies = torch.tensor((-1, -1, 0), dtype=torch.int32, device=pool.device).repeat(pool.sequences, 1)
        missing = torch.zeros((1,), dtype=torch.int32, device=pool.device)
        if rows is None:
            if max_query not in (None, 1):
                raise ValueError("max_query goes with rows")
            starts = None
            batch = self.kv_batch(pool, pool.table, lengths, max_length=max_length)
        else:
            starts = torch.zeros((pool.sequences + 1,), dtype=torch.int32, device=pool.device)
            batch = self.kv_batch(pool, pool.table, lengths, query_starts=starts, rows=int(rows),
                                  max_query=int(rows if max_query is None else max_query), max_length=max_length)
        struct = _native.KVStepStruct(lengths.data_ptr(), None if starts is None else starts.data_ptr(), copies.data_ptr(),
                                      missing.data_ptr(), batch.rows, batch.max_query, batch.max_length)
        return KVStep(batch, lengths, starts, copies, missing, pool, struct, ctypes.addressof(struct))

    @staticmethod
    def _pool_numbers(pool: KVPool, values: torch.Tensor, name: str) -> int:
        """Numbers of all sequences on the device: their address."""
        if _device_ints(values, name, 1, pool.device).shape[0] != pool.sequences:
            raise ValueError(f"{name} must have {pool.sequences} elements")
        if pool.device.type != "cuda":
            raise ValueError(f"the pool must be on the GPU, it is on {pool.device}")
        return values.data_ptr()

    def kv_assign(self, pool: KVPool, step: KVStep, new: torch.Tensor | None = None) -> None:
        """Gives the sequences pages for ``new`` tokens each (int32 ``[sequences]``, cut
        to 0 and ``max_query``; None: one each), adds them to ``pool.lengths`` and
        fills ``step``, in one launch, or two where the step's rows could need more than 4096
        pages (so a step of few tokens has its own ``kv_step``).

        Pages are the lowest that nobody holds, in the order of the sequences.  A
        partly filled page that others hold too is replaced by a page of the sequence's
        own, whose tokens ``kv_copy`` brings over, before anything is appended; where all
        its holders get tokens, the first of them keeps it.  A call that the pool
        lacks pages for, or whose tokens pass a bound, changes nothing: ``step.missing``
        is not zero, and the step's batch has no tokens (nothing is appended, its
        attention is zero)."""
        if step.pool is not pool:
            raise ValueError("the step is of another pool")
        at = None if new is None else self._pool_numbers(pool, new, "new")
        if pool.device.type != "cuda":
            raise ValueError(f"the pool must be on the GPU, it is on {pool.device}")
        self._on_device(pool.device, self._lib.rnsmx_kv_assign, pool._ref, step._ref, at)
        self._stats["kv_assign_calls"] += 1

    def kv_trim(self, pool: KVPool, lengths: torch.Tensor) -> None:
        """Cuts every sequence to ``lengths`` tokens (int32 ``[sequences]``; one that has
        no more stays, 0 ends it) and lets go of the pages past them, in one launch."""
        self._on_device(pool.device, self._lib.rnsmx_kv_trim, pool._ref, self._pool_numbers(pool, lengths, "lengths"))
        self._stats["kv_trim_calls"] += 1

    def kv_reorder(self, pool: KVPool, parents: torch.Tensor) -> None:
        """Every sequence becomes what sequence ``parents[s]`` (int32 ``[sequences]``) was
        before the call and holds its pages too; empty where that is no sequence's
        number, -1 say.  The caches are not touched."""
        self._on_device(pool.device, self._lib.rnsmx_kv_reorder, pool._ref, self._pool_numbers(pool, parents, "parents"))
        self._stats["kv_reorder_calls"] += 1

    def kv_copy(self, cache: KVCache, step: KVStep) -> None:
        """Brings the tokens of ``step.copies`` to their new pages, keys, values and
        scales of all heads, in one launch: once for each cache, between ``kv_assign`` and the
        first ``kv_append`` of the step."""
        pool = step.pool
        if cache.device != pool.device or cache.block_size != pool.block_size or cache.blocks < pool.blocks:
            raise ValueError(f"the cache must have {pool.blocks} pages of {pool.block_size} tokens on {pool.device}")
        if cache.device.type != "cuda":
            raise ValueError(f"the cache must be on the GPU, it is on {cache.device}")
        self._on_device(cache.device, self._lib.rnsmx_kv_copy, cache._ref, step.copies.data_ptr(), pool.sequences)
        self._stats["kv_copy_calls"] += 1

    def kv_slots(self, pages: KVPool | KVCache, batch: KVBatch) -> tuple[torch.Tensor, torch.Tensor]:
        """Where the rows of a batch lie among ``pages``: their tokens' positions in their
        sequences (int32 ``[rows]``) and slots, page number times ``block_size`` plus
        place in the page (int64 ``[rows]``), in one launch.  A row without a token is at
        position 0; its slot is -1, as is that of a token that the batch drops or
        whose page is not there."""
        key = (pages.blocks, pages.block_size, pages.device)
        like = batch._checked.get(key)
        if like is None:
            if batch.lengths.device != pages.device:
                raise ValueError(f"the batch must be on {pages.device}")
            if pages.device.type != "cuda":
                raise ValueError(f"the pages must be on the GPU, they are on {pages.device}")
            if batch.max_length > batch.block_table.shape[1] * pages.block_size:
                raise ValueError("the batch is of larger pages")
            # one number's memory in the outputs' shape: what they are made like costs less than their sizes
            like = batch._remember(key, tuple(torch.empty((1,), dtype=dtype, device=pages.device).expand(batch.rows)
                                              for dtype in (torch.int32, torch.int64)))
        positions = torch.empty_like(like[0], memory_format=torch.contiguous_format)
        slots = torch.empty_like(like[1], memory_format=torch.contiguous_format)
        self._on_device(pages.device, self._lib.rnsmx_kv_slots, batch._ref, pages.blocks, pages.block_size, positions.data_ptr(),
                        slots.data_ptr())
        self._stats["kv_slots_calls"] += 1
        return positions, slots
