"""Key/value cache in 8 bits and the attention that reads it.

What follows a fused query/key/value projection: the new tokens' keys and
values are quantised into pages (``kv_append``), their queries attend to the
pages (``kv_attention``), and code that wants plain tensors reads them back
(``kv_read``).  No counterpart in the reference, whose path ends with the
projections; the quantisation is its symmetric one (``rns_linear.py:154-166``)
with a scale for each page of tokens and head instead of one per tensor.
"""
from __future__ import annotations

import ctypes
import math
import operator
from dataclasses import dataclass, field
from typing import Sequence

import torch

from .. import _native

PAGE_SIZES = (16, 32, 64, 128)
MAX_LENGTH = 1 << 30
_MAX_ROWS = 2 ** 31 - 1
_MAX_CHECKED = 64  # shapes a batch remembers; a mask that grows by a column each step brings ever new ones
_FLOAT_CODES = {torch.float32: _native.FLOAT32, torch.float16: _native.FLOAT16,
                torch.bfloat16: _native.BFLOAT16}
_MASK_CODES = {**_FLOAT_CODES, torch.bool: _native.INT8}


@dataclass(frozen=True)
class KVCache:
    """Pages of keys and values, shared by any number of sequences.

    ``k_codes`` and ``v_codes``: uint8 ``[blocks, kv_heads, block_size, row_bytes]``,
    a value's code plus 128 each (``row_bytes`` is the head dimension rounded up
    to one the kernels are built for); ``scales``: float32 ``[blocks, kv_heads,
    2]``, each page's scale for a head's keys and for its values.  A value is
    ``code * scale``, its code in [-127, 127]."""

    k_codes: torch.Tensor
    v_codes: torch.Tensor
    scales: torch.Tensor
    blocks: int
    block_size: int
    kv_heads: int
    head_dim: int
    device: torch.device
    _struct: object = field(repr=False, compare=False, default=None)
    _ref: int = field(repr=False, compare=False, default=0)
    _shape: tuple = field(repr=False, compare=False, default=())  # what checks of arguments depend on

    @property
    def nbytes(self) -> int:
        return self.k_codes.nbytes + self.v_codes.nbytes + self.scales.nbytes


@dataclass(frozen=True)
class KVBatch:
    """The sequences of one call, bound once: ``block_table`` (int32 ``[S,
    W]``, the page of each ``block_size`` tokens; a number that is no page's,
    -1 say, is a page that is not there), ``lengths`` (int32 ``[S]``, tokens of
    each sequence, those of the call among them) and ``query_starts`` (int32
    ``[S + 1]``, the rows of each sequence, its last tokens; None: one row each).

    The tensors are read by the device on each call and may be written in
    between, as a decode loop (or a captured graph) does that advances
    ``lengths``; ``rows``, ``max_query`` and ``max_length`` bound what they may
    hold.  What goes past them is dropped and moves nothing: tokens from
    ``max_length`` on are not there, and a sequence's rows past its first
    ``max_query`` are not appended and zero in outputs (starts are cut to
    ``rows``).  Rows that ``query_starts`` gives to no sequence are not written in
    a call's outputs."""

    block_table: torch.Tensor
    lengths: torch.Tensor
    query_starts: torch.Tensor | None
    rows: int
    max_query: int
    max_length: int
    longest: int | None = None  # of the lengths given as numbers
    _struct: object = field(repr=False, compare=False, default=None)
    _ref: int = field(repr=False, compare=False, default=0)
    # arguments that were checked: their types, shapes and strides -> what a call passes on
    _checked: dict = field(repr=False, compare=False, default_factory=dict)

    @property
    def sequences(self) -> int:
        return int(self.lengths.shape[0])

    def _remember(self, key: tuple, value):
        if len(self._checked) >= _MAX_CHECKED:
            self._checked.clear()
        self._checked[key] = value
        return value


class _WithoutGradient(torch.autograd.Function):
    """An output as it is; a backward pass that reaches it says that it ends there."""

    @staticmethod
    def forward(ctx, out, *inputs):
        return out.view_as(out)

    @staticmethod
    def backward(ctx, *gradients):
        raise RuntimeError("kv_attention has no gradient: detach its queries and mask, or call it under torch.no_grad()")


def _device_ints(values: torch.Tensor, name: str, ndim: int, device: torch.device) -> torch.Tensor:
    if values.dtype != torch.int32 or values.ndim != ndim or values.device != device:
        raise ValueError(f"{name} must be a {ndim}-dimensional int32 tensor on {device}")
    if values.numel() and values.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return values


def _counts(values, name: str) -> list[int]:
    counts = [int(v) for v in values]
    if any(v < 0 for v in counts):
        raise ValueError(f"{name} must not be negative")
    return counts


class KVCacheOps:
    """The cache's entry points, part of ``HipRNSBackend``."""

    def create_kv_cache(self, *, device: torch.device, blocks: int, block_size: int, kv_heads: int,
                        head_dim: int) -> KVCache:
        """An empty cache of ``blocks`` pages of ``block_size`` tokens (16, 32,
        64 or 128) for ``kv_heads`` heads of 1 to 256 values."""
        if block_size not in PAGE_SIZES:
            raise ValueError(f"block_size must be one of {PAGE_SIZES}")
        if blocks < 1 or kv_heads < 1:
            raise ValueError("a cache has at least one page and one head")
        row_bytes = int(self._lib.rnsmx_kv_row_bytes(int(head_dim)))
        if row_bytes < 0:
            raise ValueError(f"head_dim must be 1 to {_native.KV_MAX_DIM}")
        shape = (int(blocks), int(kv_heads), int(block_size), row_bytes)
        k, v = (torch.full(shape, 128, dtype=torch.uint8, device=device) for _ in range(2))
        scales = torch.full(shape[:2] + (2,), torch.finfo(torch.float32).eps, dtype=torch.float32, device=device)
        struct = _native.KVCacheStruct(k.data_ptr(), v.data_ptr(), scales.data_ptr(), shape[0], shape[2], shape[1],
                                       int(head_dim), row_bytes)
        return KVCache(k, v, scales, shape[0], shape[2], shape[1], int(head_dim), scales.device, struct,
                       ctypes.addressof(struct), (shape[1], shape[2], int(head_dim), scales.device))

    def kv_batch(self, cache: KVCache, block_table: torch.Tensor, lengths, *,
                 query_lengths: Sequence[int] | None = None, query_starts: torch.Tensor | None = None,
                 rows: int | None = None, max_query: int | None = None, max_length: int | None = None) -> KVBatch:
        """Binds the sequences of a call.  ``lengths``: int32 device tensor or
        numbers.  The rows of each sequence: ``query_lengths`` as numbers, or
        ``query_starts`` on the device with ``rows`` (their number) and
        ``max_query`` (most of one sequence); neither: one each.
        ``max_length``: most tokens of one sequence while the batch is used (the
        block table's width by default); kernels split work by it."""
        device = cache.device
        table = _device_ints(block_table, "block_table", 2, device)
        width = int(table.shape[1])
        if width < 1:
            raise ValueError("block_table must have at least one column")
        room = width * cache.block_size
        top = min(room, MAX_LENGTH) if max_length is None else int(max_length)
        if not 0 <= top <= min(room, MAX_LENGTH):
            raise ValueError(f"max_length {top} is past the block table's {room} tokens")
        longest = None
        if isinstance(lengths, torch.Tensor):
            lengths = _device_ints(lengths, "lengths", 1, device)
        else:
            numbers = _counts(lengths, "lengths")
            longest = max(numbers, default=0)
            if longest > top:
                raise ValueError(f"a sequence of {longest} tokens is past max_length {top}")
            lengths = torch.tensor(numbers, dtype=torch.int32, device=device)
        seqs = int(lengths.shape[0])
        if int(table.shape[0]) != seqs:
            raise ValueError(f"block_table has {table.shape[0]} rows for {seqs} sequences")
        if query_starts is None and (rows is not None or max_query is not None):
            raise ValueError("rows and max_query go with query_starts")
        if query_lengths is not None:
            if query_starts is not None:
                raise ValueError("rows are given by query_lengths or by query_starts, not both")
            counts = _counts(query_lengths, "query_lengths")
            if len(counts) != seqs:
                raise ValueError(f"{len(counts)} query_lengths for {seqs} sequences")
            starts = [0]
            for n in counts:
                starts.append(starts[-1] + n)
            rows, max_query = starts[-1], max(counts, default=0)
            if rows <= _MAX_ROWS and (max_query != 1 or rows != seqs):
                query_starts = torch.tensor(starts, dtype=torch.int32, device=device)
        elif query_starts is not None:
            query_starts = _device_ints(query_starts, "query_starts", 1, device)
            if rows is None or max_query is None or rows < 0 or max_query < 0:
                raise ValueError("query_starts needs rows and max_query")
            if int(query_starts.shape[0]) != seqs + 1:
                raise ValueError(f"query_starts must have {seqs + 1} elements")
        else:
            rows, max_query = seqs, 1
        if rows > _MAX_ROWS:
            raise ValueError("too many rows")
        max_query = min(max_query, rows)
        struct = _native.KVBatchStruct(table.data_ptr(), table.stride(0), lengths.data_ptr(),
                                       None if query_starts is None else query_starts.data_ptr(),
                                       seqs, width, int(rows), int(max_query), top)
        return KVBatch(table, lengths, query_starts, int(rows), int(max_query), top, longest, struct,
                       ctypes.addressof(struct))

    @staticmethod
    def _check_rows(x: torch.Tensor, name: str, batch: KVBatch, heads: int | None, cache: KVCache) -> torch.Tensor:
        if x.dtype not in _FLOAT_CODES:
            raise ValueError(f"{name} must be float32, float16 or bfloat16")
        if x.device != cache.device or batch.lengths.device != cache.device:
            raise ValueError(f"{name} and the batch must be on {cache.device}")
        shape = x.shape
        if len(shape) != 3 or shape[0] != batch.rows or shape[2] != cache.head_dim or (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} must be [{batch.rows}, {'heads' if heads is None else heads}, {cache.head_dim}], "
                             f"got {tuple(shape)}")
        return x if x.stride(2) == 1 or shape[2] == 1 else x.contiguous()

    @staticmethod
    def _check_gpu(cache: KVCache) -> None:
        """A cache may be made and bound on the host, but a kernel reads none there."""
        if cache.device.type != "cuda":
            raise ValueError(f"the cache must be on the GPU, it is on {cache.device}")

    def kv_append(self, cache: KVCache, batch: KVBatch, k: torch.Tensor, v: torch.Tensor) -> None:
        """Quantises the batch's rows, ``k`` and ``v`` ``[rows, kv_heads,
        head_dim]`` of any strides, into the cache, in one launch.

        For each page and head written: ``scale = max(max|x| * fl32(1/127),
        2**-23)`` over its new tokens, ``code = clamp(round(x / scale), ±127)``,
        in float32.  A page that held tokens of the sequence before keeps the
        larger of its scale and the new tokens'; where that is larger than its
        own, its older codes are quantised again from the values they stood for;
        a token that is taken back leaves its page's scale as it made it.
        A value that is not finite makes every value of its page and head read
        as NaN.  Sequences of one call must not share pages that it writes to.  No
        gradient goes through the cache."""
        key = (k.dtype, k.shape, k.stride(), k.device, v.dtype, v.shape, v.stride(), v.device, cache._shape)
        args = batch._checked.get(key)
        if args is None:
            plain_k = self._check_rows(k, "k", batch, cache.kv_heads, cache)
            plain_v = self._check_rows(v, "v", batch, cache.kv_heads, cache)
            if k.dtype != v.dtype:
                raise ValueError("k and v must have one dtype")
            if plain_k is not k or plain_v is not v:
                return self.kv_append(cache, batch, plain_k, plain_v)
            self._check_gpu(cache)
            args = batch._remember(key, (_FLOAT_CODES[k.dtype], k.stride(0), k.stride(1), v.stride(0), v.stride(1)))
        rc = self._lib.rnsmx_kv_append(cache._ref, batch._ref, k.data_ptr(), v.data_ptr(), *args,
                                       self._stream_of(cache.device))
        if rc:
            _native.check(rc)
        self._stats["kv_append_calls"] += 1

    def kv_read(self, cache: KVCache, batch: KVBatch, *, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values of the batch's rows, ``code * scale`` rounded to
        ``dtype``: two ``[rows, kv_heads, head_dim]`` tensors, in one launch.
        Rows that have no token, and those in pages that are not there, are zero."""
        key = (dtype, cache._shape)
        like = batch._checked.get(key)
        if like is None:
            if dtype not in _FLOAT_CODES:
                raise ValueError("dtype must be float32, float16 or bfloat16")
            if batch.lengths.device != cache.device:
                raise ValueError(f"the batch must be on {cache.device}")
            self._check_gpu(cache)
            # one value's memory in the outputs' shape: what they are made like costs less than their sizes
            like = torch.empty((1,), dtype=dtype, device=cache.device).expand(batch.rows, cache.kv_heads, cache.head_dim)
            batch._remember(key, like)
        k = torch.empty_like(like, memory_format=torch.contiguous_format)
        v = torch.empty_like(like, memory_format=torch.contiguous_format)
        rc = self._lib.rnsmx_kv_read(cache._ref, batch._ref, k.data_ptr(), v.data_ptr(), _FLOAT_CODES[dtype],
                                     self._stream_of(cache.device))
        if rc:
            _native.check(rc)
        self._stats["kv_read_calls"] += 1
        return k, v

    def kv_attention(self, q: torch.Tensor, cache: KVCache, batch: KVBatch, *, scale: float | None = None,
                     causal: bool = True, window: int | None = None, mask: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the batch's rows ``q`` ``[rows, q_heads, head_dim]`` (any
        strides; ``q_heads`` a multiple of the cache's heads) over their
        sequences' cached tokens: ``softmax(scale * q . k + mask) . v``, scale
        ``head_dim ** -0.5`` by default, -> ``[rows, q_heads, head_dim]`` of q's dtype.

        A row sees the tokens up to its own (``causal``), the last ``window`` of
        them if given, or its whole sequence.  ``mask``: ``[rows, q_heads, T]`` or
        broadcast to it, bool (False hides) or float (added; minus infinity
        hides); tokens from T on are hidden, and T covers the lengths given as
        numbers.  What is hidden contributes nothing whatever it holds, and a row
        that sees no token is zero.  ``workspace``: zero-initialised uint8 of
        ``kv_attention_workspace_bytes``, by default one kept per stream (under
        graph capture one of the graph's, cleared by each replay).

        There is no gradient: where queries or mask require one, a backward pass
        through the result raises (a given ``out`` holds numbers alone)."""
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous()):
            raise ValueError("out must be contiguous and like q")
        scale = None if scale is None else float(scale)
        window = None if window is None else operator.index(window)
        key = (q.dtype, q.shape, q.stride(), q.device, cache._shape, scale, bool(causal), window,
               None if mask is None else (mask.dtype, mask.shape, mask.stride(), mask.device))
        checked = batch._checked.get(key)
        if checked is None:
            plain = self._check_rows(q, "q", batch, None, cache)
            if plain is not q:
                return self.kv_attention(plain, cache, batch, scale=scale, causal=causal, window=window, mask=mask,
                                         out=out, workspace=workspace)
            query = self._query_of(q, cache, batch, scale, causal, window, mask)
            self._check_gpu(cache)
            need = int(self._lib.rnsmx_kv_attention_workspace_bytes(cache._ref, batch._ref, ctypes.addressof(query)))
            checked = batch._remember(key, (query, ctypes.addressof(query), need))
        _, ref, need = checked
        wanted = out is None and (q.requires_grad or mask is not None and mask.requires_grad) and torch.is_grad_enabled()
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        stream = self._stream_of(cache.device)
        space, size = None, 0
        if workspace is not None:
            if workspace.dtype != torch.uint8 or workspace.device != cache.device or not workspace.is_contiguous():
                raise ValueError(f"workspace must be contiguous uint8 on {cache.device}")
            space, size = workspace.data_ptr(), workspace.numel()
        elif need > 0:
            scratch = self._kv_scratch_for(need, cache.device, stream)
            space, size = scratch.data_ptr(), scratch.numel()
        # a mask without columns has no address, and hides everything all the same
        hides = None if mask is None else mask.data_ptr() or cache.scales.data_ptr()
        rc = self._lib.rnsmx_kv_attention(cache._ref, batch._ref, ref, q.data_ptr(), hides, space, size, out.data_ptr(),
                                          stream)
        if rc:
            _native.check(rc)
        self._stats["kv_attention_calls"] += 1
        return _WithoutGradient.apply(out, q, mask) if wanted else out

    def _query_of(self, q: torch.Tensor, cache: KVCache, batch: KVBatch, scale, causal, window, mask):
        """The checked arguments of ``kv_attention`` as the library takes them."""
        heads = int(q.shape[1])
        if heads < 1 or heads % cache.kv_heads:
            raise ValueError(f"q has {heads} heads, not a multiple of the cache's {cache.kv_heads}")
        if scale is None:
            scale = 1.0 / math.sqrt(cache.head_dim)
        elif not (scale > 0 and math.isfinite(scale)):
            raise ValueError("scale must be positive and finite")
        if window is None:
            window = 0
        elif window < 1 or not causal:
            raise ValueError("window must be at least 1, of causal rows")
        mask_args, mask_code, mask_len = (0, 0, 0), _native.INT8, 0
        if mask is not None:
            self._check_mask(mask, batch, heads, cache)
            mask_len, mask_code = int(mask.shape[2]), _MASK_CODES[mask.dtype]
            mask_args = mask.expand(batch.rows, heads, mask_len).stride()
        return _native.KVQueryStruct(q.stride(0), q.stride(1), *mask_args, _FLOAT_CODES[q.dtype], heads, mask_code,
                                     mask_len, bool(causal), min(int(window), MAX_LENGTH), scale)

    def kv_attention_workspace_bytes(self, cache: KVCache, batch: KVBatch, *, q_heads: int, dtype: torch.dtype,
                                     window: int | None = None) -> int:
        """Bytes of ``workspace`` that ``kv_attention`` needs for such a call."""
        if dtype not in _FLOAT_CODES:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        query = _native.KVQueryStruct(0, 0, 0, 0, 0, _FLOAT_CODES[dtype], int(q_heads), 0, 0, 1,
                                      min(int(window or 0), MAX_LENGTH), 1.0)
        need = int(self._lib.rnsmx_kv_attention_workspace_bytes(cache._ref, batch._ref, ctypes.addressof(query)))
        if need < 0:
            _native.check(_native.EINVAL)
        return need

    @staticmethod
    def _check_mask(mask: torch.Tensor, batch: KVBatch, heads: int, cache: KVCache) -> None:
        if mask.dtype not in _MASK_CODES or mask.device != cache.device:
            raise ValueError(f"mask must be bool, float32, float16 or bfloat16 on {cache.device}")
        if mask.ndim != 3 or mask.shape[0] not in (1, batch.rows) or mask.shape[1] not in (1, heads):
            raise ValueError(f"mask must be [{batch.rows} or 1, {heads} or 1, tokens], got {tuple(mask.shape)}")
        if batch.longest is not None and mask.shape[2] < batch.longest:
            raise ValueError(f"mask covers {mask.shape[2]} tokens of sequences of up to {batch.longest}")

    def _kv_scratch_for(self, nbytes: int, device: torch.device, stream: int) -> torch.Tensor:
        """The stream's scratch, replaced by a larger one where a call needs it
        (zeroed: its counters are zero between calls).  Work in flight may still
        use the older ones, so they are kept (each less than half the next).
        Under capture it is the graph's own memory, whose counters are cleared
        on every replay: a graph may run beside other calls and other graphs."""
        if torch.cuda.is_current_stream_capturing():
            scratch = torch.empty((nbytes,), dtype=torch.uint8, device=device)
            scratch[:4 * _native.KV_TICKETS].zero_()
            return scratch
        index = device.index if device.index is not None else torch.cuda.current_device()
        held = self._kv_scratch.setdefault((index, stream), [])
        if not held or held[-1].numel() < nbytes:
            size = max(nbytes, 2 * held[-1].numel()) if held else nbytes
            held.append(torch.zeros((size,), dtype=torch.uint8, device=device))
        return held[-1]
