"""How ``rnsmx_kv_attention`` runs a call, for tests that are about one of its kernels."""
import ctypes

import torch

from rns_llm_amd import _native

DTYPES = {torch.float32: _native.FLOAT32, torch.float16: _native.FLOAT16, torch.bfloat16: _native.BFLOAT16}


def plan(seqs, heads, q_heads, rows, length, dim, *, page=16, window=0, causal=1, masked=False, dtype=torch.bfloat16, width=None):
    """(tile_rows, row_tiles, waves, splits, chunk, stream) from sizes alone:
    `rows` the most of one sequence, `length` its most tokens."""
    lib, out = _native.lib(), _native.KVPlan()
    width = max(1, -(-length // page)) if width is None else width
    cache = _native.KVCacheStruct(4096, 4096, 4096, 4, page, heads, dim, lib.rnsmx_kv_row_bytes(dim))
    batch = _native.KVBatchStruct(4096, width, 4096, 4096, seqs, width, 2 ** 31 - 1, rows, length)
    query = _native.KVQueryStruct(0, 0, 0, 0, 0, DTYPES[dtype], q_heads, 0, 0, causal, window, 0.5)
    _native.check(lib.rnsmx_kv_attention_plan(ctypes.addressof(cache), ctypes.addressof(batch), ctypes.addressof(query), masked,
                                              ctypes.addressof(out)))
    return out.as_tuple()


def plan_of(cache, batch, q_heads, dtype, *, window=None, masked=False):
    """The same of a call's cache and batch."""
    out = _native.KVPlan()
    query = _native.KVQueryStruct(0, 0, 0, 0, 0, DTYPES[dtype], q_heads, 0, 0, 1, window or 0, 0.5)
    _native.check(_native.lib().rnsmx_kv_attention_plan(cache._ref, batch._ref, ctypes.addressof(query), masked,
                                                        ctypes.addressof(out)))
    return out
