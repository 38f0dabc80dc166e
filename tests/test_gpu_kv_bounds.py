"""Sizes, lengths and row starts at the ends of what the key/value cache's entry
points take."""
import ctypes

import pytest
import torch

from rns_llm_amd import _native

pytestmark = pytest.mark.gpu

DEV = "cuda"
GPU = torch.device(DEV, 0)

# Sequences that hold nothing and ask nothing beside a test's own: with so many
# the prompts' kernel runs what few rows' would.
MANY = 170


def filled(backend, lengths, *, heads=2, dim=64, page=16, room=0, seed=1, idle=0):
    """A cache of whole sequences and its block table, `room` pages of each unused."""
    gen = torch.Generator().manual_seed(seed)
    width = -(-max(lengths) // page) + room
    table = torch.randperm(len(lengths) * width, generator=gen, dtype=torch.int32).view(len(lengths), width)
    if idle:
        table = torch.cat([table, torch.full((idle, width), -1, dtype=torch.int32)])
    table = table.to(DEV)
    cache = backend.create_kv_cache(device=GPU, blocks=len(lengths) * width, block_size=page, kv_heads=heads, head_dim=dim)
    k, v = (torch.randn((sum(lengths), heads, dim), generator=gen).half().to(DEV) for _ in range(2))
    whole = list(lengths) + [0] * idle
    backend.kv_append(cache, backend.kv_batch(cache, table, whole, query_lengths=whole), k, v)
    return cache, table, gen


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("idle", [0, MANY])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 4, 2 ** 30 + 1])
def test_windows_of_any_number(backend, window, idle):
    """Rows before a sequence's first token, next to rows that see tokens, and a
    window past what any sequence holds: as without one."""
    lengths, news = [1, 40, 0], [40, 40, 3]
    cache, table, gen = filled(backend, [1, 40, 1], idle=idle)
    batch = backend.kv_batch(cache, table, lengths + [0] * idle, query_lengths=news + [0] * idle)
    q = torch.randn((sum(news), 4, 64), generator=gen).half().to(DEV)
    want = backend.kv_attention(q, cache, batch)
    assert (want[:39] == 0).all() and (want[39:80].abs().amax(dim=(1, 2)) > 0).all()
    query = _native.KVQueryStruct(q.stride(0), q.stride(1), 0, 0, 0, _native.FLOAT16, 4, 0, 0, 1, window, 0.125)
    need = backend._lib.rnsmx_kv_attention_workspace_bytes(cache._ref, batch._ref, ctypes.addressof(query))
    space = torch.zeros((max(need, 16),), dtype=torch.uint8, device=DEV)
    out = torch.empty_like(q)
    _native.check(backend._lib.rnsmx_kv_attention(cache._ref, batch._ref, ctypes.addressof(query), q.data_ptr(), None,
                                                  space.data_ptr(), space.numel(), out.data_ptr(),
                                                  torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out, want)
