"""Sizes, lengths and row starts at the ends of what the key/value cache's entry
points take."""
import ctypes

import pytest
import torch

from kv_plans import plan_of
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
    assert plan_of(cache, batch, 4, torch.float16).tile_rows == (128 if idle else 16)
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


def poison(like):
    """Leaves NaN in the memory that the next tensor of this size gets."""
    torch.full_like(like, torch.nan)


@pytest.mark.parametrize("rows,over", [(1, 1), (1, 30), (5, 2), (5, 5), (20, 3), (20, 50)])
def test_tokens_past_max_length_are_not_appended(backend, rows, over):
    """A captured loop whose lengths run past the bound: rows that have a place
    go there, the others nowhere, and no page's codes or scales change for them."""
    top = 40  # in a page that has room
    first = [25, max(0, top + over - rows)]
    cache, table, gen = filled(backend, [25, 45], room=4)
    twin = backend.create_kv_cache(device=GPU, blocks=cache.blocks, block_size=16, kv_heads=2, head_dim=64)
    for a, b in ((twin.k_codes, cache.k_codes), (twin.v_codes, cache.v_codes), (twin.scales, cache.scales)):
        a.copy_(b)
    starts = ints(0, 2, 2 + rows)
    k, v = (30 * torch.randn((2 + rows, 2, 64), generator=gen).half().to(DEV) for _ in range(2))
    batch = backend.kv_batch(cache, table, ints(27, top + over), query_starts=starts, rows=2 + rows, max_query=max(2, rows),
                             max_length=top)
    backend.kv_append(cache, batch, k, v)
    placed = max(0, top - first[1])
    backend.kv_append(twin, backend.kv_batch(twin, table, [27, top if placed else 0], query_lengths=[2, placed]),
                      k[:2 + placed], v[:2 + placed])
    for a, b in ((twin.k_codes, cache.k_codes), (twin.v_codes, cache.v_codes), (twin.scales, cache.scales)):
        assert torch.equal(a, b)
    poison(k)
    got = backend.kv_read(cache, batch, dtype=torch.float16)
    want = backend.kv_read(cache, backend.kv_batch(cache, table, [27, 40], query_lengths=[2, placed]), dtype=torch.float16)
    for x, y in zip(got, want):
        assert torch.equal(x[:2 + placed], y) and (x[2 + placed:] == 0).all()


@pytest.mark.parametrize("single", [True, False])
def test_a_decode_step_past_the_end_overwrites_nothing(backend, single):
    cache, table, gen = filled(backend, [48, 20])
    before = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.scales)]
    lengths = ints(48, 20)
    if single:
        batch = backend.kv_batch(cache, table, lengths)
    else:
        batch = backend.kv_batch(cache, table, lengths, query_starts=ints(0, 1, 2), rows=2, max_query=1)
    k = 30 * torch.randn((2, 2, 64), generator=gen).half().to(DEV)
    for step in range(3):
        lengths += 1
        k[1] = 0.01  # the other sequence's, which has room
        backend.kv_append(cache, batch, k, k)
    pages = table[0].long()
    for was, now in zip(before, (cache.k_codes, cache.v_codes, cache.scales)):
        assert torch.equal(was[pages], now[pages])
    assert (backend.kv_read(cache, batch, dtype=torch.float32)[0][0] == 0).all()


@pytest.mark.parametrize("idle", [0, MANY])
@pytest.mark.parametrize("most", [0, 1, 3, 33])
def test_rows_past_max_query_move_no_others(backend, idle, most):
    """A sequence with more rows than the batch was told of: its first ones are
    where they belong, the others are not appended and zero in outputs."""
    cache, table, gen = filled(backend, [70, 45, 30], idle=idle)
    news, lengths = [40, 2, 0], [70, 45, 30]
    kept = [min(n, most) for n in news]
    short = [n - m + t if n else n for n, m, t in zip(lengths, news, kept)]
    starts = torch.cat([ints(0, 40, 42), ints(*[42] * (1 + idle))])
    batch = backend.kv_batch(cache, table, ints(*lengths, *[0] * idle), query_starts=starts, rows=42, max_query=most)
    plain = backend.kv_batch(cache, table, short + [0] * idle, query_lengths=kept + [0] * idle)
    pick = torch.cat([torch.arange(kept[0]), 40 + torch.arange(kept[1])]).to(DEV)
    rest = torch.ones(42, dtype=torch.bool, device=DEV)
    rest[pick] = False
    q = torch.randn((42, 4, 64), generator=gen).half().to(DEV)
    assert plan_of(cache, batch, 4, torch.float16).tile_rows == (128 if idle and most == 33 else 16)
    for window in (None, 21):
        out = torch.full_like(q, torch.nan)
        backend.kv_attention(q, cache, batch, window=window, out=out)
        assert (out[rest] == 0).all()
        if most:
            torch.testing.assert_close(out[pick], backend.kv_attention(q[pick], cache, plain, window=window), rtol=2e-3, atol=2e-3)
    k, v = (30 * torch.randn((42, 2, 64), generator=gen).half().to(DEV) for _ in range(2))
    twin = backend.create_kv_cache(device=GPU, blocks=cache.blocks, block_size=16, kv_heads=2, head_dim=64)
    for a, b in ((twin.k_codes, cache.k_codes), (twin.v_codes, cache.v_codes), (twin.scales, cache.scales)):
        a.copy_(b)
    backend.kv_append(cache, batch, k, v)
    backend.kv_append(twin, plain, k[pick], v[pick])
    for a, b in ((twin.k_codes, cache.k_codes), (twin.v_codes, cache.v_codes), (twin.scales, cache.scales)):
        assert torch.equal(a, b)
    poison(k)
    got = backend.kv_read(cache, batch, dtype=torch.float16)
    for x, y in zip(got, backend.kv_read(cache, plain, dtype=torch.float16)):
        assert torch.equal(x[pick], y) and (x[rest] == 0).all()


@pytest.mark.parametrize("idle,rows", [(0, 5), (0, 35), (MANY, 35)])
@pytest.mark.parametrize("over", [1, 4, 200, 2 ** 31 - 1 - 40])
def test_rows_past_max_length_see_what_is_there(backend, idle, rows, over):
    """Rows keep their positions: the window of one past the bound ends where it
    stands, whatever of it is there."""
    top = 40
    cache, table, gen = filled(backend, [48, 48], idle=idle)
    length = top + over
    starts = torch.cat([ints(0, rows), ints(*[2 * rows] * (1 + idle))])
    batch = backend.kv_batch(cache, table, ints(length, 40, *[0] * idle), query_starts=starts, rows=2 * rows, max_query=rows,
                             max_length=top)
    q = torch.randn((2 * rows, 4, 64), generator=gen).half().to(DEV)
    assert plan_of(cache, batch, 4, torch.float16).tile_rows == (128 if idle else 16)
    whole = backend.kv_batch(cache, table, [40, 40] + [0] * idle, query_lengths=[rows, rows] + [0] * idle)
    at = torch.arange(rows).view(-1, 1, 1) + length - rows
    token = torch.arange(40).view(1, 1, 40)
    for window in (None, 7, 2 ** 30):
        seen = (token <= at) & (token > at - (window or 2 ** 40))
        own = torch.arange(rows).view(-1, 1, 1) + 40 - rows
        mask = torch.cat([seen, (token <= own) & (token > own - (window or 2 ** 40))]).to(DEV)
        want = backend.kv_attention(q, cache, whole, causal=False, mask=mask)
        got = backend.kv_attention(q, cache, batch, window=window)
        torch.testing.assert_close(got, want, rtol=2e-3, atol=2e-3)
        assert (got[:rows][~seen.any(dim=2).view(-1).to(DEV)] == 0).all()


@pytest.mark.parametrize("starts", [(0, -2 ** 31, 4), (3, 2 ** 31 - 1, -2 ** 31), (-2 ** 31, 2 ** 31 - 1, 2), (4, 0, 4)])
def test_row_starts_of_any_number(backend, starts):
    """Cut to the rows there are; nothing out of range is touched."""
    cache, table, gen = filled(backend, [40, 17], room=1)
    batch = backend.kv_batch(cache, table, ints(40, 2 ** 31 - 1), query_starts=ints(*starts), rows=4, max_query=3, max_length=40)
    x = torch.randn((4, 2, 64), generator=gen).half().to(DEV)
    edge = torch.zeros((3, 4, 2, 64), dtype=torch.float16, device=DEV)
    backend.kv_attention(x, cache, batch, out=edge[1])
    backend.kv_append(cache, batch, x, x)
    backend.kv_read(cache, batch, dtype=torch.float16)
    torch.cuda.synchronize()
    assert (edge[0] == 0).all() and (edge[2] == 0).all() and edge.isfinite().all()


def test_calls_of_more_threads_than_a_launch_has(backend):
    """A prompt beside many sequences that hold nothing: 2^32 threads and more
    are several launches."""
    heads, rows, seqs = 1024, 2048, 2050
    pages = rows // 16
    cache, twin = (backend.create_kv_cache(device=GPU, blocks=pages, block_size=16, kv_heads=heads, head_dim=1) for _ in range(2))
    table = torch.full((seqs, pages), -1, dtype=torch.int32, device=DEV)
    gen = torch.Generator().manual_seed(33)
    k, v, q = (torch.randn((rows, heads, 1), generator=gen).half().to(DEV) for _ in range(3))
    for at in (0, seqs // 2, seqs - 1):  # in the first launch, one between, the last
        table.fill_(-1)
        table[at] = torch.randperm(pages, generator=gen, dtype=torch.int32)
        counts = [0] * seqs
        counts[at] = rows
        batch = backend.kv_batch(cache, table, counts, query_lengths=counts)
        alone = backend.kv_batch(twin, table[at:at + 1], [rows], query_lengths=[rows])
        backend.kv_append(cache, batch, k, v)
        backend.kv_append(twin, alone, k, v)
        for a, b in ((twin.k_codes, cache.k_codes), (twin.v_codes, cache.v_codes), (twin.scales, cache.scales)):
            assert torch.equal(a, b)
            a.zero_()
            b.zero_()
        backend.kv_append(cache, batch, k, v)
        backend.kv_append(twin, alone, k, v)
        for x, y in zip(backend.kv_read(cache, batch, dtype=torch.float16), backend.kv_read(twin, alone, dtype=torch.float16)):
            assert torch.equal(x, y)
        got, want = backend.kv_attention(q, cache, batch), backend.kv_attention(q, twin, alone)
        torch.testing.assert_close(got, want, rtol=2e-3, atol=2e-3)


def test_single_rows_of_more_threads_than_a_launch_has(backend):
    heads, seqs = 1024, 16500
    cache = backend.create_kv_cache(device=GPU, blocks=4, block_size=16, kv_heads=heads, head_dim=1)
    table = torch.full((seqs, 1), -1, dtype=torch.int32, device=DEV)
    real = [0, 8000, 16383, seqs - 1]
    table[real, 0] = torch.arange(4, dtype=torch.int32, device=DEV)
    counts = torch.zeros(seqs, dtype=torch.int32, device=DEV)
    counts[real] = 1
    q, k, v = (torch.randn((seqs, heads, 1), device=DEV).half() for _ in range(3))
    batch = backend.kv_batch(cache, table, counts)
    backend.kv_append(cache, batch, k, v)
    out = torch.full_like(q, torch.nan)
    backend.kv_attention(q, cache, batch, out=out)
    assert torch.equal(out[real], backend.kv_read(cache, batch, dtype=torch.float16)[1][real])  # one token has all the weight
    empty = torch.ones(seqs, dtype=torch.bool, device=DEV)
    empty[real] = False
    assert (out[empty] == 0).all()


@pytest.mark.parametrize("which", ["q", "mask"])
def test_a_backward_pass_that_gets_here_says_so(backend, which):
    cache, table, gen = filled(backend, [40, 17])
    batch = backend.kv_batch(cache, table, [40, 17], query_lengths=[3, 2])
    q = torch.randn((5, 4, 64), generator=gen).to(DEV)
    mask = torch.randn((1, 1, 40), generator=gen).to(DEV)
    want = backend.kv_attention(q, cache, batch, mask=mask)
    assert not want.requires_grad
    asks = {"q": q, "mask": mask}[which].requires_grad_()
    got = backend.kv_attention(q, cache, batch, mask=mask)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no gradient"):
        got.sum().backward()
    assert asks.grad is None
    with torch.no_grad():
        assert not backend.kv_attention(q, cache, batch, mask=mask).requires_grad
    out = torch.empty_like(want)
    assert backend.kv_attention(q, cache, batch, mask=mask, out=out) is out and not out.requires_grad
    assert not backend.kv_attention(q.detach(), cache, batch, mask=mask.detach()).requires_grad
