"""Pages handed out, shared and copied on the GPU, against a book kept one page at a time."""
import random

import pytest
import torch

from oracle import decode_oracle as do

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def pair(backend, blocks, page, seqs, width):
    return (backend.create_kv_pool(device=DEV, blocks=blocks, block_size=page, sequences=seqs, width=width),
            do.PageBook(blocks, page, seqs, width))


def same(pool, book):
    assert torch.equal(pool.table.cpu(), book.table())
    assert pool.lengths.tolist() == book.lengths and pool.refs.tolist() == book.refs
    assert pool.free[:pool.blocks].tolist() == [int(r == 0) for r in book.refs] and not pool.free[pool.blocks:].any()
    marks = pool._scratch[:2 * pool.blocks].view(2, -1)
    assert not marks[0].any() and (marks[1] == 2 ** 31 - 1).all()  # as the next call needs them


def assign(backend, pool, book, step, new):
    backend.kv_assign(pool, step, None if new is None else ints(new))
    want = book.assign([1] * book.seqs if new is None else new, step.batch.rows, step.batch.max_query, step.batch.max_length)
    assert step.lengths.tolist() == want[0] and [tuple(c) for c in step.copies.tolist()] == want[2]
    assert step.missing.tolist() == [want[3]] and (step.starts is None or step.starts.tolist() == want[1])
    same(pool, book)
    return want[3]


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("blocks,page,seqs,width", [(1, 16, 1, 1), (37, 16, 3, 9), (300, 32, 64, 12), (700, 128, 130, 5), (90, 64, 17, 40)])
def test_calls_in_any_order(backend, blocks, page, seqs, width, seed):
    rng = random.Random(seed * 1000 + seqs)
    pool, book = pair(backend, blocks, page, seqs, width)
    steps = [backend.kv_step(pool), backend.kv_step(pool, rows=seqs * 3 * page, max_query=3 * page),
             backend.kv_step(pool, rows=seqs * 2, max_query=7, max_length=width * page - page // 2)]
    outcomes = set()
    for _ in range(40):
        call = rng.choice(("assign", "assign", "assign", "trim", "reorder"))
        if call == "assign":
            step = rng.choice(steps)
            most = rng.choice((1, 2, 5, 3 * page))
            new = rng.choice((None, [rng.randint(0, 1) for _ in range(seqs)], [rng.randint(-2, most) for _ in range(seqs)],
                              [rng.randint(1, most) if rng.random() < 0.1 else 0 for _ in range(seqs)]))
            outcomes.add(min(assign(backend, pool, book, step, new), 1))
        elif call == "trim":
            to = [rng.choice((0, n, n - rng.randint(0, page), n + 5, -1, rng.randint(0, n + 1), 2 ** 31 - 1)) for n in book.lengths]
            backend.kv_trim(pool, ints(to))
            book.trim(to)
        else:
            near = rng.random() < 0.7
            parents = [max(0, s - rng.randint(0, 3)) if near else rng.choice((s, rng.randrange(seqs), -1, seqs, 2 ** 31 - 1, -2 ** 31))
                       for s in range(seqs)]
            backend.kv_reorder(pool, ints(parents))
            book.reorder(parents)
        same(pool, book)
    assert 0 in outcomes


@pytest.mark.parametrize("seqs,width,page,blocks", [
    (1500, 7, 16, 4000),    # more sequences than threads, page numbers in shared memory
    (2500, 9, 16, 9000),    # more of both
    (40, 300, 16, 12001),   # few long ones
    (1, 5000, 16, 5000),    # one, of all pages
])
def test_many_sequences_and_pages(backend, seqs, width, page, blocks):
    rng = random.Random(seqs)
    pool, book = pair(backend, blocks, page, seqs, width)
    whole = min(width, blocks // seqs) * page
    step = backend.kv_step(pool, rows=seqs * whole, max_query=whole)
    for new in ([rng.randint(0, whole // 2) for _ in range(seqs)], [rng.randint(0, 1) * rng.randint(0, whole // 4) for _ in range(seqs)]):
        assert assign(backend, pool, book, step, new) == 0
    parents = [s - s % 3 for s in range(seqs)]
    backend.kv_reorder(pool, ints(parents))
    book.reorder(parents)
    same(pool, book)
    assert assign(backend, pool, book, step, [1] * seqs) == 0
    assert assign(backend, pool, book, backend.kv_step(pool), None) == 0
    to = [rng.randint(0, n) for n in book.lengths]
    backend.kv_trim(pool, ints(to))
    book.trim(to)
    same(pool, book)
    assert assign(backend, pool, book, step, [whole - n if whole > n and rng.random() < 0.5 else 0 for n in book.lengths]) == 0
    over = [width * page - n + 1 if s == seqs - 1 else 0 for s, n in enumerate(book.lengths)]
    assert assign(backend, pool, book, backend.kv_step(pool, rows=2 * width * page), over) == -1


def test_a_pool_that_is_full(backend):
    """The last page goes, the next call says how many it lacks and changes nothing, on and on until there is room."""
    pool, book = pair(backend, 10, 16, 4, 8)
    step = backend.kv_step(pool, rows=512)
    assert assign(backend, pool, book, step, [100, 33, 0, 0]) == 0  # 7 + 3 pages
    for new, lacks in (([0, 0, 1, 0], 1), ([13, 0, 16, 17], 4), ([12, 15, 0, 0], 0), ([1, 0, 0, 0], 1), ([0, 0, 0, 0], 0)):
        assert assign(backend, pool, book, step, new) == lacks
    backend.kv_reorder(pool, ints([0, 1, 1, -1]))
    book.reorder([0, 1, 1, -1])
    assert assign(backend, pool, book, step, [0, 0, 1, 0]) == 1  # sequence 2 shares a full page: it lacks a new one
    book.trim([128, 40, 40, 0])
    backend.kv_trim(pool, ints([128, 40, 40, 0]))
    assert assign(backend, pool, book, step, [0, 1, 1, 0]) == 1  # the first keeps the page, the second lacks a copy
    assert assign(backend, pool, book, step, [0, 1, 0, 0]) == 1  # the other holds on to it
    # nothing is appended and attention is zero in a step that lacks pages
    cache = backend.create_kv_cache(device=DEV, blocks=10, block_size=16, kv_heads=1, head_dim=64)
    cache.k_codes.fill_(7)
    one = torch.ones((512, 1, 64), device=DEV)
    backend.kv_copy(cache, step)
    backend.kv_append(cache, step.batch, one, one)
    assert (cache.k_codes == 7).all() and (backend.kv_attention(one, cache, step.batch)[:1] == 0).all()


def test_bytes_past_the_last_page(backend):
    """They are no pages, whatever they hold, and of a page's byte the lowest bit counts."""
    for blocks, rows in ((37, 600), (5000, 80008)):  # as many as the first call asks for
        pool, book = pair(backend, blocks, 16, 2, blocks)
        pool.free[blocks:] = 1
        pool.free[3] = 255
        step = backend.kv_step(pool, rows=rows)
        backend.kv_assign(pool, step, ints([16 * blocks - 48, 56]))
        assert step.missing.tolist() == [1] and (pool.refs == 0).all()
        backend.kv_assign(pool, step, ints([16 * blocks - 48, 48]))
        book.assign([16 * blocks - 48, 48], rows, rows, 16 * blocks)
        assert torch.equal(pool.table.cpu(), book.table()) and pool.refs.tolist() == book.refs and not pool.free[:blocks].any()


def test_bounds_of_a_step(backend):
    pool, book = pair(backend, 50, 16, 3, 6)
    step = backend.kv_step(pool, rows=20, max_query=9, max_length=40)
    assert assign(backend, pool, book, step, [9, 9, 2]) == 0
    assert assign(backend, pool, book, step, [9, 9, 3]) == -2
    assert assign(backend, pool, book, step, [2 ** 31 - 1, 5, -2 ** 31]) == 0  # cut to nine and to none
    for new in ([9, 0, 0], [9, 0, 9], [4, 4, 4]):
        assert assign(backend, pool, book, step, new) == 0
    assert book.lengths == [40, 18, 15]
    assert assign(backend, pool, book, step, [1, 0, 0]) == -1
    assert assign(backend, pool, book, step, [0, 0, 0]) == 0
    none = backend.kv_step(pool, rows=0)
    assert assign(backend, pool, book, none, [5, 0, 0]) == 0  # cut to none


# ---- slots -------------------------------------------------------------------
def check_slots(backend, pages, batch, table, lengths, starts):
    got = backend.kv_slots(pages, batch)
    want = do.slots(table.tolist(), lengths, starts, batch.rows, pages.block_size, pages.blocks, batch.max_query, batch.max_length)
    assert got[0].dtype == torch.int32 and torch.equal(got[0].cpu(), want[0])
    assert got[1].dtype == torch.int64 and torch.equal(got[1].cpu(), want[1])


@pytest.mark.parametrize("seed", range(8))
def test_slots(backend, seed):
    """Any batch: idle sequences, rows before the first token and past the bounds, pages that are not there."""
    rng = random.Random(seed)
    page, seqs, width, blocks = rng.choice((16, 32, 64, 128)), rng.choice((1, 2, 9, 300, 5000)), rng.randint(1, 9), 1 << 20
    table = torch.tensor([[rng.choice((rng.randrange(blocks), rng.randrange(blocks), -1, blocks, 2 ** 31 - 1, -2 ** 31)) for _ in range(width)]
                          for _ in range(seqs)], dtype=torch.int32)
    lengths = [rng.choice((0, rng.randint(0, width * page), width * page + 3, -4)) for _ in range(seqs)]
    pages = backend.create_kv_pool(device=DEV, blocks=blocks, block_size=page, sequences=1, width=1)
    starts = [rng.choice((0, 0, 2))]
    for _ in range(seqs):
        starts.append(starts[-1] + rng.choice((0, 0, 1, 1, rng.randint(0, 12), rng.randint(0, 300) if seqs < 20 else 1)))
    for rows in (starts[-1], starts[-1] + 70, max(0, starts[-1] - 5)):
        batch = backend.kv_batch(pages, table.to(DEV), ints(lengths), query_starts=ints(starts), rows=rows,
                                 max_query=rng.choice((1, 5, 400)), max_length=rng.choice((width * page, width * page // 2)))
        check_slots(backend, pages, batch, table, lengths, starts)
    batch = backend.kv_batch(pages, table.to(DEV), ints(lengths))
    check_slots(backend, pages, batch, table, lengths, None)


def test_slots_of_many_rows(backend):
    """Groups of rows of one sequence and of many, a table cut out of a wider one, numbers past 32 bits."""
    rng = random.Random(3)
    blocks = 2 ** 30
    counts = [140000, 0, 3, 1, 1, 64, 130000, 63, 1] + [rng.randint(0, 3) for _ in range(300)]
    width = -(-max(counts) // 16) + 2
    table = torch.randint(0, blocks, (len(counts), width + 3), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    lengths = [n + rng.randint(0, 20) for n in counts]
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    cache = backend.create_kv_cache(device=DEV, blocks=1, block_size=16, kv_heads=1, head_dim=64)
    pages = type("Pages", (), {"device": cache.device, "block_size": 16, "blocks": blocks})()
    view = table.to(DEV)[:, 2:width + 2]
    batch = backend.kv_batch(cache, view, ints(lengths), query_starts=ints(starts), rows=starts[-1] + 9, max_query=max(counts))
    check_slots(backend, pages, batch, table[:, 2:width + 2], lengths, starts)


@pytest.mark.parametrize("seqs", [1, 2, 63, 64, 65, 127, 4095, 4096, 4097, 70000])
@pytest.mark.parametrize("many", [False, True])
def test_slots_of_many_sequences(backend, seqs, many):
    """Numbers of sequences around those that one search's steps and shared memory hold, most of them idle or not."""
    rng = random.Random(seqs + many)
    table = torch.randint(0, 500, (seqs, 4), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    lengths = [rng.randint(0, 64) for _ in range(seqs)]
    starts = [0]
    for _ in range(seqs):
        starts.append(starts[-1] + (rng.choice((0, 1, 1, 2, 40)) if many else int(rng.random() < 0.02) * 70))
    pages = backend.create_kv_pool(device=DEV, blocks=500, block_size=16, sequences=1, width=1)
    batch = backend.kv_batch(pages, table.to(DEV), ints(lengths), query_starts=ints(starts), rows=starts[-1] + 1, max_query=90)
    check_slots(backend, pages, batch, table, lengths, starts)


# ---- copies ------------------------------------------------------------------
@pytest.mark.parametrize("dim", [40, 96, 128, 160, 192, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_copies(backend, dim, page):
    gen = torch.Generator().manual_seed(dim)
    pool = backend.create_kv_pool(device=DEV, blocks=40, block_size=page, sequences=14, width=2)
    cache = backend.create_kv_cache(device=DEV, blocks=41, block_size=page, kv_heads=3, head_dim=dim)
    for codes in (cache.k_codes, cache.v_codes):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=gen, dtype=torch.uint8))
    cache.scales.copy_(torch.rand(cache.scales.shape, generator=gen))
    before = [x.clone() for x in (cache.k_codes, cache.v_codes, cache.scales)]
    step = backend.kv_step(pool)
    copies = [(0, 20, page), (0, 21, 1), (3, 22, page // 2 + 1), (-1, -1, 0), (4, 23, page - 1), (5, -1, 3), (-1, 24, 3), (41, 25, 3),
              (6, 41, 3), (2 ** 31 - 1, 26, 3), (7, 27, 0), (8, 8, 5), (9, 28, -3), (10, 29, 9999)]
    step.copies.copy_(ints(copies))
    backend.kv_copy(cache, step)
    for source, target, tokens in copies:
        if 0 <= source < 41 and 0 <= target < 41:
            for x in before[:2]:
                n = min(max(tokens, 0), page)
                x[target, :, :n] = x[source, :, :n]
            before[2][target] = before[2][source]
    for x, y in zip((cache.k_codes, cache.v_codes, cache.scales), before):
        assert torch.equal(x, y)


def test_graphs(backend):
    """A captured step hands out pages, copies and finds slots on each replay as eager calls do."""
    pool, book = pair(backend, 60, 16, 6, 8)
    step = backend.kv_step(pool)
    prompt = backend.kv_step(pool, rows=200)
    parents, to = ints([0, 0, 2, 3, 3, 5]), ints([2 ** 31 - 1] * 6)
    assign(backend, pool, book, prompt, [20, 3, 0, 40, 16, 31])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        backend.kv_trim(pool, to)
        backend.kv_reorder(pool, parents)
        backend.kv_assign(pool, step)
        positions, slots = backend.kv_slots(pool, step.batch)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(24):
        cut = [n - i % 3 for n in book.lengths]
        to.copy_(ints(cut))
        order = [0, 0, 2, 3, 3, 5] if i % 2 else [1, 0, 2, 4, 4, 5]
        parents.copy_(ints(order))
        graph.replay()
        book.trim(cut)
        book.reorder(order)
        want = book.assign([1] * 6, 6, 1, 128)
        assert step.lengths.tolist() == want[0] and [tuple(c) for c in step.copies.tolist()] == want[2]
        same(pool, book)
        places = do.slots(book.table().tolist(), want[0], None, 6, 16, 60, 1, 128)
        assert torch.equal(positions.cpu(), places[0]) and torch.equal(slots.cpu(), places[1])
