"""Pools whose sequences are too many for one launch, and reorders of tables past one workgroup's."""
import random

import pytest
import torch

from oracle import decode_oracle as do

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("log_seqs,width", [(26, 1), (24, 65)])
def test_sequences_of_several_launches(backend, log_seqs, width):
    """A workgroup for each: 2^32 threads and more."""
    seqs, blocks = 2 ** log_seqs + 3, 40
    pool = backend.create_kv_pool(device=DEV, blocks=blocks, block_size=16, sequences=seqs, width=width)
    some = torch.tensor([0, 1, 511, 2 ** (log_seqs - 1), 2 ** log_seqs - 513, 2 ** log_seqs - 512, 2 ** log_seqs - 1, 2 ** log_seqs,
                         seqs - 1], device=DEV)
    n = some.shape[0]
    pages = torch.arange(n, dtype=torch.int32, device=DEV) + 7
    pool.table[some, 0] = pages
    pool.lengths[some] = 16
    pool.refs[7:7 + n] = 1
    pool.free[7:7 + n] = 0

    def held(order, refs):
        assert pool.table[some, 0].tolist() == [pages[i].item() if i >= 0 else -1 for i in order]
        assert pool.lengths[some].tolist() == [16 * (i >= 0) for i in order]
        assert int((pool.table >= 0).sum()) == int((pool.lengths > 0).sum()) == sum(i >= 0 for i in order)
        assert pool.refs.tolist() == refs and pool.free[:blocks].tolist() == [int(r == 0) for r in refs]

    # the first becomes the last, the others the one before; one becomes empty
    parents = torch.arange(seqs, dtype=torch.int32, device=DEV)
    order = [n - 1] + list(range(n - 1))
    parents[some] = some[torch.tensor(order, device=DEV)].int()
    parents[some[4]] = -1
    order[4] = -1
    backend.kv_reorder(pool, parents)
    held(order, [1 if 7 <= p < 7 + n and p != 7 + 3 else 0 for p in range(blocks)])
    to = torch.full((seqs,), 99, dtype=torch.int32, device=DEV)
    to[some[1:]] = 0
    backend.kv_trim(pool, to)
    held([n - 1] + [-1] * (n - 1), [int(p == 7 + n - 1) for p in range(blocks)])


@pytest.mark.parametrize("seqs,width,page,blocks", [(1500, 7, 16, 9000), (40, 300, 16, 12001), (8193, 1, 128, 9000), (3, 5000, 16, 15000)])
def test_parents_of_large_tables(backend, seqs, width, page, blocks):
    """Any parents where what every sequence becomes is laid aside by one launch and takes its place in the next:
    in a ring, turned round, of one, at random, some of them no sequence's, and what pages they have given back."""
    rng = random.Random(seqs)
    pool = backend.create_kv_pool(device=DEV, blocks=blocks, block_size=page, sequences=seqs, width=width)
    book = do.PageBook(blocks, page, seqs, width)
    most = min(width * page - 3, blocks // seqs * page)
    step = backend.kv_step(pool, rows=seqs * most, max_query=most)

    def same():
        assert torch.equal(pool.table.cpu(), book.table())
        assert pool.lengths.tolist() == book.lengths and pool.refs.tolist() == book.refs
        assert pool.free[:blocks].tolist() == [int(r == 0) for r in book.refs] and not pool.free[blocks:].any()

    def assign(new):
        backend.kv_assign(pool, step, torch.tensor(new, dtype=torch.int32, device=DEV))
        want = book.assign(new, step.batch.rows, step.batch.max_query, step.batch.max_length)
        assert step.missing.tolist() == [want[3]] and [tuple(c) for c in step.copies.tolist()] == want[2]
        assert step.lengths.tolist() == want[0] and step.starts.tolist() == want[1]
        same()

    assign([rng.randint(0, most) for _ in range(seqs)])
    none = (-1, seqs, seqs + 5, 2 ** 31 - 1, -2 ** 31)
    shuffled = list(range(seqs))
    rng.shuffle(shuffled)
    for parents in ([(s + 1) % seqs for s in range(seqs)], [(s - 1) % seqs for s in range(seqs)], list(range(seqs))[::-1], shuffled,
                    [rng.randrange(seqs) for _ in range(seqs)], [rng.choice((s, rng.randrange(seqs), rng.choice(none))) for s in range(seqs)],
                    [s if s % 2 else none[s % 5] for s in range(seqs)], [seqs - 1] * seqs, [-1] * seqs):
        backend.kv_reorder(pool, torch.tensor(parents, dtype=torch.int32, device=DEV))
        book.reorder(parents)
        same()
        assign([int(rng.random() < 0.7) for _ in range(seqs)])  # pages of several holders are replaced, freed ones taken
    assert not any(book.lengths) or max(book.lengths) <= 1
