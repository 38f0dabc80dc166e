"""Pools whose sequences are too many for one launch, and reorders of tables past one workgroup's."""
import pytest
import torch

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
