"""The decoding loop's operators together: beams that share pages against beams that each
keep all of their own, the layer with rotary positions, and the beam search example."""
import importlib.util
import os

import pytest
import torch
from torch import nn

from oracle import decode_oracle as do
from rns_llm_amd import RNSCachedAttention

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("beam_decode", os.path.join(ROOT, "examples", "beam_decode.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("page,dim,kv_heads,beams", [(16, 64, 2, 3), (32, 96, 1, 4), (64, 128, 2, 2)])
def test_shared_pages_hold_what_whole_copies_do(backend, page, dim, kv_heads, beams):
    """A beam search on random projections of the tokens: every step's attention, and what the pages hold,
    bit for bit as where each beam has pages of its own and takes over all of its parent's."""
    gen = torch.Generator().manual_seed(page)
    requests, heads, vocabulary, steps = 3, 4, 97, 40
    lengths = [page + 5, 3, 2 * page]
    seqs, width = requests * beams, -(-(max(lengths) + steps) // page)
    table = torch.randn((vocabulary, heads + 2 * kv_heads, dim), generator=gen).half().to(DEV)
    read = (torch.randn((heads * dim, vocabulary), generator=gen) * 0.2).to(DEV)
    rotary = backend.create_rotary(device=DEV, rotary_dim=dim // 2, layout="interleaved")
    pool = backend.create_kv_pool(device=DEV, blocks=70, block_size=page, sequences=seqs, width=width)
    shared = backend.create_kv_cache(device=DEV, blocks=70, block_size=page, kv_heads=kv_heads, head_dim=dim)
    private = backend.create_kv_cache(device=DEV, blocks=seqs * width, block_size=page, kv_heads=kv_heads, head_dim=dim)
    own = torch.arange(seqs * width, dtype=torch.int32, device=DEV).view(seqs, width)

    def attend(step, ids):
        positions, slots = backend.kv_slots(pool, step.batch)
        x = table[ids.long()]
        q, k = backend.rotate(rotary, positions, x[:, :heads], x[:, heads:heads + kv_heads])
        v = x[:, heads + kv_heads:]
        backend.kv_copy(shared, step)
        backend.kv_append(shared, step.batch, k, v)
        got = backend.kv_attention(q, shared, step.batch)
        starts = {} if step.starts is None else dict(query_starts=step.starts, rows=step.batch.rows, max_query=step.batch.max_query)
        batch = backend.kv_batch(private, own, step.lengths, **starts)
        backend.kv_append(private, batch, k, v)
        assert torch.equal(got, backend.kv_attention(q, private, batch))
        return got

    def reorder(parents):
        backend.kv_reorder(pool, parents)
        for x in (private.k_codes, private.v_codes, private.scales):
            x.copy_(x.view(seqs, width, *x.shape[1:])[parents.long()].reshape(x.shape))

    new = torch.zeros(seqs, dtype=torch.int32)
    new[::beams] = torch.tensor(lengths, dtype=torch.int32)
    step = backend.kv_step(pool, rows=sum(lengths), max_query=max(lengths))
    backend.kv_assign(pool, step, new.to(DEV))
    out = attend(step, torch.randint(0, vocabulary, (sum(lengths),), generator=gen).to(DEV))
    ends = torch.tensor(lengths).cumsum(0) - 1
    logits = out[ends.to(DEV)].float().view(requests, -1) @ read
    scores, ids, _ = backend.beam_select(logits.view(requests, 1, -1), torch.zeros((requests, 1), device=DEV), beams)
    reorder(torch.arange(seqs, dtype=torch.int32, device=DEV) // beams * beams)
    step = backend.kv_step(pool)
    copied = 0
    for _ in range(steps):
        backend.kv_assign(pool, step)
        copied += int((step.copies[:, 1] >= 0).sum())
        logits = (attend(step, ids.view(-1)).float().view(seqs, -1) @ read).view(requests, beams, -1)
        want = do.beam_select(logits.cpu(), scores.cpu(), beams)
        scores, ids, parents = backend.beam_select(logits, scores, beams)
        assert torch.allclose(scores.cpu().double(), want[0], atol=1e-4)
        reorder(parents.view(-1))
    assert int(step.missing) == 0 and copied > 10
    held = pool.lengths.tolist()
    whole = [backend.kv_read(c, backend.kv_batch(c, t, held, query_lengths=held), dtype=torch.float32)
             for c, t in ((shared, pool.table), (private, own))]
    assert all(torch.equal(a, b) for a, b in zip(*whole))
    used = pool.table[pool.table >= 0].unique().numel()
    assert used == int((pool.refs > 0).sum()) < int((pool.table >= 0).sum())
    backend.kv_trim(pool, torch.zeros(seqs, dtype=torch.int32, device=DEV))
    assert not pool.refs.any() and pool.free[:70].all()


@pytest.mark.parametrize("layout,part", [("half", 64), ("interleaved", 32)])
@torch.no_grad()
def test_layer_is_its_parts(backend, layout, part):
    torch.manual_seed(3)
    heads, kv_heads, dim, features = 4, 2, 64, 192
    linears = [nn.Linear(features, h * dim) for h in (heads, kv_heads, kv_heads)] + [nn.Linear(heads * dim, features)]
    rotary = backend.create_rotary(device=DEV, rotary_dim=part, layout=layout)
    layer = RNSCachedAttention.from_linears(*(p.to(DEV, torch.float16) for p in linears), backend=backend, num_heads=heads,
                                            num_kv_heads=kv_heads, rotary=rotary)
    caches = [layer.create_cache(blocks=12, block_size=16) for _ in range(3)]
    table = torch.randperm(12, dtype=torch.int32).view(2, 6).to(DEV)
    for lengths, news in (([70, 33], [70, 33]), ([71, 34], [1, 1]), ([75, 35], [4, 1])):
        batch = backend.kv_batch(caches[0], table, lengths, query_lengths=news)
        x = torch.randn((sum(news), features), device=DEV, dtype=torch.float16)
        got = layer(x, caches[0], batch)
        positions = torch.cat([torch.arange(n - m, n) for n, m in zip(lengths, news)]).to(DEV)
        assert torch.equal(layer(x, caches[2], batch, positions=positions), got)
        q, k, v = (y.reshape(sum(news), -1, dim) for y in layer.projection(x))
        q, k = backend.rotate(rotary, positions, q, k)
        backend.kv_append(caches[1], batch, k, v)
        out = backend.kv_attention(q, caches[1], batch)
        assert torch.equal(got, layer.out_proj(out.reshape(sum(news), -1)))


@torch.no_grad()
def test_beam_search_example(backend):
    """Captured steps give what eager ones give; scores go down, each beam's tokens are its own, and what
    follows the end token is the end token."""
    ex = example()
    model = ex.build(layers=2, features=256, heads=4, kv_heads=2, vocabulary=300)
    model.use_rns(backend)
    gen = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 300, (n,), generator=gen).to(DEV) for n in (1, 40, 77)]
    tokens, scores = ex.search(model, backend, prompts, 4, 30, 16, 7)
    assert tokens.shape == (3, 4, 30) and scores.isfinite().all() and (scores[:, 1:] <= scores[:, :-1]).all()
    eager, eager_scores = ex.search(model, backend, prompts, 4, 30, 16, 7, graph=False)
    assert torch.equal(tokens, eager) and torch.equal(scores, eager_scores)
    for beams in tokens.tolist():
        assert len(set(map(tuple, beams))) == 4
        for row in beams:
            if 7 in row:
                assert set(row[row.index(7):]) == {7}
    # one beam is a greedy search
    tokens, scores = ex.search(model, backend, prompts, 1, 6, 32, 299)
    assert tokens.shape == (3, 1, 6) and (scores < 0).all()
