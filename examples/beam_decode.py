"""Beam search over several requests with RNS projections, rotary positions and an
8-bit paged key/value cache whose pages are handed out and shared on the device, on a
decoder of OPT-125m's sizes with random weights.

    python examples/beam_decode.py [--layers 12] [--tokens 32] [--beams 4] [--page 64]

Prompts of different lengths go through the model in one call, one sequence each; the
request's other beams go on from it and share its pages.  A step gives every beam a
page where it needs one, copies the pages that are shared and written next, runs the
model on one token a beam, selects the best continuations and reorders the sequences.
The steps are captured in a HIP graph once and replayed; nothing is read back before
the end.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rns-llm_amd"))

from rns_llm_amd import HipRNSBackend, RNSCachedAttention  # noqa: E402


class Block(nn.Module):
    """A pre-norm decoder block; ``attention`` is made by ``Decoder.use_rns``."""

    def __init__(self, features: int, heads: int, kv_heads: int):
        super().__init__()
        self.heads, self.kv_heads, kv = heads, kv_heads, features // heads * kv_heads
        self.norm_in, self.norm_out = nn.LayerNorm(features), nn.LayerNorm(features)
        self.q_proj, self.out_proj = nn.Linear(features, features), nn.Linear(features, features)
        self.k_proj, self.v_proj = nn.Linear(features, kv), nn.Linear(features, kv)
        self.up, self.down = nn.Linear(features, 2 * features), nn.Linear(2 * features, features)
        self.attention: RNSCachedAttention | None = None

    def forward(self, x, cache, batch, positions):
        x = x + self.attention(self.norm_in(x), cache, batch, positions=positions)
        return x + self.down(F.relu(self.up(self.norm_out(x))))


class Decoder(nn.Module):
    def __init__(self, vocabulary: int, features: int, heads: int, kv_heads: int, layers: int):
        super().__init__()
        self.tokens = nn.Embedding(vocabulary, features)
        self.blocks = nn.ModuleList(Block(features, heads, kv_heads) for _ in range(layers))
        self.norm = nn.LayerNorm(features)

    def use_rns(self, backend) -> None:
        rotary = backend.create_rotary(device=self.tokens.weight.device,
                                       rotary_dim=self.tokens.embedding_dim // self.blocks[0].heads)
        for b in self.blocks:
            b.attention = RNSCachedAttention.from_linears(b.q_proj, b.k_proj, b.v_proj, b.out_proj, backend=backend,
                                                          num_heads=b.heads, num_kv_heads=b.kv_heads, rotary=rotary)

    def forward(self, ids, positions, caches, batch):
        x = self.tokens(ids)
        for block, cache in zip(self.blocks, caches):
            x = block(x, cache, batch, positions)
        return self.norm(x)

    def logits(self, x: torch.Tensor) -> torch.Tensor:
        return F.linear(x, self.tokens.weight)


@torch.no_grad()
def search(model: Decoder, backend, prompts, beams: int, steps: int, page: int, end_token: int, graph: bool = True):
    """``steps`` tokens of each prompt's best ``beams`` continuations: tokens [requests, beams,
    steps] (the end token from where one has ended) and scores [requests, beams], best first."""
    device = model.tokens.weight.device
    requests, lengths = len(prompts), [int(p.shape[0]) for p in prompts]
    width = -(-(max(lengths) + steps) // page)
    # a prompt's pages are shared; a beam has its own from there on, and one that it leaves while it copies
    blocks = sum(-(-n // page) for n in lengths) + requests * beams * (-(-steps // page) + 2)
    pool = backend.create_kv_pool(device=device, blocks=blocks, block_size=page, sequences=requests * beams, width=width)
    caches = [b.attention.create_cache(blocks=blocks, block_size=page) for b in model.blocks]
    # the tokens in pages of their own, found again by the table; a page more for rows without a slot (-1)
    history = torch.full(((blocks + 1) * page,), end_token, dtype=torch.int32, device=device)

    firsts = torch.arange(requests, dtype=torch.int32, device=device) * beams
    new = torch.zeros(requests * beams, dtype=torch.int32, device=device)
    new[firsts.long()] = torch.tensor(lengths, dtype=torch.int32, device=device)
    prompt = backend.kv_step(pool, rows=sum(lengths), max_query=max(lengths))
    backend.kv_assign(pool, prompt, new)
    lacking = prompt.missing != 0  # any step of the search, asked at its end
    positions, slots = backend.kv_slots(pool, prompt.batch)
    ids = torch.cat(list(prompts)).int()
    history[slots] = ids
    x = model(ids, positions, caches, prompt.batch)
    ends = torch.tensor(lengths, device=device).cumsum(0) - 1
    scores, ids, _ = backend.beam_select(model.logits(x[ends]).unsqueeze(1), torch.zeros((requests, 1), device=device), beams,
                                         end_token=end_token)
    finished = ids == end_token
    backend.kv_reorder(pool, firsts.repeat_interleave(beams))
    step = backend.kv_step(pool)

    def advance() -> None:
        backend.kv_assign(pool, step, (~finished).int().view(-1))
        lacking.logical_or_(step.missing)
        for cache in caches:
            backend.kv_copy(cache, step)
        pages = history.view(-1, page)
        source, target = step.copies[:, 0].long(), step.copies[:, 1].long()  # -1: the page past the pool's
        pages[target] = pages[source]
        positions, slots = backend.kv_slots(pool, step.batch)
        history[slots] = ids.view(-1)
        x = model(ids.view(-1), positions, caches, step.batch)
        best = backend.beam_select(model.logits(x).view(requests, beams, -1), scores, beams, finished=finished, end_token=end_token)
        scores.copy_(best[0])
        ids.copy_(best[1])
        finished.copy_(finished.view(-1)[best[2].long()] | (best[1] == end_token))
        backend.kv_reorder(pool, best[2].view(-1))

    state = (pool.table, pool.lengths, pool.refs, pool.free, scores, ids, finished, lacking)
    replay = None
    for i in range(1, steps):
        if replay is None:
            advance()
        else:
            replay.replay()
        if graph and i == 1 and steps > 3:
            # once on the capturing stream, taken back: what it appends is written again by the next step
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                kept = [t.clone() for t in state]
                pages = [t.clone() for c in caches for t in (c.k_codes, c.v_codes, c.scales)]
                advance()
                for t, was in zip(state, kept):
                    t.copy_(was)
                for t, was in zip([t for c in caches for t in (c.k_codes, c.v_codes, c.scales)], pages):
                    t.copy_(was)
            torch.cuda.current_stream().wait_stream(side)
            replay = torch.cuda.CUDAGraph()
            with torch.cuda.graph(replay, stream=side):
                advance()
    # the tokens behind the prompts, the last one of each beam among them: it has no slot yet
    text = history.view(-1, page)[pool.table.clamp(min=0).long()].view(requests * beams, -1)
    at = torch.arange(text.shape[1], device=device)
    text = torch.where(at < pool.lengths.view(-1, 1), text, end_token)
    text = F.pad(text, (0, 1), value=end_token).scatter(1, pool.lengths.long().view(-1, 1), ids.view(-1, 1))
    first = torch.tensor(lengths, device=device).repeat_interleave(beams).view(-1, 1)
    got = text.gather(1, (first + torch.arange(steps, device=device)).clamp(max=text.shape[1] - 1))
    if bool(lacking):
        raise RuntimeError("a step of the search lacked pages")
    return got.view(requests, beams, steps), scores


def build(layers: int = 12, features: int = 768, heads: int = 12, kv_heads: int = 12, vocabulary: int = 50272,
          seed: int = 0) -> Decoder:
    torch.manual_seed(seed)
    model = Decoder(vocabulary, features, heads, kv_heads, layers)
    for p in model.parameters():
        if p.ndim == 2:
            nn.init.normal_(p, std=0.02)
    return model.to(device="cuda", dtype=torch.float16).eval()


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--layers", type=int, default=12)
    parser.add_argument("--tokens", type=int, default=32)
    parser.add_argument("--beams", type=int, default=4)
    parser.add_argument("--page", type=int, default=64, choices=(16, 32, 64, 128))
    args = parser.parse_args()
    backend = HipRNSBackend()
    model = build(args.layers)
    model.use_rns(backend)
    prompts = [torch.randint(3, 50272, (n,), device="cuda") for n in (5, 77, 300, 511)]
    search(model, backend, prompts, args.beams, 5, args.page, 2)
    torch.cuda.synchronize()
    began = time.perf_counter()
    tokens, scores = search(model, backend, prompts, args.beams, args.tokens, args.page, 2)
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    print(f"{args.beams} beams of {len(prompts)} requests, {args.tokens} tokens each in {took * 1e3:.1f} ms, prompts of "
          f"{sum(int(p.shape[0]) for p in prompts)} tokens and one capture among them")
    for r in range(len(prompts)):
        print(f"request {r}: {scores[r, 0].item():.3f}", tokens[r, 0, :8].tolist())


if __name__ == "__main__":
    main()
