"""Greedy decoding of several requests with RNS projections and an 8-bit paged
key/value cache, on a decoder of OPT-125m's sizes with random weights.

    python examples/cached_decode.py [--layers 12] [--tokens 64] [--page 64]

Prompts of different lengths go through the model in one call; then each step
appends one token per request.  The pages of the longest run are handed out
beforehand, so a step only adds one to the lengths; the steps are captured in a
HIP graph once and replayed.
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
    """A pre-norm decoder block; its attention's projections are plain until
    ``Decoder.use_rns``."""

    def __init__(self, features: int, heads: int):
        super().__init__()
        self.heads = heads
        self.norm_in, self.norm_out = nn.LayerNorm(features), nn.LayerNorm(features)
        self.q_proj, self.k_proj, self.v_proj, self.out_proj = (nn.Linear(features, features) for _ in range(4))
        self.up, self.down = nn.Linear(features, 2 * features), nn.Linear(2 * features, features)
        self.attention: RNSCachedAttention | None = None

    def rest(self, x: torch.Tensor, attended: torch.Tensor) -> torch.Tensor:
        x = x + attended
        return x + self.down(F.relu(self.up(self.norm_out(x))))


class Decoder(nn.Module):
    def __init__(self, vocabulary: int, features: int, heads: int, layers: int, positions: int):
        super().__init__()
        self.tokens, self.positions = nn.Embedding(vocabulary, features), nn.Embedding(positions, features)
        self.blocks = nn.ModuleList(Block(features, heads) for _ in range(layers))
        self.norm = nn.LayerNorm(features)

    def use_rns(self, backend) -> None:
        for block in self.blocks:
            block.attention = RNSCachedAttention.from_linears(block.q_proj, block.k_proj, block.v_proj, block.out_proj,
                                                              backend=backend, num_heads=block.heads)

    def logits(self, x: torch.Tensor) -> torch.Tensor:
        return F.linear(self.norm(x), self.tokens.weight)

    def cached(self, ids: torch.Tensor, positions: torch.Tensor, caches, batch) -> torch.Tensor:
        """The last hidden states of a batch's rows."""
        x = self.tokens(ids) + self.positions(positions)
        for block, cache in zip(self.blocks, caches):
            x = block.rest(x, block.attention(block.norm_in(x), cache, batch))
        return x

    def dense(self, ids: torch.Tensor) -> torch.Tensor:
        """The hidden states of one whole sequence with plain projections and attention."""
        n = ids.shape[0]
        x = self.tokens(ids) + self.positions(torch.arange(n, device=ids.device))
        hidden = torch.ones((n, n), dtype=torch.bool, device=ids.device).triu(1)
        for block in self.blocks:
            y = block.norm_in(x)
            q, k, v = (p(y).view(n, block.heads, -1).transpose(0, 1) for p in (block.q_proj, block.k_proj, block.v_proj))
            scores = torch.matmul(q, k.transpose(1, 2).contiguous()) * q.shape[-1] ** -0.5
            p = torch.softmax(scores.masked_fill(hidden, -torch.inf), dim=-1)
            x = block.rest(x, block.out_proj(torch.matmul(p, v).transpose(0, 1).reshape(n, -1)))
        return x


@torch.no_grad()
def generate(model: Decoder, backend, prompts, steps: int, page: int, graph: bool = True):
    """``steps`` greedy tokens for each prompt (a 1-D tensor of ids): the tokens
    [requests, steps] and the logits they were taken from."""
    device = model.tokens.weight.device
    lengths = [int(p.shape[0]) for p in prompts]
    width = -(-(max(lengths) + steps) // page)
    table = torch.arange(len(prompts) * width, dtype=torch.int32, device=device).view(len(prompts), width)
    caches = [b.attention.create_cache(blocks=table.numel(), block_size=page) for b in model.blocks]

    prompt = backend.kv_batch(caches[0], table, lengths, query_lengths=lengths)
    positions = torch.cat([torch.arange(n, device=device) for n in lengths])
    x = model.cached(torch.cat(list(prompts)), positions, caches, prompt)
    last = torch.tensor(lengths, device=device).cumsum(0) - 1
    scores = model.logits(x[last])
    ids = scores.argmax(dim=-1)
    taken, seen = [ids.clone()], [scores]

    held = torch.tensor(lengths, dtype=torch.int32, device=device)  # advanced on the device
    batch = backend.kv_batch(caches[0], table, held)

    def step():
        held.add_(1)
        out = model.logits(model.cached(ids, held - 1, caches, batch))
        ids.copy_(out.argmax(dim=-1))
        return out

    replay, captured = None, None
    for i in range(1, steps):
        if replay is None:
            out = step()
        else:
            replay.replay()
            out = captured.clone()
        taken.append(ids.clone())
        seen.append(out)
        if graph and i == 1 and steps > 2:
            # weights are prepared and workspaces made; the capture runs nothing
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                kept = (held.clone(), ids.clone())
                step()  # once on the capturing stream; taken back below
                held.copy_(kept[0])
                ids.copy_(kept[1])
            torch.cuda.current_stream().wait_stream(side)
            replay = torch.cuda.CUDAGraph()
            with torch.cuda.graph(replay, stream=side):
                captured = step()
    return torch.stack(taken, dim=1), torch.stack(seen, dim=1)


def build(layers: int = 12, features: int = 768, heads: int = 12, vocabulary: int = 50272, positions: int = 2048,
          seed: int = 0) -> Decoder:
    torch.manual_seed(seed)
    model = Decoder(vocabulary, features, heads, layers, positions)
    for p in model.parameters():
        if p.ndim == 2:
            nn.init.normal_(p, std=0.02)
    return model.to(device="cuda", dtype=torch.float16).eval()


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--layers", type=int, default=12)
    parser.add_argument("--tokens", type=int, default=64)
    parser.add_argument("--page", type=int, default=64, choices=(16, 32, 64, 128))
    args = parser.parse_args()
    backend = HipRNSBackend()
    model = build(args.layers)
    model.use_rns(backend)
    prompts = [torch.randint(0, 50272, (n,), device="cuda") for n in (5, 77, 300, 511)]
    generate(model, backend, prompts, 4, args.page)
    torch.cuda.synchronize()
    began = time.perf_counter()
    tokens, _ = generate(model, backend, prompts, args.tokens, args.page)
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    print(f"{tokens.numel()} tokens of {len(prompts)} requests in {took * 1e3:.1f} ms, prompts of "
          f"{sum(int(p.shape[0]) for p in prompts)} tokens and one capture among them")
    print("first tokens:", tokens[:, :8].tolist())


if __name__ == "__main__":
    main()
