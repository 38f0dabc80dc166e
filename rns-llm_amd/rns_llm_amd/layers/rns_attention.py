"""Self-attention on the RNS path with an 8-bit key/value cache.

One fused q/k/v product (``RNSQKVProjection``), rotary positions where the model
has them, the new tokens' keys and values quantised into the cache as the product's column blocks lie, attention over the
cached codes, and the output projection.  Prompts and single tokens take the same
call: the rows of a ``KVBatch``.  No counterpart in the reference, which leaves
what follows its projections to the model."""
from __future__ import annotations

import torch
from torch import nn

from ..backends.kv_cache import KVBatch, KVCache
from ..backends.rotary import Rotary
from .rns_linear import RNSLinear
from .rns_qkv import RNSQKVProjection


class RNSCachedAttention(nn.Module):
    """Causal self-attention of ``num_heads`` query heads over ``num_kv_heads``
    (default: as many) cached ones, with ``rotary`` positions if given.  ``forward``
    takes the rows of a batch, ``[rows, features]``, and returns as many."""

    def __init__(self, projection: RNSQKVProjection, out_proj: nn.Module, *, backend, num_heads: int,
                 num_kv_heads: int | None = None, scale: float | None = None, rotary: Rotary | None = None) -> None:
        super().__init__()
        kv_heads = num_heads if num_kv_heads is None else int(num_kv_heads)
        q_size, k_size, v_size = projection.split_sizes
        if num_heads < 1 or kv_heads < 1 or num_heads % kv_heads or q_size % num_heads:
            raise ValueError(f"{num_heads} query heads over {kv_heads} key/value heads do not fit {q_size} features")
        head_dim = q_size // num_heads
        if k_size != kv_heads * head_dim or v_size != k_size:
            raise ValueError(f"{kv_heads} heads of {head_dim} do not fit k and v of {k_size} and {v_size} features")
        if rotary is not None and rotary.rotary_dim > head_dim:
            raise ValueError(f"rotary positions of {rotary.rotary_dim} values do not fit heads of {head_dim}")
        self.rotary = rotary
        self.projection = projection
        self.out_proj = out_proj
        self.backend = backend
        self.num_heads, self.num_kv_heads, self.head_dim = int(num_heads), kv_heads, head_dim
        self.scale = scale

    @classmethod
    def from_linears(cls, q_proj: nn.Linear, k_proj: nn.Linear, v_proj: nn.Linear, out_proj: nn.Linear, *, backend,
                     num_heads: int, num_kv_heads: int | None = None, scale: float | None = None,
                     rotary: Rotary | None = None, quant_bits: int = 8,
                     adaptive_channels: bool = False) -> "RNSCachedAttention":
        """From a model's four projections, which become RNS layers."""
        options = dict(backend=backend, mode="rns", quant_bits=quant_bits, adaptive_channels=adaptive_channels)
        projection = RNSQKVProjection.from_linears(q_proj, k_proj, v_proj, **options)
        return cls(projection, RNSLinear.from_linear(out_proj, **options), backend=backend, num_heads=num_heads,
                   num_kv_heads=num_kv_heads, scale=scale, rotary=rotary).eval()

    def create_cache(self, *, blocks: int, block_size: int) -> KVCache:
        """An empty cache for this layer's heads."""
        return self.backend.create_kv_cache(device=self.projection.combined.weight.device, blocks=blocks,
                                            block_size=block_size, kv_heads=self.num_kv_heads, head_dim=self.head_dim)

    def forward(self, hidden: torch.Tensor, cache: KVCache, batch: KVBatch, *, window: int | None = None,
                mask: torch.Tensor | None = None, positions: torch.Tensor | None = None) -> torch.Tensor:
        """``positions`` of the rows are those of ``kv_slots`` by default: a model's layers
        save that call by sharing them."""
        if hidden.ndim != 2 or hidden.shape[0] != batch.rows:
            raise ValueError(f"hidden must hold the batch's {batch.rows} rows, got {tuple(hidden.shape)}")
        q, k, v = self.projection(hidden)
        rows = batch.rows
        q = q.view(rows, self.num_heads, self.head_dim)
        k, v = (x.view(rows, self.num_kv_heads, self.head_dim) for x in (k, v))
        if self.rotary is not None:
            if positions is None:
                positions = self.backend.kv_slots(cache, batch)[0]
            # not in place: the product's columns are also a forward hook's on the projection
            q, k = self.backend.rotate(self.rotary, positions, q, k)
        self.backend.kv_append(cache, batch, k, v)
        out = self.backend.kv_attention(q, cache, batch, scale=self.scale, window=window, mask=mask)
        return self.out_proj(out.view(rows, self.num_heads * self.head_dim))
