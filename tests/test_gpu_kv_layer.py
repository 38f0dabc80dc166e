"""The cached attention layer and the decoding example: the layer is its parts,
and a decoder that runs on it stays near its dense form."""
import importlib.util
import os

import pytest
import torch
from torch import nn

from rns_llm_amd import RNSCachedAttention

pytestmark = pytest.mark.gpu

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("cached_decode", os.path.join(ROOT, "examples", "cached_decode.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("kv_heads", [4, 2])
@torch.no_grad()
def test_layer_is_its_parts(backend, dtype, kv_heads):
    torch.manual_seed(3)
    heads, dim, features = 4, 64, 192
    linears = [nn.Linear(features, heads * dim), nn.Linear(features, kv_heads * dim), nn.Linear(features, kv_heads * dim),
               nn.Linear(heads * dim, features)]
    layer = RNSCachedAttention.from_linears(*(p.to(DEV, dtype) for p in linears), backend=backend, num_heads=heads,
                                            num_kv_heads=kv_heads)
    caches = [layer.create_cache(blocks=12, block_size=16) for _ in range(2)]
    table = torch.randperm(12, dtype=torch.int32).view(2, 6).to(DEV)
    for lengths, news in (([70, 33], [70, 33]), ([71, 34], [1, 1]), ([75, 35], [4, 1])):
        batch = backend.kv_batch(caches[0], table, lengths, query_lengths=news)
        x = torch.randn((sum(news), features), device=DEV, dtype=dtype)
        got = layer(x, caches[0], batch)
        q, k, v = layer.projection(x)
        rows = x.shape[0]
        backend.kv_append(caches[1], batch, k.reshape(rows, kv_heads, dim), v.reshape(rows, kv_heads, dim))
        out = backend.kv_attention(q.reshape(rows, heads, dim), caches[1], batch)
        assert torch.equal(got, layer.out_proj(out.reshape(rows, heads * dim)))


def test_layer_refuses(backend):
    def make(q=64, k=64, v=64, **options):
        parts = [nn.Linear(32, n).to(DEV) for n in (q, k, v)] + [nn.Linear(q, 32).to(DEV)]
        return RNSCachedAttention.from_linears(*parts, backend=backend, **options)

    for options in ({"num_heads": 3}, {"num_heads": 0}, {"num_heads": 4, "num_kv_heads": 3}, {"num_heads": 4, "num_kv_heads": 2},
                    {"v": 32, "num_heads": 2}):
        with pytest.raises(ValueError):
            make(**options)
    layer = make(num_heads=2)
    cache = layer.create_cache(blocks=2, block_size=16)
    batch = backend.kv_batch(cache, torch.zeros((1, 1), dtype=torch.int32, device=DEV), [3])
    with pytest.raises(ValueError, match="rows"):
        layer(torch.zeros((2, 32), device=DEV), cache, batch)


@torch.no_grad()
def test_decoding_stays_near_the_dense_model(backend):
    """Logits of every step against the dense model on the tokens taken: 8-bit
    activations and weights in four projections a block and 8-bit keys and values
    leave the mean error within 5 % of the mean logit, as the fused projections
    alone are held to.  Captured steps give what eager ones give."""
    ex = example()
    model = ex.build(layers=3, features=256, heads=4, vocabulary=1000, positions=256)
    model.use_rns(backend)
    gen = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 1000, (n,), generator=gen).to(DEV) for n in (1, 40, 77)]
    tokens, logits = ex.generate(model, backend, prompts, 12, 16)
    assert tokens.shape == (3, 12) and logits.isfinite().all()
    for i, prompt in enumerate(prompts):
        ids = torch.cat([prompt, tokens[i, :-1]])
        want = model.logits(model.dense(ids))[len(prompt) - 1:].float()
        off = (logits[i].float() - want).abs().mean()
        assert off < 0.05 * want.abs().mean()
    eager, eager_logits = ex.generate(model, backend, prompts, 12, 16, graph=False)
    assert torch.equal(tokens, eager) and torch.equal(logits, eager_logits)
