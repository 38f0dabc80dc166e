"""What the key/value cache's entry points keep from the kernels, on the host."""
import pytest
import torch

from rns_llm_amd import HipRNSBackend, _native

CPU = torch.device("cpu")


def backend():
    b = object.__new__(HipRNSBackend)  # no GPU here
    b._lib = _native.lib()
    return b


def cache(**changes):
    sizes = dict(device=CPU, blocks=4, block_size=16, kv_heads=2, head_dim=40)
    sizes.update(changes)
    return backend().create_kv_cache(**sizes)


def batch(c, **options):
    return backend().kv_batch(c, torch.zeros((2, 2), dtype=torch.int32), [20, 7], **options)


class NoLaunch:
    """The library without what starts a kernel."""

    rnsmx_kv_attention_workspace_bytes = staticmethod(lambda *args: 0)

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called with host addresses")


@pytest.mark.parametrize("call", [
    lambda b, c, x, q: b.kv_append(c, batch(c), x, x),
    lambda b, c, x, q: b.kv_read(c, batch(c), dtype=torch.float16),
    lambda b, c, x, q: b.kv_attention(q, c, batch(c)),
    lambda b, c, x, q: b.kv_attention(q, c, batch(c), mask=torch.zeros((1, 1, 20)), out=torch.empty_like(q)),
], ids=["append", "read", "attention", "masked"])
def test_caches_in_host_memory_reach_no_kernel(call, monkeypatch):
    """A kernel that reads a host address faults the GPU."""
    b = backend()
    b._lib = NoLaunch()
    monkeypatch.setattr(type(b), "_stream_of", staticmethod(lambda device: 0))
    x, q = (torch.zeros((2, n, 40), dtype=torch.float16) for n in (2, 4))
    for _ in range(2):
        with pytest.raises(ValueError, match="on the GPU"):
            call(b, cache(), x, q)


def test_a_batch_remembers_few_shapes(monkeypatch):
    """A mask that grows with the sequence is a new shape each step; what a batch
    keeps of them does not grow."""

    class Counts:
        rnsmx_kv_attention_workspace_bytes = staticmethod(lambda *args: 0)
        masks = []

        def rnsmx_kv_attention(self, cache, batch, query, *args):
            self.masks.append(_native.KVQueryStruct.from_address(query).mask_len)
            return 0

    b = backend()
    b._lib, b._stats = Counts(), {"kv_attention_calls": 0}
    monkeypatch.setattr(type(b), "_stream_of", staticmethod(lambda device: 0))
    monkeypatch.setattr(type(b), "_check_gpu", staticmethod(lambda cache: None))
    c = cache()
    step = backend().kv_batch(c, torch.zeros((2, 2), dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    q, most = torch.zeros((2, 4, 40), dtype=torch.float16), 0
    for n in range(1, 1000):
        b.kv_attention(q, c, step, mask=torch.zeros((1, 1, n)))
        b.kv_attention(q, c, step)
        most = max(most, len(step._checked))
    assert b._lib.masks == [m for n in range(1, 1000) for m in (n, 0)]
    assert most <= 64
