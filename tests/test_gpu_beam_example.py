"""The beam search example where its pool runs out of pages."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("beam_decode", os.path.join(ROOT, "examples", "beam_decode.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


class Short:
    """A backend with one call, counted from 0, whose step lacks a page: others that hold all free ones for its time."""

    def __init__(self, backend, call):
        self._backend, self._left, self.lacked = backend, call, 0

    def __getattr__(self, name):
        return getattr(self._backend, name)

    def kv_assign(self, pool, step, new=None):
        if self._left:
            self._left -= 1
            return self._backend.kv_assign(pool, step, new)
        self._left = -1  # no more
        kept = pool.free.clone()
        pool.free.zero_()
        self._backend.kv_assign(pool, step, new)
        pool.free.copy_(kept)
        self.lacked = int(step.missing)


@pytest.mark.parametrize("call", [0, 1, 17])
@torch.no_grad()
def test_a_step_that_lacks_pages(backend, call):
    """The prompts', the first step's or a later one's, after which there is room again."""
    ex = example()
    model = ex.build(layers=1, features=256, heads=4, kv_heads=2, vocabulary=300)
    model.use_rns(backend)
    # prompts that end with their page: beams need one at the first step, and again 16 later
    prompts = [torch.arange(16, device=DEV), torch.arange(16, device=DEV) + 9]
    short = Short(backend, call)
    with pytest.raises(RuntimeError, match="lacked"):
        ex.search(model, short, prompts, 2, 30, 16, 299, graph=False)
    assert short.lacked > 0
