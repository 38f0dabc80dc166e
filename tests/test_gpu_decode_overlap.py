"""Rotations of queries and keys that lie in one tensor, some of them in place."""
import ctypes

import pytest
import torch

from rns_llm_amd import _native

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("first", ["q", "k"])
def test_one_in_place_the_other_elsewhere(backend, first):
    """Through the library: columns of one product, of which the first block is turned where it lies."""
    rotary = backend.create_rotary(device=DEV, rotary_dim=16)
    positions = torch.arange(3, 10, dtype=torch.int32, device=DEV)
    wide = torch.randn((7, 5 * 24 + 3 * 24 + 5), generator=torch.Generator().manual_seed(1)).half().to(DEV)
    held = wide.clone()
    q, k = wide[:, :120].view(7, 5, 24), wide[:, 120:192].view(7, 3, 24)
    want = backend.rotate(rotary, positions, q, k)
    outs = [torch.full((7, h, 24), 9.0, dtype=torch.float16, device=DEV) for h in (5, 3)]
    mine = first == "k"
    outs[mine] = (q, k)[mine]
    rows = _native.RotaryRowsStruct(7, *q.stride()[:2], *k.stride()[:2], *outs[0].stride()[:2], *outs[1].stride()[:2], 5, 3, 24,
                                    _native.FLOAT16, _native.INT32, 0)
    _native.check(_native.lib().rnsmx_rotate(rotary._ref, ctypes.addressof(rows), positions.data_ptr(), q.data_ptr(), k.data_ptr(),
                                             outs[0].data_ptr(), outs[1].data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert all(torch.equal(x, y) for x, y in zip(outs, want))
    held.view(-1).as_strided((7, (5, 3)[mine], 24), (held.stride(0), 24, 1), 120 * mine).copy_(want[mine])
    assert torch.equal(wide, held)  # nothing else has changed
