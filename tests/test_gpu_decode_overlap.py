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


def grids(gen):
    """Tensors whose heads or rows lie among each other's and share no value: name, all of the memory, q, k."""
    def made(*shape):
        return torch.randn(shape, generator=gen).half().to(DEV)

    x = made(7, 9, 24)
    yield "every other head of nine", x, x[:, 0::2], x[:, 1::2]
    yield "every third, of fewer", x, x[:, 0::3], x[:, 1:8:3]
    x = made(7, 4 * 48 + 5)  # a head's query and key side by side, rows that are no multiple of them
    yield "pairs in padded rows", x, *x[:, :192].view(7, 4, 2, 24).unbind(2)
    x = made(7, 3 * 72 + 8)  # three query heads to a key head, of which one is taken
    yield "groups in padded rows", x, x[:, :216].view(7, 3, 72)[..., 24:48], x[:, :216].view(7, 3, 72)[..., 48:]
    x = made(7, 10, 24)
    yield "other strides of heads", x, x[:, 0::4], x[:, 1::2]
    x = made(9, 7, 24).transpose(0, 1)
    yield "heads first", x, x[:, 0::2], x[:, 1::2]


@pytest.mark.parametrize("rows", [7, 1])
def test_heads_among_each_other(backend, rows):
    """They share no value, so they are turned in place, and what lies between them stays."""
    rotary = backend.create_rotary(device=DEV, rotary_dim=16)
    positions = torch.arange(3, 3 + rows, dtype=torch.int32, device=DEV)
    for name, x, q, k in grids(torch.Generator().manual_seed(2)):
        q, k = q[:rows], k[:rows]
        for a, b in ((q, k), (k, q)):
            want = backend.rotate(rotary, positions, a.clone(), b.clone())
            held = x.clone()
            backend.rotate(rotary, positions, a, b, inplace=True)
            assert torch.equal(a, want[0]) and torch.equal(b, want[1]), name
            after = x.clone()
            rest = []
            for whole in (held, after):  # but for the turned values
                x.copy_(whole)
                a.zero_()
                b.zero_()
                rest.append(x.clone())
            assert torch.equal(*rest), name
            x.copy_(after)


def test_heads_that_share_values(backend):
    """Some head of the one a part of a head of the other, in this row or in another."""
    rotary = backend.create_rotary(device=DEV, rotary_dim=16)
    positions = torch.arange(7, device=DEV)
    x = torch.zeros((9, 10, 24), dtype=torch.float16, device=DEV)
    flat = x.view(9, 240)
    for q, k in ((x[:7, 0::2], x[:7, 2:9:3]), (x[:7, 0::2], x[2:, 4:5]), (x[:7, 1::3], x[:7, 0::2]),
                 (x[:7, 0::2], flat[:7, 5:5 + 24 * 4].view(7, 4, 24)), (x[:7, 8:], flat.view(-1)[240 - 23:][:7 * 240].view(7, 10, 24)[:, :1])):
        for a, b in ((q, k), (k, q)):
            with pytest.raises(ValueError, match="share values"):
                backend.rotate(rotary, positions, a, b, inplace=True)
    assert not x.any()
