"""What the decoding loop's calls tell autograd, on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def made(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def test_calls_in_place_are_seen_by_autograd(backend):
    """A value that an operation keeps for its backward pass and that is then turned in place: the pass raises."""
    rotary, positions = backend.create_rotary(device=DEV, rotary_dim=8), torch.tensor([3, 4], device=DEV)
    q, k = made(2, 3, 8), made(2, 1, 8)
    for x in (q, k):
        w = torch.ones_like(x).requires_grad_()
        kept = (w * x).sum()
        backend.rotate(rotary, positions, q, k, inplace=True)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
    # one tensor, a view of what was kept
    wide = made(2, 40).requires_grad_()
    kept = wide.tanh()
    with torch.no_grad():
        backend.rotate(rotary, positions, kept[:, 8:32].view(2, 3, 8), inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()
