"""What the decoding loop's calls tell autograd, with a stand-in for the library on tensors in host memory."""
import pytest
import torch

from oracle import decode_oracle as do
from rns_llm_amd import HipRNSBackend, _native

CPU = torch.device("cpu")


class HostBackend(HipRNSBackend):
    """Rotations as the library makes them, past torch: through the addresses."""

    def __init__(self):  # no GPU here
        self._lib = _native.lib()

    def _rotated(self, rotary, positions, q, k, back, inplace):
        cos, sin = do.rotary_angles(rotary.frequencies, positions.tolist())
        outs = []
        for x in (q, k):
            if x is None:
                outs.append(None)
                continue
            y = do.rotate(x.detach(), cos, -sin if back else sin, rotary.interleaved, rotary.magnitude).to(x.dtype)
            if inplace:
                x.detach().numpy()[...] = y.numpy()
            outs.append(x if inplace else y)
        return tuple(outs)


def turning(backend, dim=8):
    return backend.create_rotary(device=CPU, rotary_dim=dim)


def made(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def test_calls_in_place_are_seen_by_autograd():
    """A value that an operation keeps for its backward pass and that is then turned in place: the pass raises."""
    b = HostBackend()
    rotary, positions = turning(b), torch.tensor([3, 4])
    q, k = made(2, 3, 8), made(2, 1, 8)
    for index in range(2):
        x = (q, k)[index]
        w = torch.ones_like(x).requires_grad_()
        kept = (w * x).sum()
        versions = q._version, k._version
        b.rotate(rotary, positions, q, k, inplace=True)
        assert q._version > versions[0] and k._version > versions[1]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
    # of a view, and under no_grad: the whole tensor's version is one
    wide = made(2, 40).requires_grad_()
    kept = wide.tanh()
    with torch.no_grad():
        b.rotate(rotary, positions, kept[:, 8:32].view(2, 3, 8), inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()
    # calls that leave their inputs as they are do not count as changes
    version = q._version
    b.rotate(rotary, positions, q, k)
    assert q._version == version
    with torch.inference_mode():  # tensors without a version
        b.rotate(rotary, positions, made(2, 3, 8), inplace=True)
