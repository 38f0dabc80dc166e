"""What the decoding loop's calls tell autograd, with a stand-in for the library on tensors in host memory."""
from collections import Counter

import pytest
import torch
from torch import nn
from torch.autograd import forward_ad

from oracle import decode_oracle as do
from rns_llm_amd import HipRNSBackend, KVCache, RNSCachedAttention, _native

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
            plain = torch.from_numpy(x.detach().numpy().copy())  # a tangent stays behind
            y = do.rotate(plain, cos, -sin if back else sin, rotary.interleaved, rotary.magnitude).to(x.dtype)
            if inplace:
                x.detach().numpy()[...] = y.numpy()
            outs.append(x if inplace else y)
        return tuple(outs)

    def kv_slots(self, pages, batch):
        return torch.arange(batch.rows, dtype=torch.int32), None

    def kv_append(self, cache, batch, k, v):
        pass

    def kv_attention(self, q, cache, batch, **options):
        return q.clone()



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


class Projection(nn.Module):
    split_sizes = (16, 8, 8)

    def forward(self, hidden):
        return hidden.split(self.split_sizes, dim=-1)


class Batch:
    rows = 5


@pytest.mark.parametrize("gradients", [True, False])
def test_the_layer_leaves_its_projection_alone(gradients):
    """What a hook keeps of the projection stays as it was, and can be trained on."""
    b = HostBackend()
    layer = RNSCachedAttention(Projection(), nn.Identity(), backend=b, num_heads=2, num_kv_heads=1, rotary=turning(b))
    kept = []
    layer.projection.register_forward_hook(lambda module, inputs, outputs: kept.extend(outputs))
    hidden = made(5, 32, seed=1)
    before = hidden.clone()
    head = torch.ones(16, requires_grad=True)
    with torch.set_grad_enabled(gradients):
        out = layer(hidden, None, Batch())
    assert not torch.equal(out, before[:, :16]) and torch.equal(hidden, before)
    assert torch.equal(torch.cat(kept, dim=1), before)
    (head * kept[0]).sum().backward()
    assert torch.equal(head.grad, before[:, :16].sum(0))


@pytest.mark.parametrize("gradients", [True, False])
def test_tangents_turn_with_their_values(gradients):
    """Forward mode: of queries, of keys, of both; the rotation is linear."""
    b = HostBackend()
    rotary, positions = turning(b, 6), torch.tensor([3, 700])
    q, k, tq, tk = (made(2, h, 8, seed=i) for i, h in enumerate((3, 1, 3, 1)))
    want = b.rotate(rotary, positions, q, k)
    turned = b.rotate(rotary, positions, tq, tk)
    with forward_ad.dual_level(), torch.set_grad_enabled(gradients):
        dq, dk = forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk)
        for args, tangents in (((dq, dk), turned), ((dq, k), (turned[0], None)), ((q, dk), (None, turned[1])), ((q, k), (None, None))):
            got = [forward_ad.unpack_dual(x) for x in b.rotate(rotary, positions, *args)]
            for x, y, t in zip(got, want, tangents):
                assert torch.equal(x.primal, y) and (x.tangent is None if t is None else torch.equal(x.tangent, t))
        assert torch.equal(forward_ad.unpack_dual(b.rotate(rotary, positions, dk)).tangent, turned[1])
        for args in ((dq, k), (q, dk), (dq, None)):
            with pytest.raises(ValueError, match="no gradient"):
                b.rotate(rotary, positions, *args, inplace=True)
        assert torch.equal(b.rotate(rotary, positions, q.clone(), inplace=True), want[0])


def test_tangents_and_gradients_together():
    """Forward over reverse: of the sum of y^3, y = R x, the Hessian's product with a direction."""
    b = HostBackend()
    rotary, positions = turning(b), torch.tensor([3, 70])
    x, t = made(2, 3, 8, seed=1), made(2, 3, 8, seed=2)

    def loss(y):
        return (y ** 3).sum()

    with forward_ad.dual_level():
        leaf = x.clone().requires_grad_()
        gradient, = torch.autograd.grad(loss(b.rotate(rotary, positions, forward_ad.make_dual(leaf, t))), leaf)
        got = forward_ad.unpack_dual(gradient).tangent
    # R' (6 y R t)
    y, turned = b.rotate(rotary, positions, x), b.rotate(rotary, positions, t)
    g = 6 * y * turned
    want = b._rotated(rotary, positions, g, None, True, False)[0]
    # some four roundings of 2^-24 before both values of a pair are turned, one after
    assert ((got - want).abs() <= 2.0 ** -22 * 2 * g.abs().amax(dim=2, keepdim=True)).all()
    # a tangent that itself has a gradient
    with forward_ad.dual_level():
        direction = t.clone().requires_grad_()
        out = forward_ad.unpack_dual(b.rotate(rotary, positions, forward_ad.make_dual(x, direction))).tangent
        got, = torch.autograd.grad(out, direction, y)
    assert ((got - x).abs() <= 2.0 ** -22 * 2 * x.abs().amax(dim=2, keepdim=True)).all()  # R' R x


class NoLibrary:
    """Calls that succeed and do nothing, sizes that are small."""

    def __getattr__(self, name):
        return lambda *args: 0 if name.startswith("rnsmx_kv_attention") else 64


class CallsBackend(HostBackend):
    """Selection and attention as far as the call, whose outputs nothing is written to."""

    def __init__(self):
        self._lib, self._beam_checked, self._stats = NoLibrary(), {}, Counter()

    kv_attention = HipRNSBackend.kv_attention

    @staticmethod
    def _plain_beams(logits, scores, k, finished, end_token):
        return logits, scores, finished

    def _kv_scratch_for(self, need, device, stream):
        return torch.zeros(need, dtype=torch.uint8)

    def _on_device(self, device, call, *args):
        pass

    _stream_of = staticmethod(lambda device: 0)
    _check_gpu = staticmethod(lambda cache: None)


def test_calls_without_a_gradient_refuse_tangents():
    """Their results would read as if they did not depend on what carries one."""
    b = CallsBackend()
    cache = KVCache(None, None, made(1, 1, 2), 1, 16, 1, 8, CPU, _shape=(1, 16, 8, CPU))
    batch = b.kv_batch(cache, torch.zeros((2, 1), dtype=torch.int32), [3, 4])
    q, mask, logits, scores = made(2, 3, 8), made(2, 3, 16), made(2, 3, 5), made(2, 3)
    assert b.kv_attention(q, cache, batch, mask=mask).shape == q.shape and b.beam_select(logits, scores, 2)[0].shape == (2, 2)
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for gradients in (True, False):
            with torch.set_grad_enabled(gradients):
                for call in (lambda: b.kv_attention(dual(q), cache, batch), lambda: b.kv_attention(q, cache, batch, mask=dual(mask)),
                             lambda: b.beam_select(dual(logits), scores, 2), lambda: b.beam_select(logits, dual(scores), 2)):
                    with pytest.raises(RuntimeError, match="nor a tangent"):
                        call()
        # numbers alone
        assert b.kv_attention(dual(q), cache, batch, out=torch.empty_like(q)).shape == q.shape
        assert b.beam_select(logits, scores, 2)[0].shape == (2, 2)


def test_a_given_output_is_seen_by_autograd():
    """What an operation keeps of an attention's result, and the next call writes over: the backward pass raises."""
    b = CallsBackend()
    cache = KVCache(None, None, made(1, 1, 2), 1, 16, 1, 8, CPU, _shape=(1, 16, 8, CPU))
    batch = b.kv_batch(cache, torch.zeros((2, 1), dtype=torch.int32), [3, 4])
    q, out = made(2, 3, 8), made(2, 3, 8)
    w = torch.ones_like(out).requires_grad_()
    kept = (w * b.kv_attention(q, cache, batch, out=out)).sum()
    b.kv_attention(q, cache, batch, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
