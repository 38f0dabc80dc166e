"""What the decoding loop's calls tell autograd, on the GPU."""
import pytest
import torch
from torch import nn
from torch.autograd import forward_ad

from rns_llm_amd import RNSCachedAttention

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


@pytest.mark.parametrize("gradients", [True, False])
def test_the_layer_leaves_its_projection_alone(backend, gradients):
    """What a hook keeps of the fused product stays as it was, and can be trained on."""
    torch.manual_seed(5)
    linears = [nn.Linear(m, n).to(DEV) for m, n in ((64, 128), (64, 64), (64, 64), (128, 64))]
    layer = RNSCachedAttention.from_linears(*linears, backend=backend, num_heads=2, num_kv_heads=1,
                                            rotary=backend.create_rotary(device=DEV, rotary_dim=64))
    kept = []
    layer.projection.combined.register_forward_hook(lambda module, inputs, output: kept.append(output))
    cache = layer.create_cache(blocks=2, block_size=16)
    batch = backend.kv_batch(cache, torch.tensor([[0, 1]], dtype=torch.int32, device=DEV), [5], query_lengths=[5])
    hidden = made(5, 64, seed=2)
    with torch.no_grad():
        want = layer.projection(hidden)[0].clone()
    kept.clear()
    with torch.set_grad_enabled(gradients):
        layer(hidden, cache, batch)
    head = torch.ones(128, device=DEV, requires_grad=True)
    assert torch.equal(kept[0][:, :128], want)
    (head * kept[0][:, :128].detach()).sum().backward()
    assert torch.equal(head.grad, want.sum(0))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_tangents_turn_with_their_values(backend, layout):
    """Forward mode: the rotation is linear, so a tangent is turned like a value, bit for bit, and a column of
    differences agrees; in reverse over it too."""
    rotary = backend.create_rotary(device=DEV, rotary_dim=24, layout=layout, magnitude=1.5)
    positions = torch.tensor([3, 700, 2 ** 20], device=DEV)
    q, k, tq, tk = (made(3, h, 40, seed=i) for i, h in enumerate((5, 2, 5, 2)))
    want, turned = (backend.rotate(rotary, positions, *x) for x in ((q, k), (tq, tk)))
    with forward_ad.dual_level():
        dq, dk = forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk)
        for args, tangents in (((dq, dk), turned), ((dq, k), (turned[0], None)), ((q, dk), (None, turned[1]))):
            for x, y, t in zip(backend.rotate(rotary, positions, *args), want, tangents):
                x = forward_ad.unpack_dual(x)
                assert torch.equal(x.primal, y) and (x.tangent is None if t is None else torch.equal(x.tangent, t))
        for args in ((dq, k), (q, dk)):
            with pytest.raises(ValueError, match="no gradient"):
                backend.rotate(rotary, positions, *args, inplace=True)
        leaf = q.clone().requires_grad_()
        y = backend.rotate(rotary, positions, forward_ad.make_dual(leaf, tq))
        gradient, = torch.autograd.grad((y ** 3).sum(), leaf)
        got = forward_ad.unpack_dual(gradient).tangent
    # the same values but for some four roundings of 2^-24 (powers, products, a rotation's sum), turned back: a
    # value of a pair by 2^-22 of both of its pair, each no larger than the row's largest
    x = q.clone().requires_grad_()
    g = 6 * want[0] * turned[0]
    product, = torch.autograd.grad(backend.rotate(rotary, positions, x), x, g)
    assert ((got - product).abs() <= 2.0 ** -22 * 2 * 1.5 * g.abs().amax(dim=2, keepdim=True)).all()


def test_calls_without_a_gradient_refuse_tangents(backend):
    """Their results would read as if they did not depend on what carries one; detached it carries none."""
    cache = backend.create_kv_cache(device=DEV, blocks=1, block_size=16, kv_heads=1, head_dim=64)
    batch = backend.kv_batch(cache, torch.zeros((2, 1), dtype=torch.int32, device=DEV), [3, 4])
    q, logits, scores = made(2, 3, 64), made(2, 3, 50), made(2, 3)
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for call in (lambda x: backend.kv_attention(x, cache, batch), lambda x: backend.beam_select(x[..., :50], scores, 2)[0],
                     lambda x: backend.beam_select(logits, x[..., 0], 2)[0]):
            with pytest.raises(RuntimeError, match="nor a tangent"):
                call(dual(q))
            assert torch.equal(call(dual(q).detach()), call(q))
