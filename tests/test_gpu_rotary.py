"""Rotary positions on the GPU against angles of whole-number turns in 64 bits."""
import math

import pytest
import torch

from oracle import decode_oracle as do

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def reach(x, pairs, interleaved):
    """|u| + |v| of each value's pair; 0 of those that are in none."""
    u = x.double().abs()
    total = torch.zeros_like(u)
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    total[..., first] = total[..., second] = u[..., first] + u[..., second]
    return total


def bound(x, want, pairs, interleaved, magnitude=1.0):
    """What a rotated value may be off by.  A cosine or sine: 2^-32 of a turn cut off (2 pi 2^-32 <
    2^-29), an eighth of a turn converted to float32 (pi / 4 2^-24), the functions themselves 4 units of
    2^-24, and the magnitude's product 2^-24: below 6 2^-24.  The two products and their sum: 2^-24 each of
    what they are at most.  Together below 2^-20 (|u| + |v|) magnitude; then the output's rounding."""
    least = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[x.dtype]  # half of the smallest float16
    return reach(x, pairs, interleaved) * 2.0 ** -20 * magnitude + want.abs() * torch.finfo(x.dtype).eps / 2 * (1 + 2.0 ** -20) + least


def check(got, x, cos, sin, pairs, interleaved, magnitude=1.0):
    want = do.rotate(x.cpu(), cos, sin, interleaved, magnitude)
    off = (got.double().cpu() - want).abs()
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    assert (off <= bound(x.cpu(), want, pairs, interleaved, magnitude)).all(), off.max()
    assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])


SHAPES = [  # rows, q heads, k heads (0: none), dim, rotary dim
    (1, 1, 1, 2, 2), (3, 5, 0, 7, 6), (17, 12, 12, 64, 64), (5, 32, 8, 128, 128), (2, 7, 7, 65, 64), (9, 4, 2, 80, 32),
    (300, 3, 1, 256, 250), (1025, 2, 1, 40, 20), (8200, 1, 1, 16, 16), (33, 1, 3, 1024, 1024), (2100, 1, 0, 8, 8), (63, 9, 2, 96, 16),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotation(backend, shape, layout, dtype):
    rows, q_heads, k_heads, dim, part = shape
    gen = torch.Generator().manual_seed(rows + dim)
    q, k = (torch.randn((rows, h, dim), generator=gen).to(dtype).to(DEV) for h in (q_heads, k_heads))
    positions = torch.randint(0, 5000, (rows,), generator=gen, dtype=torch.int32)
    rotary = backend.create_rotary(device=DEV, rotary_dim=part, layout=layout, magnitude=1.25)
    got = backend.rotate(rotary, positions.to(DEV), q, k if k_heads else None)
    angles = do.rotary_angles(rotary.frequencies, positions)
    for y, x in zip(got if k_heads else (got,), (q, k)):
        check(y, x, *angles, part // 2, layout == "interleaved", 1.25)
    # in place: the same bits
    held = [x.clone() for x in (q, k)]
    out = backend.rotate(rotary, positions.to(DEV), held[0], held[1] if k_heads else None, inplace=True)
    for y, x, z in zip(got if k_heads else (got,), out if k_heads else (out,), held):
        assert x is z and torch.equal(x, y)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64], ids=str)
def test_far_positions(backend, kind):
    """No position is too far, whole ones of 64 bits and negative ones among them."""
    far = [0, 1, -1, 131071, 10 ** 6 + 7, 2 ** 30, 2 ** 31 - 1, -2 ** 31]
    if kind == torch.int64:
        far += [2 ** 40 + 3, 2 ** 53 + 1, -2 ** 62, 2 ** 63 - 1]
    rotary = backend.create_rotary(device=DEV, rotary_dim=128)
    x = torch.randn((len(far), 2, 128), generator=torch.Generator().manual_seed(1)).to(DEV)
    got = backend.rotate(rotary, torch.tensor(far, dtype=kind, device=DEV), x)
    # a step is off by 2^-65 turns a position: seen from 2^40 on, so the reference takes the steps
    # themselves there
    near = [i for i, p in enumerate(far) if abs(p) < 2 ** 33]
    cos, sin = do.rotary_angles(rotary.frequencies, [far[i] for i in near])
    check(got[near], x[near], cos, sin, 64, False)
    turns = torch.tensor([[(p * int(s) % 2 ** 64) / 2 ** 64 for s in rotary.steps.tolist()] for p in far], dtype=torch.float64)
    angle = turns.view(len(far), 1, -1) * (2 * math.pi)
    check(got, x, angle.cos(), angle.sin(), 64, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_strides(backend, dtype):
    """Column blocks of a product, heads before rows, values apart, one head for all, odd offsets."""
    gen = torch.Generator().manual_seed(2)
    rotary = backend.create_rotary(device=DEV, rotary_dim=16)
    positions = torch.arange(50, 57, device=DEV)
    wide = torch.randn((7, 12 * 24 + 1), generator=gen).to(dtype).to(DEV)
    forms = [wide[:, :5 * 24].view(7, 5, 24), wide[:, 1:5 * 24 + 1].as_strided((7, 5, 24), (wide.stride(0), 24, 1), 1),
             torch.randn((5, 7, 24), generator=gen).to(dtype).to(DEV).transpose(0, 1),
             torch.randn((7, 24, 5), generator=gen).to(dtype).to(DEV).transpose(1, 2),
             torch.randn((7, 1, 24), generator=gen).to(dtype).to(DEV).expand(7, 5, 24),
             torch.randn((1, 5, 24), generator=gen).to(dtype).to(DEV).expand(7, 5, 24)]
    for x in forms:
        want = backend.rotate(rotary, positions, x.contiguous())
        q, k = backend.rotate(rotary, positions, x, x[:, :3])
        assert torch.equal(q, want) and torch.equal(k, want[:, :3])
    # q and k of one product in place, the columns after them as they were
    q, k, rest = wide[:, :96].view(7, 4, 24), wide[:, 96:144].view(7, 2, 24), wide[:, 144:].clone()
    want = backend.rotate(rotary, positions, q.clone(), k.clone())
    backend.rotate(rotary, positions, q, k, inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(wide[:, 144:], rest)
    # of one tensor with the heads first, with rows of several products side by side, heads in turn
    for make in (lambda: torch.randn((9, 7, 24), generator=gen).to(dtype).to(DEV).transpose(0, 1),
                 lambda: torch.randn((7, 2, 9, 24), generator=gen).to(dtype).to(DEV)[:, 1],
                 lambda: torch.randn((7, 9, 48), generator=gen).to(dtype).to(DEV)):
        x = make()
        pairs = [(x[:, 2:6], x[:, 6:8]), (x[:, 6:8], x[:, :5])] if x.shape[2] == 24 else [(x[..., :24], x[..., 24:]), (x[..., 24:], x[..., :24])]
        for q, k in pairs:
            want = backend.rotate(rotary, positions, q.clone(), k.clone())
            backend.rotate(rotary, positions, q, k, inplace=True)
            assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    for q, k in ((x, x), (x[:, :5, :24], x[:, 4:, :24]), (x[..., :24], x[..., 8:32])):
        with pytest.raises(ValueError, match="share values"):
            backend.rotate(rotary, positions, q, k, inplace=True)
    assert torch.equal(backend.rotate(rotary, torch.arange(100, 114, device=DEV)[::2], wide[:, :96].view(7, 4, 24)),
                       backend.rotate(rotary, torch.arange(100, 114, 2, device=DEV), wide[:, :96].view(7, 4, 24)))


def test_values_that_are_not_finite(backend):
    """They reach their pair alone."""
    rotary = backend.create_rotary(device=DEV, rotary_dim=8)
    x = torch.ones((2, 2, 10), device=DEV)
    x[0, 0, 1], x[0, 1, 9] = math.nan, math.inf
    got = backend.rotate(rotary, torch.tensor([3, 4], device=DEV), x)
    odd = ~torch.isfinite(got)
    assert odd.nonzero().tolist() == [[0, 0, 1], [0, 0, 5], [0, 1, 9]]


@pytest.mark.parametrize("rows,q_heads,k_heads", [(0, 2, 1), (3, 0, 1), (3, 2, 0), (0, 0, 0)])
def test_nothing_to_turn(backend, rows, q_heads, k_heads):
    rotary = backend.create_rotary(device=DEV, rotary_dim=8)
    q, k = (torch.ones((rows, h, 8), device=DEV) for h in (q_heads, k_heads))
    got = backend.rotate(rotary, torch.zeros(rows, dtype=torch.int32, device=DEV), q, k)
    assert torch.equal(got[0], q) and torch.equal(got[1], k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradients(backend, layout, dtype):
    """Against the formula, and, the rotation being linear, against differences: <R x, g> = <x, R' g>."""
    gen = torch.Generator().manual_seed(4)
    rotary = backend.create_rotary(device=DEV, rotary_dim=40, layout=layout, magnitude=0.75)
    positions = torch.randint(0, 4000, (29,), generator=gen).to(DEV)
    q, k = (torch.randn((29, h, 48), generator=gen).to(dtype).to(DEV).requires_grad_() for h in (6, 2))
    gq, gk = (torch.randn((29, h, 48), generator=gen).to(dtype).to(DEV) for h in (6, 2))
    out = backend.rotate(rotary, positions, q, k)
    grads = torch.autograd.grad(out, (q, k), (gq, gk))
    cos, sin = do.rotary_angles(rotary.frequencies, positions.tolist())
    for got, g in zip(grads, (gq, gk)):
        check(got, g, cos, -sin, 20, layout == "interleaved", 0.75)
    if dtype == torch.float32:
        far = lambda x: reach(x, 20, layout == "interleaved")  # noqa: E731
        for x, y, g, d in zip((q, k), out, (gq, gk), grads):
            x, y = x.detach(), y.detach()
            off = (y.double() * g.double()).sum() - (x.double() * d.double()).sum()
            assert off.abs() <= 2.0 ** -20 * ((far(x) * g.abs()).sum() + (far(g) * x.abs()).sum())
            h = torch.randn(x.shape, generator=gen).to(DEV)
            moved = backend.rotate(rotary, positions, x + h).double() - y.double()
            off = (moved * g.double()).sum() - ((x + h).double() - x.double()).mul(d.double()).sum()
            assert off.abs() <= 2.0 ** -20 * (((far(x + h) + far(x)) * g.abs()).sum() + (far(g) * h.abs()).sum() * (1 + 2.0 ** -10))


def test_gradients_of_parts(backend):
    """Of one output alone, of broadcast inputs, of gradients, and none where none are asked for."""
    gen = torch.Generator().manual_seed(5)
    rotary = backend.create_rotary(device=DEV, rotary_dim=8)
    positions = torch.arange(5, device=DEV)
    q, k = (torch.randn((5, h, 8), generator=gen).to(DEV).requires_grad_() for h in (3, 2))
    g = torch.randn((5, 3, 8), generator=gen).to(DEV)
    full = torch.autograd.grad(backend.rotate(rotary, positions, q, k), (q, k), (g, g[:, :2]))
    assert torch.equal(torch.autograd.grad(backend.rotate(rotary, positions, q, k)[0], q, g)[0], full[0])
    assert torch.equal(torch.autograd.grad(backend.rotate(rotary, positions, q, k)[1], k, g[:, :2])[0], full[1])
    assert torch.equal(torch.autograd.grad(backend.rotate(rotary, positions, q), q, g)[0], full[0])
    plain = torch.randn((5, 3, 8), generator=gen).to(DEV)
    assert torch.equal(torch.autograd.grad(backend.rotate(rotary, positions, plain, k)[1], k, g[:, :2])[0], full[1])
    one = torch.randn((5, 1, 8), generator=gen).to(DEV).requires_grad_()
    got, = torch.autograd.grad(backend.rotate(rotary, positions, one.expand(5, 3, 8)), one, g)
    assert torch.allclose(got, full[0].sum(dim=1, keepdim=True), atol=1e-5)
    got, = torch.autograd.grad(backend.rotate(rotary, positions, q).sum(), q)  # a gradient that is broadcast
    assert torch.equal(got, torch.autograd.grad(backend.rotate(rotary, positions, q), q, torch.ones_like(g))[0])
    # the gradient's gradient: y = R x, d = R' (2 y), so d's gradient along v is 2 R' R v = 2 v
    y = backend.rotate(rotary, positions, q)
    d, = torch.autograd.grad((y * y).sum(), q, create_graph=True)
    again, = torch.autograd.grad(d, q, g)
    assert torch.allclose(again, 2 * g, atol=1e-5)
    with torch.no_grad():
        assert not backend.rotate(rotary, positions, q).requires_grad
    moved = positions.clone()
    y = backend.rotate(rotary, moved, q)
    moved.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_streams_and_graphs(backend):
    """On a stream of its own, and captured: replays turn by the positions of the moment."""
    gen = torch.Generator().manual_seed(6)
    rotary = backend.create_rotary(device=DEV, rotary_dim=64, layout="interleaved")
    q, k = (torch.randn((4, h, 64), generator=gen).half().to(DEV) for h in (12, 3))
    positions = torch.tensor([5, 0, 900, 77], dtype=torch.int32, device=DEV)
    want = backend.rotate(rotary, positions, q, k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = backend.rotate(rotary, positions, q, k)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            positions.add_(1)
            held = backend.rotate(rotary, positions, q, k)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for _ in range(3):
        graph.replay()
        want = backend.rotate(rotary, positions, q, k)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    assert positions.tolist() == [8, 3, 903, 80]


def test_captured_gradients(backend):
    """Forward and backward in one graph; every replay's gradients are those of the moment's positions."""
    gen = torch.Generator().manual_seed(8)
    rotary = backend.create_rotary(device=DEV, rotary_dim=32)
    q, k, gq, gk = (torch.randn((5, h, 40), generator=gen).to(DEV) for h in (6, 2, 6, 2))
    positions = torch.tensor([3, 0, 700, 2 ** 20, 12], dtype=torch.int64, device=DEV)

    def gradients():
        leaves = [x.detach().requires_grad_() for x in (q, k)]
        return torch.autograd.grad(backend.rotate(rotary, positions, *leaves), leaves, (gq, gk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gradients()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            positions.add_(1)
            held = gradients()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        graph.replay()
        want = gradients()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        cos, sin = do.rotary_angles(rotary.frequencies, positions.cpu())
        for got, g in zip(held, (gq, gk)):
            check(got, g, cos, -sin, 16, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("part", [128, 96, 16])
def test_past_the_caches(backend, part, layout, dtype):
    """More than the caches hold: the same bits as in small calls, one of which is checked."""
    rows, heads, dim = 264000 // (4 if dtype == torch.float32 else 2) // 8, 33, 128
    gen = torch.Generator(device=DEV).manual_seed(part)
    q = torch.randn((rows, heads - 1, dim), generator=gen, device=DEV, dtype=torch.float32).to(dtype)
    k = torch.randn((rows, 1, dim), generator=gen, device=DEV, dtype=torch.float32).to(dtype)
    assert 2 * (q.numel() + k.numel()) * q.element_size() > 256 << 20
    positions = torch.randint(0, 9000, (rows,), generator=gen, device=DEV, dtype=torch.int32)
    rotary = backend.create_rotary(device=DEV, rotary_dim=part, layout=layout)
    got = backend.rotate(rotary, positions, q, k)
    for a in range(0, rows, 2000):
        want = backend.rotate(rotary, positions[a:a + 2000], q[a:a + 2000], k[a:a + 2000])
        assert all(torch.equal(x[a:a + 2000], y) for x, y in zip(got, want))
    n = rows - 9
    angles = do.rotary_angles(rotary.frequencies, positions[n:].cpu())
    check(got[0][n:], q[n:], *angles, part // 2, layout == "interleaved")
    again = [x.clone() for x in (q, k)]
    backend.rotate(rotary, positions, *again, inplace=True)
    assert all(torch.equal(x, y) for x, y in zip(again, got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_every_size(backend, layout, dtype):
    """Every head dimension and part of it up to 42, wherever rows begin, apart and in place; what is not turned
    is copied, what lies between the rows stays."""
    gen = torch.Generator().manual_seed(17)
    for dim in range(2, 43):
        part = 2 * (1 + (dim * 7) % (dim // 2))
        wide = torch.randn((5, 3 * dim + 3), generator=gen).to(dtype).to(DEV)
        positions = torch.tensor([0, 3, 9, 1000, 77], dtype=torch.int64, device=DEV)
        rotary = backend.create_rotary(device=DEV, rotary_dim=part, layout=layout)
        angles = do.rotary_angles(rotary.frequencies, positions.cpu())
        x = wide[:, 1:1 + 3 * dim].view(5, 3, dim)
        got = backend.rotate(rotary, positions, x)
        check(got, x, *angles, part // 2, layout == "interleaved")
        held = wide.clone()
        backend.rotate(rotary, positions, x, inplace=True)
        assert torch.equal(x, got)
        assert torch.equal(wide[:, :1], held[:, :1]) and torch.equal(wide[:, 1 + 3 * dim:], held[:, 1 + 3 * dim:])
