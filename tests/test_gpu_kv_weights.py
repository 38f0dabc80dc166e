"""Softmax weights far below a row's largest, where they are what its result is
made of: a first token, say, that has nearly all the weight and next to no value."""
import math

import pytest
import torch

from kv_plans import plan_of
from test_gpu_kv import DEV, MANY, ROUND, TYPES, World, bound

pytestmark = pytest.mark.gpu


def most_off(dtype, out, spread, length, largest):
    """What each element may be off by.  Scores of up to 64 in powers of two have
    24 bits, a few times over on the way to a weight: less than 2^-15 of it.  A
    weight has 11 bits, or 22 in two halves (float32), and float16's spacing of
    2^-24 ends both where the largest weight is 2^10 or more: 2^-35 of it, and 2^11
    less for the second half; `largest`: the largest value of the sequence, which
    the largest weight goes with."""
    weights, ends = (2.0 ** -21, 2.0 ** -46) if dtype == torch.float32 else (2.0 ** -11, 2.0 ** -35)
    return ROUND[dtype] * out.abs() + (weights + 2.0 ** -15) * spread + length * ends * largest + 1e-30


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("gap", [10, 16])
@pytest.mark.parametrize("length,at,rows,dim,idle", [
    (1100, 0, 1, 64, 0), (1100, 700, 3, 128, 0), (6000, 3, 1, 128, 0), (6000, 5990, 2, 40, 0),
    (700, 0, 60, 64, MANY), (700, 333, 60, 128, MANY), (1500, 20, 60, 160, MANY), (3000, 1, 600, 64, 8),
    (700, 0, 130, 64, MANY), (700, 333, 130, 128, MANY), (1500, 20, 130, 160, MANY), (3000, 1, 640, 64, 18), (3000, 2900, 640, 40, 18),
])
@pytest.mark.parametrize("masked", [False, True])
def test_small_weights_count(backend, dtype, gap, length, at, rows, dim, idle, masked):
    w = World(backend, lengths=[length], heads=1, dim=dim, page=16, seed=gap + dim, idle=idle)
    q = torch.randn((1, 1, dim), generator=w.gen) + 0.02 * torch.randn((rows, 1, dim), generator=w.gen)
    k, v = (torch.randn((length, 1, dim), generator=w.gen) for _ in range(2))
    # its score: some four deviations for the largest of the others, and the gap
    k[at] = (4 + gap) * math.sqrt(dim) * q[0] / (q[0] ** 2).sum()
    v[at] = 0.01 * v[at]
    v[at, :, ::2] = 0
    w.append([length], torch.float32, k=k, v=v)
    news, q = [rows], q.to(dtype)
    mask = torch.zeros((1, 1, length)) if masked else None
    kernel = plan_of(w.cache, w.batch(news), 1, dtype, masked=masked)
    assert kernel.tile_rows == (128 if rows in (130, 640) else 16) and (kernel.splits > 1) == (length == 6000 or rows == 640)
    got = w.backend.kv_attention(q.to(DEV), w.cache, w.batch(news), mask=None if mask is None else mask.to(DEV)).cpu().double()
    some = [0, rows - 1, rows // 2]
    out, spread, _ = (x[some] for x in w.want(q, news))
    most = most_off(dtype, out, spread, length, v.abs().max())
    off = (got[some] - out).abs()
    assert (off <= most).all(), f"off by {float((off / most).max()):.3g} of the bound, {float(off.norm() / out.norm()):.3g} of the result"


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,group,dim", [(150, 1, 128), (60, 4, 64), (150, 1, 256)])
@pytest.mark.parametrize("window", [None, 2500])
def test_tiles_of_16_rows_are_split(backend, dtype, rows, group, dim, window):
    """Several tiles of 16 rows to a sequence and several splits to a tile, beside
    sequences that need fewer of either."""
    lengths, news = [4100, 130, 2700, 0], [rows, min(130, rows), rows // 2, 1]
    w = World(backend, lengths=lengths, heads=1, dim=dim, page=16, seed=dim)
    w.append(lengths, dtype)
    kernel = plan_of(w.cache, w.batch(news), group, dtype, window=window)
    assert kernel.tile_rows == 16 and kernel.row_tiles > 1 and kernel.splits > 1
    w.check(news, dtype, group, **({} if window is None else {"window": window}))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("mask_dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,idle,dim", [(2, 0, 64), (50, MANY, 64), (50, MANY, 128), (20, 0, 200)])
@pytest.mark.parametrize("heads_apart", [False, True])
def test_the_lowest_value_hides_as_minus_infinity_does(backend, dtype, mask_dtype, rows, idle, dim, heads_apart):
    """Within the bound of the same call without a mask: tokens at the type's lowest
    value have no weight where a row has others; where it has none, what it sees
    weighs the same."""
    lengths = [100, 61]
    w = World(backend, lengths=lengths, heads=2, dim=dim, page=16, seed=35, idle=idle)
    w.append(lengths, dtype)
    news = [rows, rows]
    q = torch.randn((2 * rows, 4, dim), generator=w.gen).to(dtype)
    low = torch.rand((2 * rows, 4 if heads_apart else 1, 100), generator=w.gen) < 0.4
    low[1::4] = True
    low[3::8] = False
    kernel = plan_of(w.cache, w.batch(news), 4, dtype, masked=True)
    assert kernel.tile_rows == (128 if idle else 16)
    mask = torch.where(low, torch.finfo(mask_dtype).min, 0.0).to(mask_dtype)
    got = w.backend.kv_attention(q.to(DEV), w.cache, w.batch(news), mask=mask.to(DEV)).cpu().double()
    out, spread, reach = w.want(q, news, mask=~low)
    at = 0
    for i, n in enumerate(lengths):
        k, _ = w.k.values(w.table[i], n)
        v, _ = w.v.values(w.table[i], n)
        v = v.repeat_interleave(2, dim=1)
        for r in range(rows):
            seen = n - rows + r + 1
            full = low[at + r].expand(4, 100)[:, :seen].all(dim=1)  # heads whose tokens are all at the lowest
            out[at + r, full] = v[:seen].mean(dim=0)[full]
            spread[at + r, full] = v[:seen].abs().mean(dim=0)[full]
            reach[at + r, full] = 0.0
        at += rows
    most = bound(dtype, out, spread, reach, dim, 100, None)
    assert ((got - out).abs() <= most).all(), f"off by {float(((got - out).abs() / most).max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 13, 2.0 ** 15, 2.0 ** 30])
@pytest.mark.parametrize("lengths,rows,dim,idle,masked", [
    ([300, 70], 1, 64, 0, False), ([300, 70], 3, 128, 0, True), ([4100, 1], 1, 128, 0, False), ([300, 70], 70, 64, MANY, False),
    ([300, 170], 170, 128, MANY, False), ([300, 70], 70, 128, MANY, True), ([1100, 700], 20, 256, 0, False),
])
def test_scores_of_any_size(backend, dtype, size, lengths, rows, dim, idle, masked):
    """Scores of 2^16 to 2^60, each one that float32 holds: a row's result is the
    value of its largest, which is ahead of the next by far."""
    w = World(backend, lengths=lengths, heads=2, dim=dim, page=16, seed=41, idle=idle)
    total = sum(lengths)
    k, v = (torch.randn((total, 2, dim), generator=w.gen) for _ in range(2))
    v = v * 2.0 ** torch.randint(-9, 9, (total, 1, 1), generator=w.gen)  # pages of different scales
    w.append(lengths, torch.float32, k=size * k, v=v)
    news = [min(rows, n) for n in lengths]
    q = (size * torch.randn((sum(news), 4, dim), generator=w.gen)).to(dtype)
    mask = torch.zeros((1, 1, max(lengths))) if masked else None
    got = w.backend.kv_attention(q.to(DEV), w.cache, w.batch(news), mask=None if mask is None else mask.to(DEV)).cpu().double()
    assert got.isfinite().all()
    at, checked = 0, 0
    for i, (n, m) in enumerate(zip(lengths, news)):
        kk, _ = w.k.values(w.table[i], n)
        vv, _ = w.v.values(w.table[i], n)
        for r in range(0, m, max(1, m // 7)):
            for h in range(4):
                seen = n - m + r + 1
                x = kk[:seen, h // 2] @ q[at + r, h].double() / math.sqrt(dim)
                top = x.sort(descending=True)
                # as far ahead as the scores' own roundings, and 64 for the next to have no weight
                if seen > 1 and top.values[0] - top.values[1] < 64 + 2.0 ** -18 * x.abs().max():
                    continue
                want = vv[int(top.indices[0]), h // 2]
                most = ROUND[dtype] * want.abs() + 2.0 ** (-20 if dtype == torch.float32 else -10) * want.abs().max()
                assert ((got[at + r, h] - want).abs() <= most).all(), (i, r, h)
                checked += 1
        at += m
    assert checked
