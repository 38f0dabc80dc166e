"""The 8-bit key/value cache on the GPU against the CPU oracle: codes and scales
bit for bit, values read back exactly, attention within bounds that follow from
its roundings (``bound``)."""
import math

import pytest
import torch

from oracle import kv_oracle as ko

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


# Sequences that hold nothing and ask nothing beside a test's own: with so many
# the prompts' kernel runs what few rows' would.
MANY = 170


class World:
    """A cache on the GPU and its oracle, filled alike."""

    def __init__(self, backend, *, lengths, heads, dim, page, seed, spare=2, idle=0):
        self.idle = idle
        self.backend, self.heads, self.dim, self.page = backend, heads, dim, page
        self.gen = torch.Generator().manual_seed(seed)
        pages = [max(1, -(-n // page)) for n in lengths]
        blocks = sum(pages) + spare
        order = torch.randperm(blocks, generator=self.gen, dtype=torch.int32)
        # entries past a sequence's end hold numbers that are no page's
        self.table = torch.full((len(lengths) + idle, max(pages)), 2 ** 31 - 1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(pages):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.cache = backend.create_kv_cache(device=torch.device(DEV, 0), blocks=blocks, block_size=page, kv_heads=heads,
                                             head_dim=dim)
        self.k, self.v = (ko.Store(blocks, heads, page, dim) for _ in range(2))
        self.lengths = list(lengths)

    def batch(self, news, lengths=None, **more):
        lengths = self.lengths if lengths is None else lengths
        return self.backend.kv_batch(self.cache, self.table.to(DEV), list(lengths) + [0] * self.idle,
                                     query_lengths=list(news) + [0] * self.idle, **more)

    def tokens(self, rows, dtype, heads=None):
        x = torch.randn((rows, heads or self.heads, self.dim), generator=self.gen)
        return (x * torch.exp(0.5 * torch.randn((1, heads or self.heads, self.dim), generator=self.gen))).to(dtype)

    def append(self, news, dtype, lengths=None, k=None, v=None):
        lengths = self.lengths if lengths is None else lengths
        rows = sum(news)
        k = self.tokens(rows, dtype) if k is None else k
        v = self.tokens(rows, dtype) if v is None else v
        self.backend.kv_append(self.cache, self.batch(news, lengths), k.to(DEV), v.to(DEV))
        at = 0
        for i, n in enumerate(news):
            self.k.append(self.table[i], lengths[i], k[at:at + n])
            self.v.append(self.table[i], lengths[i], v[at:at + n])
            at += n
        return k, v

    def same(self):
        torch.cuda.synchronize()
        for part, (codes, store) in enumerate(((self.cache.k_codes, self.k), (self.cache.v_codes, self.v))):
            assert torch.equal(codes.cpu()[..., :self.dim].float() - 128, store.codes)
            assert torch.equal(codes.cpu()[..., self.dim:], torch.full_like(codes.cpu()[..., self.dim:], 128))
            assert torch.equal(self.cache.scales.cpu()[..., part].nan_to_num(-1.0), store.scales.nan_to_num(-1.0))

    def want(self, q, news, lengths=None, mask=None, **options):
        lengths = self.lengths if lengths is None else lengths
        parts, at = [], 0
        for i, n in enumerate(news):
            k, there = self.k.values(self.table[i], lengths[i])
            v, _ = self.v.values(self.table[i], lengths[i])
            m = None if mask is None else mask.expand(sum(news), -1, -1)[at:at + n]
            parts.append(ko.attention(q[at:at + n], k, v, there, mask=m, **options))
            at += n
        return [torch.cat(p) for p in zip(*parts)]

    def check(self, news, dtype, q_heads, lengths=None, mask=None, q=None, **options):
        q = torch.randn((sum(news), q_heads, self.dim), generator=self.gen).to(dtype) if q is None else q
        got = self.backend.kv_attention(q.to(DEV), self.cache, self.batch(news, lengths),
                                        mask=None if mask is None else mask.to(DEV), **options)
        out, spread, reach = self.want(q, news, lengths, mask, **{k: v for k, v in options.items() if k in ("scale", "causal", "window")})
        assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous()
        got = got.cpu().double()
        assert torch.equal(got.isnan(), out.isnan())
        off = (got - out).abs().nan_to_num(0.0)
        most = bound(dtype, out, spread, reach, self.dim, max([1] + (self.lengths if lengths is None else lengths)), mask)
        assert (off <= most.nan_to_num(0.0)).all(), f"off by {float((off / most).nan_to_num(0.0).max()):.3g} of the bound"
        return got


def bound(dtype, out, spread, reach, dim, length, mask):
    """The output's rounding; the weights' (to 11 bits; to 22 in float32); the
    scores': a dot product's float32 sum is off by up to dim + 4 roundings of
    2^-24 of sum |q||k| (two products each in float32), and as much again for
    the exponent's own roundings, which goes into the weights twice (numerator
    and sum); weights under float16's smallest, 2^-25 of the largest each, and
    the float32 sums over the tokens."""
    weights = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -11
    size = reach + (0 if mask is None or mask.dtype == torch.bool else
                    float(mask[mask.isfinite()].float().abs().clamp(max=1e5).max()) if mask.isfinite().any() else 0)
    score = 2 * 2.0 ** -24 * (2 * (dim + 4) * reach + 16 * (size + 32))
    sums = 2.0 ** -24 * (length ** 0.5 + 64) * 2
    top = spread.amax(dim=-1, keepdim=True)
    return ROUND[dtype] * out.abs() + (weights + score + sums) * spread + length * 2.0 ** -27 * top + 1e-30


# ---------------------------------------------------------------------------
# Writing and reading
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,dim,page", [(1, 1, 16), (3, 40, 16), (2, 64, 32), (5, 65, 64), (2, 80, 128), (4, 96, 16),
                                            (1, 128, 128), (3, 160, 32), (2, 192, 64), (1, 250, 16), (2, 256, 128)])
def test_prompts_of_any_length(backend, dtype, heads, dim, page):
    lengths = [0, 1, page - 1, page, page + 1, 3 * page + 7]
    w = World(backend, lengths=lengths, heads=heads, dim=dim, page=page, seed=dim)
    w.append(lengths, dtype)
    w.same()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("page", [16, 64])
def test_token_by_token_the_scale_grows(backend, dtype, page):
    """Each token larger than those before in some heads: older codes are
    quantised again, step after step."""
    w = World(backend, lengths=[page + 9, page + 9], heads=4, dim=72, page=page, seed=5)
    for step in range(1, page + 9, 2):
        lengths = [step, max(0, step - 3)]
        news = [1 if step == 1 else 2, 0 if step < 4 else 1 if step == 5 else 2]
        k, v = (w.tokens(sum(news), dtype) * (1 + 0.2 * step * torch.tensor([1.0, 0.0, 1.0, 0.0]).view(1, 4, 1)).to(dtype)
                for _ in range(2))
        w.append(news, dtype, lengths, k.to(dtype), v.to(dtype))
    w.same()


def test_append_again_changes_nothing(backend):
    w = World(backend, lengths=[37, 80], heads=3, dim=64, page=32, seed=6)
    w.append([37, 80], torch.bfloat16)
    k, v = w.append([7, 9], torch.bfloat16)
    once = [t.clone() for t in (w.cache.k_codes, w.cache.v_codes, w.cache.scales)]
    w.backend.kv_append(w.cache, w.batch([7, 9]), k.to(DEV), v.to(DEV))
    assert all(torch.equal(x, y) for x, y in zip(once, (w.cache.k_codes, w.cache.v_codes, w.cache.scales)))
    w.same()


@pytest.mark.parametrize("dim,offset", [(64, 0), (64, 1), (50, 0), (50, 3)])
def test_views_of_a_fused_projection(backend, dim, offset):
    """k and v as column blocks of one tensor, rows and heads at its strides,
    aligned or not; and heads outermost."""
    rows, heads = 45, 4
    w = World(backend, lengths=[rows], heads=heads, dim=dim, page=16, seed=7)
    whole = torch.randn((rows, 3 * heads * dim + 8), generator=w.gen).to(torch.float16).to(DEV)
    k = whole[:, offset:offset + heads * dim].view(rows, heads, dim)
    v = whole[:, offset + heads * dim:offset + 2 * heads * dim].view(rows, heads, dim)
    w.backend.kv_append(w.cache, w.batch([rows]), k, v)
    w.k.append(w.table[0], rows, k.cpu())
    w.v.append(w.table[0], rows, v.cpu())
    w.same()
    outer = torch.randn((heads, rows, dim), generator=w.gen).to(DEV)
    turned = torch.randn((rows, dim, heads), generator=w.gen).to(DEV)  # last dimension strided: copied first
    w.backend.kv_append(w.cache, w.batch([rows]), outer.transpose(0, 1), turned.transpose(1, 2))
    w.k.append(w.table[0], rows, outer.transpose(0, 1).cpu())
    w.v.append(w.table[0], rows, turned.transpose(1, 2).cpu())
    w.same()


def test_more_rows_than_tokens_and_pages_that_are_not_there(backend):
    """Idle slots, rows before a sequence's first token, and page numbers out of
    range: nothing is written for them, zeros are read."""
    page, dim = 16, 40
    w = World(backend, lengths=[0, 3, 40, 33], heads=2, dim=dim, page=page, seed=8)
    w.table[2, 1] = -1
    w.table[3, 2] = w.cache.blocks
    news = [1, 5, 40, 33]
    w.append(news, torch.float32)
    w.same()
    k, v = w.backend.kv_read(w.cache, w.batch(news), dtype=torch.float32)
    at = 0
    for i, n in enumerate(news):
        for got, store in ((k, w.k), (v, w.v)):
            values, _ = store.values(w.table[i], w.lengths[i])
            want = torch.cat([torch.zeros((max(0, n - w.lengths[i]), 2, dim), dtype=torch.float64), values])
            assert torch.equal(got[at:at + n].cpu(), want.float())
        at += n
    got = w.check(news, torch.float32, 4)
    assert (got[0] == 0).all() and (got[1:3] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [1, 40, 65, 96, 128, 256])
def test_read_rounds_once(backend, dtype, dim):
    lengths = [1, 50, 129]
    w = World(backend, lengths=lengths, heads=3, dim=dim, page=32, seed=9)
    w.append(lengths, torch.float32)
    for news in (lengths, [1, 1, 1], [0, 19, 100]):
        k, v = w.backend.kv_read(w.cache, w.batch(news), dtype=dtype)
        for got, store in ((k, w.k), (v, w.v)):
            want = torch.cat([store.values(w.table[i], n)[0][n - m:] for i, (n, m) in enumerate(zip(lengths, news))])
            assert torch.equal(got.cpu(), want.float().to(dtype))


def test_not_finite_poisons_its_page_and_head_only(backend):
    w = World(backend, lengths=[40], heads=2, dim=64, page=16, seed=10)
    k, v = w.tokens(40, torch.float32), w.tokens(40, torch.float32)
    k[20, 0, 5], v[33, 1, 7] = math.inf, math.nan
    w.append([40], torch.float32, k=k, v=v)
    got_k, got_v = (x.cpu() for x in w.backend.kv_read(w.cache, w.batch([40]), dtype=torch.float32))
    assert got_k[16:32, 0].isnan().all() and got_v[32:, 1].isnan().all()
    assert got_k[:, 1].isfinite().all() and got_v[:, 0].isfinite().all()
    assert got_k[:16].isfinite().all() and got_k[32:].isfinite().all() and got_v[:32].isfinite().all()
    q = torch.randn((40, 2, 64), generator=w.gen)
    out = w.backend.kv_attention(q.to(DEV), w.cache, w.batch([40])).cpu()
    # rows that see the page, and no others
    assert out[:16].isfinite().all() and out[16:, 0].isnan().all()
    assert out[:32, 1].isfinite().all() and out[32:, 1].isnan().all()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,group,dim,page", [(1, 1, 1, 16), (2, 1, 40, 32), (3, 1, 64, 16), (2, 4, 65, 64), (2, 5, 80, 16),
                                                  (1, 16, 96, 128), (2, 17, 128, 64), (1, 3, 160, 16), (1, 8, 192, 32), (2, 2, 256, 128)])
def test_single_tokens(backend, dtype, heads, group, dim, page):
    lengths = [0, 1, 2, 15, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 257, 300]
    w = World(backend, lengths=lengths, heads=heads, dim=dim, page=page, seed=dim + group)
    w.append(lengths, dtype)
    w.check([1] * len(lengths), dtype, heads * group)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("group,dim,page", [(1, 64, 16), (3, 128, 32), (4, 80, 64)])
@pytest.mark.parametrize("causal,window", [(True, None), (False, None), (True, 1), (True, 45)])
@pytest.mark.parametrize("idle", [0, MANY])
def test_several_tokens(backend, dtype, group, dim, page, causal, window, idle):
    lengths, news = [70, 5, 200, 0, 33, 128], [70, 5, 3, 2, 1, 37]
    w = World(backend, lengths=lengths, heads=2, dim=dim, page=page, seed=dim + page, idle=idle)
    w.append(lengths, dtype)
    options = {"causal": causal} if window is None else {"window": window}
    w.check(news, dtype, 2 * group, **options)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("idle", [0, MANY])
def test_windows_of_any_place_in_a_step(backend, dim, idle):
    """A window's first step starts up to 63 tokens before it; its last tokens
    are seen all the same, in a table that has room for many more."""
    lengths = [286, 287, 285, 256, 320, 319, 190, 100]
    news = [100, 100, 99, 100, 100, 100, 100, 100]
    w = World(backend, lengths=lengths, heads=2, dim=dim, page=16, seed=27, idle=idle)
    w.append(lengths, torch.float16)
    for window in (1, 28, 29, 60, 61, 92, 93):
        w.check(news, torch.float16, 2, window=window)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,dim,page", [(1, 1, 16), (3, 40, 32), (2, 65, 64), (1, 160, 16), (1, 192, 128), (1, 250, 64), (1, 256, 32)])
def test_prompts_of_any_head(backend, dtype, heads, dim, page):
    lengths, news = [129, 40, 190, 1, 64], [129, 40, 70, 1, 64]
    w = World(backend, lengths=lengths, heads=heads, dim=dim, page=page, seed=dim, idle=MANY)
    w.append(lengths, dtype)
    w.check(news, dtype, heads)
    w.check(news, dtype, 2 * heads, window=50)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,group,dim,page,lengths,news,idle", [
    (1, 1, 64, 16, [3000, 700], [640, 65], 18), (2, 2, 40, 64, [2600, 130], [300, 130], 8), (1, 3, 128, 32, [3000, 1], [600, 1], 5),
    (1, 1, 160, 16, [3000, 0], [640, 1], 18), (1, 2, 250, 128, [3000, 90], [640, 66], 8),
])
def test_prompts_split_over_their_tokens(backend, dtype, heads, group, dim, page, lengths, news, idle):
    """Long prompts of a few workgroups, whose tokens are split."""
    w = World(backend, lengths=lengths, heads=heads, dim=dim, page=page, seed=dim + page, idle=idle)
    w.append(lengths, dtype)
    batch = w.batch(news)
    need = w.backend.kv_attention_workspace_bytes(w.cache, batch, q_heads=heads * group, dtype=dtype)
    assert need > 0
    w.check(news, dtype, heads * group)
    space = torch.zeros(need, dtype=torch.uint8, device=DEV)
    q = torch.randn((sum(news), heads * group, dim), generator=w.gen).to(dtype).to(DEV)
    first = w.backend.kv_attention(q, w.cache, batch, workspace=space)
    for _ in range(5):
        assert torch.equal(w.backend.kv_attention(q, w.cache, batch, workspace=space), first)
    assert (space[:4 * 16384] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("group,dim", [(1, 128), (4, 64), (1, 256)])
def test_some_rows_split_over_their_tokens(backend, dtype, group, dim):
    """Up to a few hundred rows of few sequences take 16 to a workgroup, split."""
    lengths, news = [1500, 130, 700, 0], [150, 130, 65, 1]
    w = World(backend, lengths=lengths, heads=1, dim=dim, page=16, seed=dim)
    w.append(lengths, dtype)
    w.check(news, dtype, group)
    w.check(news, dtype, group, window=300)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_of_many_sequences(backend, dtype, dim):
    """Enough workgroups that each runs on four waves."""
    seqs = 150
    lengths = [60 + 7 * (i % 15) for i in range(seqs)]
    news = [66 + (i % 3) if n >= 70 else n for i, n in enumerate(lengths)]
    w = World(backend, lengths=lengths, heads=8, dim=dim, page=32, seed=26)
    w.append(lengths, dtype)
    q = torch.randn((sum(news), 8, dim), generator=w.gen).to(dtype)
    got = w.backend.kv_attention(q.to(DEV), w.cache, w.batch(news)).cpu().double()
    at = 0
    for i, n in enumerate(news):
        if i % 29 == 0:
            k, there = w.k.values(w.table[i], lengths[i])
            v, _ = w.v.values(w.table[i], lengths[i])
            out, spread, reach = ko.attention(q[at:at + n], k, v, there)
            assert ((got[at:at + n] - out).abs() <= bound(dtype, out, spread, reach, dim, lengths[i], None)).all()
        at += n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_scale_and_large_products(backend, dtype):
    w = World(backend, lengths=[190, 7], heads=2, dim=64, page=16, seed=12)
    w.append([190, 7], dtype)
    w.check([2, 1], dtype, 4, scale=0.3)
    # one key dominates by far, then none does
    q = 30 * torch.randn((3, 4, 64), generator=w.gen)
    w.check([2, 1], dtype, 4, q=q.to(dtype))
    w.check([2, 1], dtype, 4, q=torch.zeros((3, 4, 64), dtype=dtype))


def test_values_of_very_different_pages(backend):
    """Value scales from page to page by up to 2^30, in either order."""
    w = World(backend, lengths=[160, 160], heads=1, dim=64, page=16, seed=13)
    turn = torch.cat([torch.arange(160), torch.arange(159, -1, -1)]) // 16
    v = w.tokens(320, torch.float32) * 2.0 ** (3 * turn - 20).view(-1, 1, 1)
    w.append([160, 160], torch.float32, v=v)
    w.check([1, 1], torch.float32, 2)
    w.check([5, 5], torch.bfloat16, 2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim,page,news,idle", [(64, 16, [1, 1, 1, 1], 0), (96, 32, [5, 3, 1, 9], 0), (128, 64, [40, 21, 3, 2], 0),
                                                (64, 32, [77, 21, 70, 2], MANY), (128, 16, [40, 21, 3, 2], MANY)])
def test_bool_masks(backend, dtype, dim, page, news, idle):
    lengths = [77, 21, 150, 2]
    w = World(backend, lengths=lengths, heads=2, dim=dim, page=page, seed=dim, idle=idle)
    w.append(lengths, dtype)
    rows = sum(news)
    mask = torch.rand((rows, 4, 150), generator=w.gen) < 0.7
    mask[1::3] = False  # rows that see nothing
    got = w.check(news, dtype, 4, mask=mask)
    assert (got[1::3] == 0).all()
    w.check(news, dtype, 4, mask=mask[:, :1])
    w.check(news, dtype, 4, mask=mask[:1, :, :])
    w.check(news, dtype, 4, mask=mask[:1, :1, :], window=30)
    wide = torch.rand((150, rows, 4), generator=w.gen) < 0.5  # tokens outermost
    w.check(news, dtype, 4, mask=wide.permute(1, 2, 0))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("mask_dtype", TYPES, ids=str)
@pytest.mark.parametrize("idle", [0, MANY])
def test_additive_masks(backend, dtype, mask_dtype, idle):
    lengths, news = [90, 33, 140], [4, 33, 1]
    w = World(backend, lengths=lengths, heads=2, dim=64, page=16, seed=14, idle=idle)
    w.append(lengths, dtype)
    mask = torch.randn((38, 4, 140), generator=w.gen)
    mask[torch.rand(mask.shape, generator=w.gen) < 0.2] = -math.inf
    mask[3::7] = -math.inf  # rows that see nothing
    mask = mask.to(mask_dtype)
    got = w.check(news, dtype, 4, mask=mask)
    assert (got[3::7] == 0).all()


@pytest.mark.parametrize("kind", [torch.bool, torch.float32, torch.float16])
@pytest.mark.parametrize("rows,idle", [(1, 0), (60, MANY)])
@pytest.mark.parametrize("columns", [0, 1, 37, 64, 130, 199])
def test_masks_that_end_before_the_tokens(backend, kind, rows, idle, columns):
    """With lengths on the device a mask may be shorter: what is past it is
    hidden, to the bit as by a mask that says so."""
    w = World(backend, lengths=[200, 150], heads=2, dim=72, page=16, seed=31, idle=idle)
    w.append([200, 150], torch.float16)
    news = [rows, rows] + [0] * idle
    starts = torch.tensor([0] + news, dtype=torch.int32).cumsum(0).to(dtype=torch.int32, device=DEV)
    lengths = torch.tensor([200, 150] + [0] * idle, dtype=torch.int32, device=DEV)
    batch = backend.kv_batch(w.cache, w.table.to(DEV), lengths, query_starts=starts, rows=2 * rows, max_query=rows)
    q = torch.randn((2 * rows, 4, 72), generator=w.gen).half().to(DEV)
    whole = torch.rand((2 * rows, 1, 208), generator=w.gen) < 0.7
    whole[:, :, columns:] = False
    if kind != torch.bool:
        whole = torch.where(whole, torch.randn(whole.shape, generator=w.gen), torch.tensor(-torch.inf)).to(kind)
    got = backend.kv_attention(q, w.cache, batch, mask=whole[:, :, :columns].contiguous().to(DEV))
    assert torch.equal(got, backend.kv_attention(q, w.cache, batch, mask=whole.to(DEV)))
    if columns == 0:
        assert (got == 0).all()


@pytest.mark.parametrize("mask_dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,idle", [(2, 0), (50, MANY)])
def test_masks_of_the_lowest_value(backend, mask_dtype, rows, idle):
    """The type's lowest value swallows the score: where a row has others, the
    token has no weight; where it has none, all its tokens weigh the same."""
    w = World(backend, lengths=[100, 61], heads=2, dim=64, page=16, seed=15, idle=idle)
    w.append([100, 61], torch.float32)
    low = torch.finfo(mask_dtype).min
    mask = torch.zeros((2 * rows, 1, 100), dtype=mask_dtype)
    mask[0, :, 40:] = low
    mask[1] = low
    mask[2, :, ::2] = low
    mask[3::5] = low
    w.check([rows, rows], torch.float32, 2, mask=mask)


@pytest.mark.parametrize("rows,idle", [(1, 0), (17, MANY)])
def test_hidden_places_may_hold_anything(backend, rows, idle):
    """NaN, infinities and codes of other sequences past the lengths, in pages
    beside the sequence's and under the mask."""
    w = World(backend, lengths=[50, 17], heads=2, dim=64, page=16, seed=16, spare=4, idle=idle)
    w.append([50, 17], torch.float32)
    heads = 4 if rows == 1 else 8  # enough rows for either kernel
    news = [rows, rows]
    q = torch.randn((2 * rows, heads, 64), generator=w.gen)
    mask = torch.ones((2 * rows, 1, 50), dtype=torch.bool)
    mask[:rows, :, 16:32] = False
    want = w.check(news, torch.float32, heads, q=q, mask=mask)
    used = torch.cat([w.table[0, :4], w.table[1, :2]]).long()
    free = torch.ones(w.cache.blocks, dtype=torch.bool)
    free[used] = False
    w.cache.scales[free.to(DEV)] = math.nan
    w.cache.scales[w.table[0, 1].item()] = math.nan  # under the mask
    w.cache.k_codes[w.table[0, 3].item(), :, 2:] = 255
    w.cache.v_codes[w.table[0, 3].item(), :, 2:] = 0
    w.table[1, 2:] = int(free.nonzero()[0])  # past the end
    hidden = torch.where(mask, 0.0, -math.inf)
    hidden[rows:, :, 17:] = math.nan  # past the sequence's end
    for m in (mask, hidden):
        got = w.backend.kv_attention(q.to(DEV), w.cache, w.batch(news), mask=m.to(DEV)).cpu().double()
        assert got.isfinite().all()
        assert torch.allclose(got, want, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("rows,idle", [(3, 0), (40, 700)])
def test_infinite_masks_are_not_numbers(backend, rows, idle):
    w = World(backend, lengths=[40], heads=1, dim=64, page=16, seed=17, idle=idle)
    w.append([40], torch.float32)
    mask = torch.zeros((rows, 1, 40))
    mask[0, 0, 0], mask[1, 0, 1] = math.inf, math.nan
    out = w.backend.kv_attention(torch.ones((rows, 1, 64), device=DEV), w.cache, w.batch([rows]), mask=mask.to(DEV)).cpu()
    assert out[:2].isnan().all() and out[2:].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,group,dim,lengths", [(2, 4, 128, [9001]), (1, 1, 64, [5000, 0, 1, 3333]), (8, 2, 80, [2100] * 3)])
def test_long_sequences_are_split(backend, dtype, heads, group, dim, lengths):
    w = World(backend, lengths=lengths, heads=heads, dim=dim, page=64, seed=18)
    w.append(lengths, dtype)
    news = [1] * len(lengths)
    assert w.backend.kv_attention_workspace_bytes(w.cache, w.batch(news), q_heads=heads * group, dtype=dtype) > 0
    w.check(news, dtype, heads * group)
    w.check(news, dtype, heads * group, window=1500)


def test_split_counters_stay_zero_and_results_are_the_same_bits(backend):
    w = World(backend, lengths=[7000, 90, 4000], heads=2, dim=128, page=32, seed=19)
    w.append([7000, 90, 4000], torch.float16)
    q = torch.randn((3, 8, 128), generator=w.gen).half().to(DEV)
    batch = w.batch([1, 1, 1])
    need = w.backend.kv_attention_workspace_bytes(w.cache, batch, q_heads=8, dtype=torch.float16)
    space = torch.zeros(need, dtype=torch.uint8, device=DEV)
    first = w.backend.kv_attention(q, w.cache, batch, workspace=space)
    for _ in range(20):
        assert torch.equal(w.backend.kv_attention(q, w.cache, batch, workspace=space), first)
    assert (space[:4 * 16384] == 0).all()
    small = w.batch([1, 1, 1], [20, 30, 4000])  # another shape on the same workspace
    a = w.backend.kv_attention(q, w.cache, small, workspace=space)
    assert torch.equal(a, w.backend.kv_attention(q, w.cache, small))
    with pytest.raises(RuntimeError, match="workspace"):
        w.backend.kv_attention(q, w.cache, batch, workspace=space[:need - 16])


def test_strided_queries_and_given_output(backend):
    w = World(backend, lengths=[45], heads=2, dim=72, page=16, seed=20)
    w.append([45], torch.bfloat16)
    whole = torch.randn((9, 3 * 4 * 72 + 5), generator=w.gen).bfloat16().to(DEV)
    for offset in (0, 1, 8):
        q = whole[:, offset:offset + 4 * 72].view(9, 4, 72)
        want = w.backend.kv_attention(q.contiguous(), w.cache, w.batch([9]))
        out = torch.empty_like(want)
        assert w.backend.kv_attention(q, w.cache, w.batch([9]), out=out) is out
        assert torch.equal(out, want)
        assert torch.equal(w.backend.kv_attention(q.transpose(0, 1).contiguous().transpose(0, 1), w.cache, w.batch([9])), want)


def test_cache_past_four_gigabytes(backend):
    """Pages whose codes start past 2^32 bytes."""
    heads, dim, page = 8, 256, 128
    blocks = 2 ** 32 // (heads * dim * page) + 40
    cache = backend.create_kv_cache(device=torch.device(DEV, 0), blocks=blocks, block_size=page, kv_heads=heads, head_dim=dim)
    gen = torch.Generator().manual_seed(21)
    x = torch.randn((2, 300, heads, dim), generator=gen).half()
    table = torch.tensor([[blocks - 1, blocks - 30, 2]], dtype=torch.int32)
    stores = [ko.Store(4, heads, page, dim) for _ in range(2)]
    for store, t in zip(stores, x):
        store.append([0, 1, 2], 300, t)
    batch = backend.kv_batch(cache, table.to(DEV), [300], query_lengths=[300])
    backend.kv_append(cache, batch, x[0].to(DEV), x[1].to(DEV))
    (k, there), (v, _) = (s.values([0, 1, 2], 300) for s in stores)
    got = backend.kv_read(cache, batch, dtype=torch.float32)
    assert torch.equal(got[0].cpu(), k.float()) and torch.equal(got[1].cpu(), v.float())
    q = torch.randn((1, heads, dim), generator=gen).half()
    out = backend.kv_attention(q.to(DEV), cache, backend.kv_batch(cache, table.to(DEV), [300])).cpu().double()
    want, spread, reach = ko.attention(q, k, v, there)
    assert ((out - want).abs() <= bound(torch.float16, want, spread, reach, dim, 300, None)).all()


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 128), (torch.float16, 128), (torch.bfloat16, 256), (torch.bfloat16, 96)], ids=str)
def test_rows_past_the_caches(backend, dtype, dim):
    """Keys and values of 128 MB and more."""
    rows = 2 ** 27 // (2 * dtype.itemsize * 64 * dim) + 1
    lengths = [rows - 213, 213]
    w = World(backend, lengths=lengths, heads=64, dim=dim, page=32, seed=29)
    w.append(lengths, dtype)
    w.same()
    got = backend.kv_read(w.cache, w.batch(lengths), dtype=dtype)
    at = 0
    for i, n in enumerate(lengths):
        for x, store in zip(got, (w.k, w.v)):
            assert torch.equal(x[at:at + n].cpu(), store.values(w.table[i], n)[0].float().to(dtype))
        at += n


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("group,dim", [(1, 40), (8, 64), (2, 96), (1, 128), (4, 160), (2, 256)])
def test_attention_past_the_caches(backend, dtype, group, dim):
    """Tables with room for 128 MB of codes and more; what is in them is short."""
    lengths = [300, 1, 0, 33, 1100, 70, 129, 64]
    w = World(backend, lengths=lengths, heads=2, dim=dim, page=16, seed=dim + 30)
    w.append(lengths, dtype)
    w.table = torch.cat((w.table, torch.full((len(lengths), 8192), -1, dtype=torch.int32)), dim=1)
    w.check([1] * len(lengths), dtype, 2 * group)


def test_another_stream(backend):
    w = World(backend, lengths=[2600, 40], heads=2, dim=64, page=16, seed=22)
    w.append([2600, 40], torch.float16)
    q = torch.randn((2, 4, 64), generator=w.gen).half().to(DEV)
    batch = w.batch([1, 1])
    want = w.backend.kv_attention(q, w.cache, batch)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            got = w.backend.kv_attention(q, w.cache, batch)
    side.synchronize()
    assert torch.equal(got, want)


def test_a_captured_decode_step_advances(backend):
    """Append and attend captured once; lengths, tokens and queries are written
    between the replays, and every replay is checked against eager calls."""
    heads, dim, page, top = 2, 64, 16, 700
    w = World(backend, lengths=[top, top], heads=heads, dim=dim, page=page, seed=23)
    start = [600, 3]
    w.append(start, torch.float16, start)
    twin = backend.create_kv_cache(device=torch.device(DEV, 0), blocks=w.cache.blocks, block_size=page, kv_heads=heads, head_dim=dim)
    for a, b in ((twin.k_codes, w.cache.k_codes), (twin.v_codes, w.cache.v_codes), (twin.scales, w.cache.scales)):
        a.copy_(b)
    lengths = torch.tensor([601, 4], dtype=torch.int32, device=DEV)
    batch = backend.kv_batch(w.cache, w.table.to(DEV), lengths)
    q, k, v = (torch.zeros((2, n, dim), dtype=torch.float16, device=DEV) for n in (4, heads, heads))

    def step(cache):
        backend.kv_append(cache, batch, k, v)
        return backend.kv_attention(q, cache, batch)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(w.cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(w.cache)
    for a, b in ((w.cache.k_codes, twin.k_codes), (w.cache.v_codes, twin.v_codes), (w.cache.scales, twin.scales)):
        a.copy_(b)
    for i in range(20):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=w.gen).half() * (1 + 0.1 * i))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, step(twin))
        torch.cuda.synchronize()
        lengths.add_(1)
    assert torch.equal(w.cache.k_codes, twin.k_codes) and torch.equal(w.cache.scales, twin.scales)


def test_graphs_have_scratch_of_their_own(backend):
    """Two graphs captured with no call before them, the second replayed first,
    eager calls on the capturing stream and others between."""
    w = World(backend, lengths=[3000, 2500], heads=2, dim=64, page=16, seed=28)
    w.append([3000, 2500], torch.float16)
    batch = w.batch([1, 1])
    qs = [torch.randn((2, 4, 64), generator=w.gen).half().to(DEV) for _ in range(2)]
    assert w.backend.kv_attention_workspace_bytes(w.cache, batch, q_heads=4, dtype=torch.float16) > 0
    wants = [w.backend.kv_attention(q, w.cache, batch) for q in qs]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(w.backend.kv_attention(q, w.cache, batch))
    for which in (1, 0, 1, 1, 0):
        graphs[which].replay()
        assert torch.equal(outs[which], wants[which])
        assert torch.equal(w.backend.kv_attention(qs[which], w.cache, batch), wants[which])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = w.backend.kv_attention(qs[1 - which], w.cache, batch)
        side.synchronize()
        assert torch.equal(got, wants[1 - which])


def test_empty_calls(backend):
    w = World(backend, lengths=[5], heads=2, dim=64, page=16, seed=24)
    none = torch.empty((0, 2, 64), device=DEV)
    batch = w.batch([0])
    backend.kv_append(w.cache, batch, none, none)
    assert backend.kv_read(w.cache, batch, dtype=torch.float16)[0].shape == (0, 2, 64)
    assert backend.kv_attention(none, w.cache, batch).shape == (0, 2, 64)
    nobody = backend.kv_batch(w.cache, torch.zeros((0, 1), dtype=torch.int32, device=DEV), [])
    assert backend.kv_attention(none, w.cache, nobody).shape == (0, 2, 64)
    w.same()


def test_lengths_past_the_bounds_are_cut_off(backend):
    """Device-side lengths and row starts that lie: nothing out of range is
    read or written, and sequences within them are as they were."""
    w = World(backend, lengths=[40, 40], heads=2, dim=64, page=16, seed=25)
    w.append([40, 40], torch.float32)
    q = torch.randn((2, 2, 64), generator=w.gen).to(DEV)
    good = w.backend.kv_attention(q, w.cache, w.batch([1, 1]))
    table = w.table.to(DEV)
    lengths = torch.tensor([40, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    batch = backend.kv_batch(w.cache, table, lengths, max_length=40)
    assert torch.equal(w.backend.kv_attention(q, w.cache, batch), good)
    starts = torch.tensor([0, 1, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    batch = backend.kv_batch(w.cache, table, lengths, query_starts=starts, rows=2, max_query=1, max_length=40)
    assert torch.equal(w.backend.kv_attention(q, w.cache, batch), good)
    starts = torch.tensor([-5, -9, 7], dtype=torch.int32, device=DEV)
    batch = backend.kv_batch(w.cache, table, lengths, query_starts=starts, rows=2, max_query=2, max_length=40)
    w.backend.kv_attention(q, w.cache, batch)
    w.backend.kv_read(w.cache, batch, dtype=torch.float32)
    torch.cuda.synchronize()
    w.same()
