"""Beam search's selection on the GPU against all candidates' scores in 64 bits."""
import math

import pytest
import torch

from oracle import decode_oracle as do
from rns_llm_amd import _native

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def slack(size, score):
    """What a score may be off by.  The logarithm of the sum of exponentials e^(x - m): a term's
    exponent is rounded three times (difference, product, the factor log2 e), 2^-24 each of itself, and the
    mean of |x - m| under the terms' weights is at most ln V; the exponential itself 2^-23; a thread's
    at most 33 additions 2^-24 each.  Then the score's rounding to float32."""
    return (math.log(size + 1) * 3 + 2 + 33) * 2.0 ** -24 + abs(score) * 2.0 ** -24


def check(backend, logits, scores, k, finished=None, end_token=None):
    """Every place has a candidate that is there, once, with its score; the scores go down, are the
    oracle's of their place, and candidates of one beam are in their order.  Where no two of the
    oracle's best are nearer than the scores' slack the candidates are the oracle's."""
    ended = {} if finished is None else {"finished": finished.to(DEV), "end_token": end_token}
    if finished is None and end_token is not None:
        ended = {"end_token": end_token}
    x = logits if logits.is_cuda else logits.to(DEV)
    got = [t.cpu() for t in backend.beam_select(x, scores.to(DEV), k, **ended)]
    requests, beams, size = logits.shape
    assert all(t.shape == (requests, k) for t in got) and [t.dtype for t in got] == [torch.float32, torch.int32, torch.int32]
    logits = logits.cpu()
    want = do.beam_select(logits, scores, k + 1 if k < beams * size else k, finished, end_token)
    every = do.beam_scores(logits, scores, finished, end_token)
    for r in range(requests):
        places = [(int(p) - r * beams, int(t)) for p, t in zip(got[2][r], got[1][r])]
        assert all(0 <= b < beams and 0 <= t < size for b, t in places)
        near = False
        for j, (b, t) in enumerate(places):
            score, best = got[0][r, j].item(), want[0][r, j].item()
            if best == -math.inf:
                assert score == -math.inf and (t, b) == (end_token or 0, j % beams)
                continue
            assert abs(score - every[r, b, t].item()) <= slack(size, score) and abs(score - best) <= slack(size, score)
            following = want[0][r, j + 1].item() if j + 1 < want[0].shape[1] else -math.inf
            near = near or (best - following <= 2 * slack(size, score) and want[2][r, j + 1] != want[2][r, j])
        live = [c for c, s in zip(places, got[0][r].tolist()) if s > -math.inf]
        assert len(set(live)) == len(live)
        for b in range(beams):
            mine = [t for c, t in live if c == b]
            if finished is None or not finished[r, b]:
                row = logits[r, b].double()
                assert mine == sorted(mine, key=lambda t: (-row[t].item(), t))
        if not near:
            assert torch.equal(got[1][r], want[1][r, :k]) and torch.equal(got[2][r], want[2][r, :k])
    return got


def made(requests, beams, size, dtype, seed=0, spread=2.0):
    gen = torch.Generator().manual_seed(seed + size)
    logits = (torch.randn((requests, beams, size), generator=gen) * spread).to(dtype)
    return logits, -torch.rand((requests, beams), generator=gen) * 5 - 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("requests,beams,k,size", [
    (1, 1, 1, 1), (2, 3, 4, 1), (1, 2, 5, 2), (3, 1, 1, 7), (2, 4, 8, 9), (1, 4, 64, 15), (2, 5, 7, 255), (1, 64, 64, 33), (1, 4, 4, 4095),
    (1, 4, 8, 4097), (2, 2, 3, 8192), (1, 3, 6, 16385), (1, 1, 64, 50257), (70, 2, 4, 1001), (1, 16, 32, 20011), (300, 4, 2, 4100),
])
def test_selection(backend, requests, beams, k, size, dtype):
    logits, scores = made(requests, beams, size, dtype)
    check(backend, logits, scores, k)


def test_a_long_vocabulary(backend):
    """Chunks of the most values, in float32 as long as the registers hold them."""
    logits, scores = made(2, 40, 65536 * 2 + 3, torch.float32)
    check(backend, logits, scores, 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size", [700, 4099, 17000])
@pytest.mark.parametrize("k", [1, 5, 64])
def test_equal_logits(backend, size, k, dtype):
    """All the same, of a few values, and of beams that are the same: the lower beam, the lower token first."""
    gen = torch.Generator().manual_seed(7)
    for logits in (torch.zeros((2, 3, size)), torch.randint(0, 3, (2, 3, size), generator=gen).float(),
                   torch.where(torch.arange(size) % 2 == 0, 0.0, -0.0).expand(2, 3, size)):
        logits = logits[:, :1].expand(2, 3, size).contiguous().to(dtype)
        got = backend.beam_select(logits.to(DEV), torch.full((2, 3), -1.5, device=DEV), k)
        want = do.beam_select(logits, torch.full((2, 3), -1.5), k)
        for a, b in zip(got[1:], want[1:]):
            assert torch.equal(a.cpu(), b)
    # rows that begin at odd addresses, of one beam's logits
    one = torch.randn(size, generator=gen).to(dtype)
    wide = torch.zeros((2, 3, size + 1), dtype=dtype, device=DEV)
    wide[..., 1:] = one.to(DEV)
    got = backend.beam_select(wide[..., 1:], torch.zeros((2, 3), device=DEV), k)
    want = do.beam_select(one.expand(2, 3, size), torch.zeros((2, 3)), k)
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=str)
@pytest.mark.parametrize("k", [3, 64])
def test_logits_in_order(backend, k, dtype):
    """The largest side by side, at either end and in the middle: more than a list holds reach the bound."""
    size = 12000
    up = torch.linspace(-9, 9, size).to(dtype)
    middle = torch.full((size,), -20.0, dtype=dtype)
    middle[5000:7300] = torch.linspace(1, 2, 2300).to(dtype)
    logits = torch.stack([up, up.flip(0), middle]).view(1, 3, size)
    check(backend, logits, torch.tensor([[-1.0, -1.25, -2.0]]), k)


def test_what_is_no_candidate(backend):
    """Forbidden tokens, beams without any, not-a-numbers, infinities, dead and finished beams."""
    inf, nan = math.inf, math.nan
    logits, scores = made(1, 9, 300, torch.float32, seed=3)
    logits[0, 0, :297] = -inf                       # three left
    logits[0, 1] = -inf                             # none
    logits[0, 2, 5] = nan
    logits[0, 3, 299] = inf
    logits[0, 4] = nan
    logits[0, 5, ::2] = torch.finfo(torch.float32).min
    scores[0, 6], scores[0, 7] = -inf, nan
    for k in (1, 4, 64):
        check(backend, logits, scores, k)
        ended = torch.tensor([[False, True, True, False, True, False, True, True, True]])
        check(backend, logits, scores, k, ended, 17)
        check(backend, logits[:, :5], scores[:, :5], k, ended[:, :5] & False, 0)
        check(backend, logits[:, 1:5], scores[:, 1:5], k, end_token=299)
    scores[0, 8] = inf
    check(backend, logits[:, 6:], scores[:, 6:], 3)


@pytest.mark.parametrize("beams,k,left", [(16, 32, 1), (16, 32, 3), (64, 64, 2), (8, 64, 1)])
def test_most_beams_finished(backend, beams, k, left):
    """Few chunks beside many finished beams, which give a low bound or none."""
    logits, scores = made(2, beams, 30011, torch.float16, seed=9)
    finished = torch.ones((2, beams), dtype=torch.bool)
    finished[:, 1:1 + left] = False
    check(backend, logits, scores, k, finished, 2)


@pytest.mark.parametrize("scale", [1e-30, 1e4, 3e37])
def test_small_and_large_logits(backend, scale):
    logits, scores = made(1, 2, 900, torch.float32, spread=1.0)
    logits = logits * scale
    if scale > 1e3:  # one token has nearly all of a beam: the others' scores are as far away as their logits
        got = [t.cpu() for t in backend.beam_select(logits.to(DEV), scores.to(DEV), 6)]
        want = do.beam_select(logits, scores, 6)
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        assert torch.allclose(got[0].double(), want[0], rtol=2.0 ** -23)
    else:
        check(backend, logits, scores, 6)


def test_strides(backend):
    logits, scores = made(3, 4, 1000, torch.float16, seed=5)
    gpu = logits.to(DEV)
    want = backend.beam_select(gpu, scores.to(DEV), 5)
    wide = torch.zeros((3, 4, 1003), dtype=torch.float16, device=DEV)
    wide[..., 2:1002] = gpu
    forms = [wide[..., 2:1002], gpu.transpose(0, 1).contiguous().transpose(0, 1), gpu.transpose(1, 2).contiguous().transpose(1, 2)]
    for x in forms:
        got = backend.beam_select(x, scores.t().contiguous().t().to(DEV), 5)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # the first step: one row for all of a request's beams, of which one counts
    first = torch.full((3, 4), -math.inf)
    first[:, 0] = 0
    got = backend.beam_select(gpu[:, :1].expand(3, 4, 1000), first.to(DEV), 4)
    best = do.beam_select(logits[:, :1], torch.zeros((3, 1)), 4)
    assert torch.equal(got[1].cpu(), best[1]) and torch.equal(got[2].cpu(), torch.arange(3, dtype=torch.int32).view(3, 1).expand(3, 4) * 4)


def test_more_requests_than_counters(backend):
    """A launch counts arrivals for so many requests; the others come in launches after it."""
    n = _native.KV_TICKETS + 70
    logits, scores = made(n, 2, 5, torch.float32)
    got = [t.cpu() for t in backend.beam_select(logits.to(DEV), scores.to(DEV), 2)]
    some = list(range(0, n, 257)) + list(range(_native.KV_TICKETS - 2, n))
    want = do.beam_select(logits[some], scores[some], 2)
    assert torch.equal(got[1][some], want[1])
    assert torch.equal(got[2][some] - 2 * torch.tensor(some, dtype=torch.int32).view(-1, 1),
                       want[2] - 2 * torch.arange(len(some), dtype=torch.int32).view(-1, 1))
    empty = backend.beam_select(torch.zeros((0, 2, 5), device=DEV), torch.zeros((0, 2), device=DEV), 3)
    assert all(t.shape == (0, 3) for t in empty)


def test_no_gradient(backend):
    logits, scores = made(1, 2, 50, torch.float32)
    out = backend.beam_select(logits.to(DEV).requires_grad_(), scores.to(DEV), 2)
    with pytest.raises(RuntimeError, match="no gradient"):
        out[0].sum().backward()
    with torch.no_grad():
        assert not backend.beam_select(logits.to(DEV).requires_grad_(), scores.to(DEV), 2)[0].requires_grad


def test_the_same_results_each_time(backend):
    """Also beside attention calls that keep their counters in the same memory, on another stream and from a graph."""
    logits, scores = made(5, 4, 50272, torch.bfloat16, seed=8)
    x, s = logits.to(DEV), scores.to(DEV)
    want = [t.clone() for t in backend.beam_select(x, s, 8)]
    cache = backend.create_kv_cache(device=DEV, blocks=300, block_size=16, kv_heads=1, head_dim=64)
    batch = backend.kv_batch(cache, torch.arange(300, dtype=torch.int32, device=DEV).view(1, 300), [4800])
    q = torch.randn((1, 1, 64), device=DEV)
    attended = backend.kv_attention(q, cache, batch)
    for _ in range(5):
        assert torch.equal(backend.kv_attention(q, cache, batch), attended)
        assert all(torch.equal(a, b) for a, b in zip(backend.beam_select(x, s, 8), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = backend.beam_select(x, s, 8)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = backend.beam_select(x, s, 8)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for i in range(3):
        x.copy_(x.roll(1, dims=0))
        graph.replay()
        again = backend.beam_select(x, s, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, again))


@pytest.mark.parametrize("requests,beams,k,size", [
    (2, 5, 64, 3 * 4096 - 40), (3, 16, 32, 9 * 4096), (1, 33, 64, 4 * 4096 + 9), (1, 64, 64, 5 * 4096), (1, 64, 50, 262144 - 3), (1, 8, 9, 17 * 4096),
])
def test_joins(backend, requests, beams, k, size):
    """Many chunks of a request: the best spread over them, of one beam, side by side in one chunk,
    and as many as are wanted in each chunk."""
    logits, scores = made(requests, beams, size, torch.bfloat16, seed=11)
    check(backend, logits, scores, k)
    check(backend, logits, scores - torch.arange(beams) * 7.0, k)
    logits[:, :, size // 2:size // 2 + 70] += 14
    check(backend, logits, scores, k)
    logits[:, 1:, size // 2:size // 2 + 70] -= 14
    check(backend, logits, scores, k)
    finished = torch.rand((requests, beams), generator=torch.Generator().manual_seed(2)) < 0.4
    check(backend, logits, scores, k, finished, 3)


@pytest.mark.parametrize("values", [1, 2, 40])
def test_joins_of_equal_logits(backend, values):
    """More chunks than are looked at side by side, whose best are the same."""
    gen = torch.Generator().manual_seed(12)
    logits = torch.randint(0, values, (1, 5 * 4096), generator=gen).half().expand(64, -1)[None].contiguous()
    for k in (3, 8, 64):
        got = backend.beam_select(logits.to(DEV), torch.full((1, 64), -0.5, device=DEV), k)
        want = do.beam_select(logits, torch.full((1, 64), -0.5), k)
        for a, b in zip(got[1:], want[1:]):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("requests,beams,k,size", [(3, 16, 16, 1100), (2, 16, 33, 2000), (2, 13, 64, 1000), (2, 2, 64, 4096 * 6), (1, 7, 48, 700)])
def test_joins_of_few_chunks(backend, requests, beams, k, size):
    """As many results as lists hold, and more, of chunks that are all looked at; k about where bounds change."""
    for dtype in (torch.float32, torch.float16):
        logits, scores = made(requests, beams, size, dtype, seed=13)
        for n in (k, k - 1):
            check(backend, logits, scores, n)
        check(backend, logits, scores * 8, k)
