"""The order of different beams' continuations, which is exact down to the rounding of their log-sums."""
import math

import pytest
import torch

from oracle import decode_oracle as do

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def bound(size):
    """Of a log-sum: an exponent is rounded three times, 2^-24 each of |x - max|, whose mean under the terms'
    weights is at most ln V; an exponential 2 2^-24; at most 33 additions of a thread's."""
    return (3 * math.log(size + 1) + 35) * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size", [700, 20011, 128257])
@pytest.mark.parametrize("apart", [0.0, 2.25])
def test_beams_of_the_same_logits_in_another_order(backend, size, apart, dtype):
    """Their log-sums are equal by definition.  From twice the bound on the better beam goes first, nearer either
    may; a beam's own order, its tokens and all scores are right in any case, and for more requests too."""
    gen = torch.Generator().manual_seed(size)
    one = (torch.randn(size, generator=gen) * 2).clamp(max=8)
    one[torch.randperm(size, generator=gen)[:12]] = 10 + torch.arange(12) * 0.25  # the best, exact in every type
    one = one.to(dtype)
    logits = torch.stack([one[torch.randperm(size, generator=gen)] for _ in range(4)]).view(1, 4, size)
    scores = -1.0 - torch.tensor([[2.0, 0.0, 3.0, 1.0]], dtype=torch.float64) * apart * bound(size)
    scores = scores.float()  # moves none by more than 2^-24; a quarter of the bound is 13 of them and more
    want = do.beam_select(logits, scores, 16)
    for requests in (1, 90):
        got = backend.beam_select(logits.expand(requests, 4, size).to(DEV), scores.expand(requests, 4).contiguous().to(DEV), 16)
        assert all(torch.equal(x[0].expand(requests, 16), x - (4 * torch.arange(requests, device=DEV).view(-1, 1) if i == 2 else 0))
                   for i, x in enumerate(got))
        values, tokens, parents = (x[0].cpu() for x in got)
        off = (values.double() - want[0][0]).abs()
        assert (off <= bound(size) + want[0][0].abs() * 2.0 ** -24).all()
        assert sorted(zip(parents.tolist(), tokens.tolist())) == sorted(zip(want[2][0].tolist(), want[1][0].tolist()))
        for b in range(4):
            assert tokens[parents == b].tolist() == want[1][0][want[2][0] == b].tolist()
        if apart:
            assert torch.equal(parents, want[2][0]) and torch.equal(tokens, want[1][0])
