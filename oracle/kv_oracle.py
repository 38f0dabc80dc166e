"""CPU restatement of the 8-bit key/value cache and its attention: float32
where the definition says so (scales and codes), 64 bits everywhere else."""
from __future__ import annotations

import math

import torch

QMAX = 127.0
EPS = 2.0 ** -23


def float_scale(amax: torch.Tensor) -> torch.Tensor:
    """Scale of a page and head from the largest |x| (float32; NaN stays NaN)."""
    s = amax.float() * torch.tensor(1.0 / QMAX, dtype=torch.float32)
    return torch.where(s < EPS, torch.full_like(s, EPS), s)


def codes_of(x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Integer codes; a quotient that is not a number has code 0."""
    return torch.nan_to_num(torch.round(x.float() / scale), nan=0.0, posinf=QMAX, neginf=-QMAX).clamp(-QMAX, QMAX)


class Store:
    """The pages of one tensor (keys or values): integer codes [blocks, heads,
    page, dim] and float32 scales [blocks, heads]."""

    def __init__(self, blocks: int, heads: int, page: int, dim: int):
        self.page = page
        self.codes = torch.zeros((blocks, heads, page, dim))
        self.scales = torch.full((blocks, heads), EPS)

    def append(self, pages, length: int, x: torch.Tensor) -> None:
        """x [n, heads, dim]: the last n of a sequence's `length` tokens (those
        before its first have no place), its pages by number."""
        n = x.shape[0]
        x = x.float()[max(0, n - length):]
        at = length - x.shape[0]
        while at < length:
            index, offset = at // self.page, at % self.page
            take = min(self.page - offset, length - at)
            page = int(pages[index])
            if 0 <= page < self.codes.shape[0]:
                part = x[:take].transpose(0, 1)  # [heads, take, dim]
                s = float_scale(part.abs().amax(dim=(1, 2)))
                if offset:
                    held = self.scales[page]
                    s = torch.maximum(s, held)
                    old = self.codes[page, :, :offset] * held.view(-1, 1, 1)
                    self.codes[page, :, :offset] = codes_of(old, s.view(-1, 1, 1))
                self.codes[page, :, offset:offset + take] = codes_of(part, s.view(-1, 1, 1))
                self.scales[page] = s
            x = x[take:]
            at += take

    def values(self, pages, length: int) -> tuple[torch.Tensor, torch.Tensor]:
        """float64 [length, heads, dim] and which tokens are there."""
        heads, dim = self.codes.shape[1], self.codes.shape[3]
        out = torch.zeros((length, heads, dim), dtype=torch.float64)
        there = torch.zeros(length, dtype=torch.bool)
        for t in range(0, length, self.page):
            page, n = int(pages[t // self.page]), min(self.page, length - t)
            if 0 <= page < self.codes.shape[0]:
                out[t:t + n] = (self.codes[page, :, :n].double() * self.scales[page].double().view(-1, 1, 1)).transpose(0, 1)
                there[t:t + n] = True
        return out, there


def attention(q, k, v, there, *, scale=None, causal=True, window=0, mask=None):
    """One sequence: q [n, q_heads, dim], k and v float64 [length, heads, dim]
    -> (out, spread, reach) in 64 bits: the result, sum_t p_t |v_t| and sum |q||k| scale
    of the largest product of each row and head (what error bounds are made of)."""
    n, q_heads, dim = q.shape
    length, heads = k.shape[0], k.shape[1]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    out = torch.zeros((n, q_heads, dim), dtype=torch.float64)
    spread = torch.zeros_like(out)
    reach = torch.zeros((n, q_heads, 1), dtype=torch.float64)
    if length == 0 or n == 0:
        return out, spread, reach
    group = q_heads // heads
    kk, vv = (x.repeat_interleave(group, dim=1).transpose(0, 1) for x in (k, v))  # [q_heads, length, dim]
    qq = q.double().transpose(0, 1)
    own = length - n + torch.arange(n).view(1, n, 1)
    t = torch.arange(length).view(1, 1, length)
    seen = there.view(1, 1, length) & (((t <= own) & (t > own - (window or length + n + 1))) if causal else (t >= 0))
    seen = seen.expand(q_heads, n, length)
    # a hidden token may hold anything: out of the products before they are made
    x = torch.matmul(qq, torch.nan_to_num(kk, nan=0.0).transpose(1, 2)) * scale
    x = x + torch.where(kk.isnan().any(dim=2), math.nan, 0.0).view(q_heads, 1, length)
    size = torch.matmul(qq.abs(), torch.nan_to_num(kk, nan=0.0).abs().transpose(1, 2)) * scale
    if mask is not None:
        part = torch.zeros((n, q_heads, length), dtype=mask.dtype)
        wide = min(length, mask.shape[2])
        part[:, :, :wide] = mask.expand(n, q_heads, mask.shape[2])[:, :, :wide]
        if wide < length and mask.dtype != torch.bool:
            part[:, :, wide:] = -math.inf
        part = part.transpose(0, 1)
        if mask.dtype == torch.bool:
            seen = seen & part
        else:
            seen = seen & (part != -math.inf)
            x = x + part.double()
    size = torch.where(seen, size, 0.0)
    reach = size.amax(dim=-1, keepdim=True).transpose(0, 1)
    x = torch.where(seen, x, -math.inf)
    most = x.amax(dim=-1, keepdim=True)
    p = torch.where(seen, torch.exp(x - torch.where(most == -math.inf, 0.0, most)), 0.0)
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    held = torch.where(seen.any(dim=1).unsqueeze(-1), vv, 0.0)  # tokens no row sees
    for h in range(q_heads):
        for i in range(n):  # 0 * NaN of a token that this row does not see
            w = torch.where(seen[h, i].unsqueeze(-1), held[h], 0.0)
            out[i, h] = p[h, i] @ w
            spread[i, h] = p[h, i] @ w.abs()
    return out, spread, reach
