"""What a decoding loop does around the key/value cache, as cases that can be timed.

Each case is a plain dict; its "op" names what a pass calls:

  rotate  ``HipRNSBackend.rotate``: queries and keys turned by their positions,
          forward, or forward and backward
  pages   ``kv_trim``, ``kv_assign``, ``kv_slots``: a scheduler's step.  Tokens
          that were drafted and rejected are taken back, each sequence gets
          pages for its new tokens, and the rows of the step get their
          positions and slots
  fork    ``kv_trim``, ``kv_reorder``, ``kv_assign``, ``kv_slots``, ``kv_copy``:
          a beam search's step on the cache.  Every beam goes on from its
          parent, whose pages it shares but for the one written next
  select  ``HipRNSBackend.beam_select``: the best continuations of each request's
          beams, from logits

The rules.  A pair (a, b) of a head at position p becomes (a cos t - b sin t, b cos
t + a sin t) times a factor, t = p f, f the pair's frequency.  A sequence's tokens
lie in the pages of its row of the table, -1 past them.  Pages are held by any
number of sequences; new ones are the lowest that nobody holds, given to the
sequences in their order and to a sequence in its pages' order.  A page that is
partly filled and held by others too is replaced by a copy for every sequence
that goes on in it; where all its holders do, the first of them keeps it.  A
continuation's score is its beam's plus the token's log-probability, in 64 bits;
of equal ones the lower beam goes first, within a beam the larger logit, then the
lower token.  A finished beam goes on as it is, with the end token.

Sizes: 12 heads of 64 and 50272 tokens are OPT-125m's, 32 heads of 128 OPT-6.7B's;
fewer key/value heads than query heads are grouped heads.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda"
FLOATS = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BASE = 10000.0
ORIGINAL = 4096  # tokens a scaled model was trained on
LOW, HIGH = 1.0, 32.0  # turns over them below which a pair is slowed down whole, from which not at all


def _rotate_case(name, rows, q_heads, heads, dim, part, layout, dtype, top, scaling="", factor=1.0, grad=False):
    return dict(name=name, op="rotate", rows=rows, q_heads=q_heads, heads=heads, dim=dim, part=part, layout=layout, dtype=dtype,
                top=top, scaling=scaling, factor=factor, grad=grad)


def _pages_case(name, seqs, length, new, block):
    return dict(name=name, op="pages", seqs=seqs, length=length, new=new, block=block)


def _fork_case(name, requests, beams, length, heads, dim, block):
    return dict(name=name, op="fork", requests=requests, beams=beams, length=length, heads=heads, dim=dim, block=block)


def _select_case(name, requests, beams, k, vocabulary, dtype, finished=False):
    return dict(name=name, op="select", requests=requests, beams=beams, k=k, vocabulary=vocabulary, dtype=dtype,
                finished=finished)


def listed() -> list[dict]:
    return [
        # one new token of one request: launches and host time
        _rotate_case("rotate 1 token", 1, 12, 12, 64, 64, "half", "float16", 2047),
        # a decode step of 64 requests far into long contexts, scaled by bands
        _rotate_case("rotate 64 requests", 64, 32, 8, 128, 128, "half", "bfloat16", 131071, "bands", 32.0),
        # prompts of a batch: bandwidth
        _rotate_case("rotate prompts", 16383, 32, 8, 128, 128, "half", "bfloat16", 16383),
        # a training step on part of each head, neighbours as pairs
        _rotate_case("rotate part, gradients", 4095, 40, 8, 80, 32, "interleaved", "float32", 4095, "linear", 4.0, grad=True),
        # a decode step: one token each, some of them on a new page
        _pages_case("pages 64 requests", 64, 4096, 1, 16),
        # every other slot takes a prompt, the others go on by a token
        _pages_case("pages prompts", 512, 8191, 0, 64),
        # four beams of one short request
        _fork_case("fork 1 request", 1, 4, 150, 12, 64, 16),
        # four beams of 64 requests, grouped heads
        _fork_case("fork 64 requests", 64, 4, 1500, 8, 128, 64),
        # four beams of one request
        _select_case("select 1 request", 1, 4, 4, 50272, "float16"),
        # a beam search over a batch, twice as many candidates as beams
        _select_case("select 64 requests", 64, 4, 8, 50272, "bfloat16"),
        # wide beams in float32, an odd vocabulary, beams that have ended
        _select_case("select wide float32", 12, 16, 32, 128257, "float32", finished=True),
    ]


def _log(rng: random.Random, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng: random.Random) -> dict:
    heads = ((12, 12), (32, 32), (32, 8), (40, 8), (16, 1), (7, 7), (8, 2))
    while True:
        op = rng.choice(("rotate", "pages", "fork", "select"))
        if op == "rotate":
            q_heads, kv = rng.choice(heads)
            dim = rng.choice((40, 64, 65, 80, 96, 128, 160, 256))
            part = rng.choice((dim // 2 * 2, dim // 4 * 2, dim // 2 * 2, 2 * rng.randint(1, dim // 2)))
            scaling = rng.choice(("", "", "linear", "base", "bands"))
            c = _rotate_case("", _log(rng, 1, 16383), q_heads, kv, dim, part, rng.choice(("half", "interleaved")),
                             rng.choice(tuple(FLOATS)), _log(rng, 16, 1000000), scaling if part > 2 or scaling != "base" else "",
                             rng.choice((2.0, 8.0, 32.0)) if scaling else 1.0, grad=rng.random() < 0.3)
            fits = work(c)["bytes"] <= 3.4e8
        elif op == "pages":
            seqs = _log(rng, 1, 1024)
            c = _pages_case("", seqs, _log(rng, 2, 131071 if seqs < 8 else 8191), rng.choice((1, 1, rng.randint(2, 9), 0)),
                            rng.choice((16, 32, 64, 128)))
            fits = seqs * c["length"] <= 512 * 8191
        elif op == "fork":
            c = _fork_case("", _log(rng, 1, 64), rng.choice((1, 2, 3, 4, 5, 8)), _log(rng, 16, 4095),
                           rng.choice((1, 2, 7, 8, 12)), rng.choice((40, 64, 80, 128)), rng.choice((16, 32, 64, 128)))
            fits = c["requests"] * c["length"] * c["heads"] <= 64 * 1500 * 8 and c["requests"] * c["beams"] <= 256
        else:
            beams = rng.choice((1, 2, 3, 4, 5, 8, 16))
            c = _select_case("", _log(rng, 1, 64), beams, rng.choice((1, beams, beams, 2 * beams)), _log(rng, 500, 131071),
                             rng.choice(tuple(FLOATS)), finished=rng.random() < 0.3)
            fits = work(c)["bytes"] <= 9.9e7
        if fits:
            del c["name"]
            return c


def _spread(i: int, top: int, turn: float) -> int:
    return max(1, int(top * (0.125 + 0.875 * (1.0 - (i * turn) % 1.0))))


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


# ---------------------------------------------------------------------------
# Sizes and the histories of pools
# ---------------------------------------------------------------------------
PARKED = 3  # requests that wait: they hold pages and take no part in a "pages" step


def _groups(case: dict) -> int:
    return case["requests"] if case["op"] == "fork" else case["seqs"]


def _order(case: dict, seed: int | None) -> list[int]:
    """Which request is in which slot; as they come without a seed."""
    order = list(range(_groups(case)))
    if seed is not None:
        random.Random(seed).shuffle(order)
    return order


def _parked(case: dict, seed: int | None) -> list[int]:
    if case["op"] == "fork":
        return []
    rng = random.Random(seed or 0)
    return [rng.randint(1, 16 * case["block"]) for _ in range(PARKED)]


def _lengths(case: dict, seed: int | None = None) -> list[int]:
    """Tokens of every sequence after the step."""
    beams = case.get("beams", 1)
    return _parked(case, seed) + [max(2, _spread(i, case["length"], 0.6180339887)) for i in _order(case, seed) for _ in range(beams)]


def _news(case: dict, seed: int | None = None) -> list[int]:
    lengths = _lengths(case, seed)
    if case["op"] == "fork":
        return [1] * len(lengths)
    news, lengths = [0] * PARKED, lengths[PARKED:]
    for i, n in zip(_order(case, seed), lengths):
        if case["new"] == 0:  # prompts beside running requests
            news.append(n if i % 2 == 0 else 1)
        else:
            news.append(min(_spread(i, case["new"], 0.7548776662) if case["new"] > 1 else 1, n))
    return news


def _pages(n: int, block: int) -> int:
    return -(-n // block)


def _blocks(case: dict) -> int:
    """Pages of the pool, an eighth of them spare: enough for any sharing that comes about."""
    beams, block = case.get("beams", 1), case["block"]
    lengths = _lengths(case)[0 if beams > 1 or case["op"] == "fork" else PARKED:]
    whole = sum(_pages(n, block) for n in lengths[::beams])
    return whole + whole // 8 + len(lengths) * (4 if beams > 1 else 1) + 16 * PARKED + 5


def _width(case: dict) -> int:
    return max(_pages(case["length"], case["block"]), 16) + 1


def _parents(case: dict, turn: float) -> list[int]:
    """Each beam's parent among its request's: some go on themselves, some end, some go on twice."""
    beams, out = case["beams"], []
    for s in range(case["requests"] * beams):
        first, chance = s - s % beams, (s * turn) % 1.0
        kept = [i for i in range(first, s) if i == first or (i * turn) % 1.0 < 0.5]
        out.append(s if s == first or chance < 0.5 else first if chance < 0.8 else kept[-1])
    return out


def _history(case: dict, seed: int) -> list[tuple[str, list[int]]]:
    """The calls that brought a pool to where the step finds it."""
    lengths, news = _lengths(case, seed), _news(case, seed)
    held = [n - m for n, m in zip(lengths, news)]
    if case["op"] == "pages":  # requests came and went: pages in use are scattered
        early = [h // 2 + (h % 3) * (h > 3) for h in held]
        left = [0 if i % 2 else e // 3 for i, e in enumerate(early)]
        return [("assign", early), ("trim", left), ("assign", [h - t for h, t in zip(held, left)])]
    beams = case["beams"]
    prompt = [max(0, h - 5) if i % beams == 0 else 0 for i, h in enumerate(held)]
    rest = [h - prompt[i - i % beams] for i, h in enumerate(held)]
    first = [min(1, r) for r in rest]
    return [("assign", prompt), ("reorder", [i - i % beams for i in range(len(held))]), ("assign", first),
            ("reorder", _parents(case, 0.3247179572)), ("assign", [r - f for r, f in zip(rest, first)])]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)

    if case["op"] == "rotate":
        dtype, rows = FLOATS[case["dtype"]], case["rows"]
        # the column blocks of a fused projection, as they lie
        wide = normal(rows, case["q_heads"] + 2 * case["heads"], case["dim"], dtype=dtype)
        q, k = wide[:, :case["q_heads"]], wide[:, case["q_heads"]:case["q_heads"] + case["heads"]]
        if rows == 1:
            at = torch.randint(0, case["top"], (1,), generator=gen, device=DEVICE, dtype=torch.int32)
        elif rows <= 256:
            at = torch.randint(0, case["top"], (rows,), generator=gen, device=DEVICE, dtype=torch.int32)
        else:  # runs of tokens
            run = torch.randint(max(1, rows // 8), rows, (1,), generator=gen, device=DEVICE)
            start = torch.randint(0, case["top"], (2,), generator=gen, device=DEVICE)
            row = torch.arange(rows, device=DEVICE)
            at = (torch.where(row < run, start[0] + row, start[1] + row - run) % case["top"]).to(torch.int32)
        got = {"q": q, "k": k, "positions": at}
        if case["grad"]:
            got.update(dq=normal(rows, case["q_heads"], case["dim"], dtype=dtype),
                       dk=normal(rows, case["heads"], case["dim"], dtype=dtype))
        return got
    if case["op"] == "select":
        rows, size = case["requests"] * case["beams"], case["vocabulary"]
        logits = normal(rows, size).mul_(2.5)
        # some tokens are forbidden, a few stand out
        top = torch.randint(0, size, (rows, 8), generator=gen, device=DEVICE)
        logits.scatter_add_(1, top, 4.0 * normal(rows, 8).abs_())
        banned = torch.randint(0, size, (rows, 3), generator=gen, device=DEVICE)
        logits.scatter_(1, banned, -math.inf)
        scores = -3.0 * normal(case["requests"], case["beams"]).abs_() - 10.0
        got = {"logits": logits.to(FLOATS[case["dtype"]]).view(case["requests"], case["beams"], size), "scores": scores}
        if case["finished"]:
            got["finished"] = torch.rand(scores.shape, generator=gen, device=DEVICE) < 0.2
        return got
    if case["op"] == "fork":
        shape = (_blocks(case), case["heads"], case["block"], _row_bytes(case["dim"]))
        return {name: torch.randint(1, 256, shape, generator=gen, device=DEVICE, dtype=torch.uint8) for name in ("k", "v")} | {
            "scales": normal(shape[0], shape[1], 2).abs_()}
    return {}


def _row_bytes(dim: int) -> int:
    return next(d for d in (64, 96, 128, 160, 192, 256) if d >= dim)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _frequencies(case: dict) -> torch.Tensor:
    part, base, factor = case["part"], BASE, case["factor"]
    if case["scaling"] == "base":  # the slowest pair is slowed down by the factor, the fastest not at all
        base *= factor ** (part / (part - 2))
    f = torch.tensor(base, dtype=torch.float64) ** (-torch.arange(0, part, 2, dtype=torch.float64) / part)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "bands":
        turns = ORIGINAL * f / (2 * math.pi)
        keep = ((turns - LOW) / (HIGH - LOW)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f


def _halves(x: torch.Tensor, part: int, layout: str):
    if layout == "half":
        return x[..., :part // 2], x[..., part // 2:part]
    return x[..., 0:part:2], x[..., 1:part:2]


def _turned(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, part: int, layout: str) -> torch.Tensor:
    y = x.clone()
    a, b = _halves(x, part, layout)
    to_a, to_b = _halves(y, part, layout)
    to_a.copy_(a * cos - b * sin)
    to_b.copy_(b * cos + a * sin)
    return y


def _plain_rotate(state: dict) -> tuple:
    c = state["case"]
    angle = state["positions"].double().view(-1, 1, 1) * state["frequencies"]
    cos, sin = angle.cos().float(), angle.sin().float()
    turned = [_turned(state[n].float(), cos, sin, c["part"], c["layout"]).to(state[n].dtype) for n in ("q", "k")]
    if c["grad"]:
        turned += [_turned(state[n].float(), cos, -sin, c["part"], c["layout"]).to(state[n].dtype) for n in ("dq", "dk")]
    return tuple(turned)


class _Pool:
    """Pages by elementary operations, nothing read back."""

    def __init__(self, blocks: int, block: int, seqs: int, width: int):
        self.blocks, self.block = blocks, block
        self.table = torch.full((seqs, width), -1, dtype=torch.int32, device=DEVICE)
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device=DEVICE)
        self.refs = torch.zeros(blocks + 1, dtype=torch.int32, device=DEVICE)  # the last is nobody's
        self.column = torch.arange(width, device=DEVICE).view(1, -1)

    def _held(self, pages: torch.Tensor) -> torch.Tensor:
        return torch.where(pages < 0, self.blocks, pages).long()

    def _count(self, pages: torch.Tensor, add: torch.Tensor) -> None:
        self.refs.scatter_add_(0, self._held(pages).view(-1), add.to(torch.int32).reshape(-1))

    def trim(self, to: torch.Tensor) -> None:
        self.lengths = torch.minimum(self.lengths, to.clamp(min=0))
        gone = (self.column >= ((self.lengths + self.block - 1) // self.block).view(-1, 1)) & (self.table >= 0)
        self._count(self.table, -gone.int())
        self.table = torch.where(gone, -1, self.table)

    def reorder(self, parents: torch.Tensor) -> None:
        parents = parents.long()
        table = self.table[parents]
        self._count(table, (table >= 0).int())
        self._count(self.table, -(self.table >= 0).int())
        self.table, self.lengths = table, self.lengths[parents]

    def assign(self, new: torch.Tensor):
        """Lengths and row starts of the step, its copies (from, to, tokens) and what it lacks."""
        block, blocks, seqs = self.block, self.blocks, self.lengths.shape[0]
        old, ends = self.lengths, self.lengths + new
        inside = old % block
        column = (old // block).clamp(max=self.table.shape[1] - 1).long()
        tail = self.table.gather(1, column.view(-1, 1)).view(-1)
        page = self._held(tail)
        shared = (new > 0) & (inside > 0) & (self.refs[page] > 1)
        at = torch.where(shared, page, blocks)
        going = torch.zeros_like(self.refs).scatter_add_(0, at, shared.int())
        seq = torch.arange(seqs, dtype=torch.int32, device=DEVICE)
        first = torch.full_like(self.refs, seqs).scatter_reduce_(0, at, seq, "amin")
        copy = shared & ~((going[at] == self.refs[at]) & (first[at] == seq))
        begin = (old + block - 1) // block - copy.int()
        need = torch.where(new > 0, (ends + block - 1) // block - begin, 0)
        rank = need.cumsum(0) - need
        free = self.refs[:blocks] == 0
        lacks = (need.sum() - free.sum()).clamp(min=0)
        ok = lacks == 0
        order = torch.where(free, free.cumsum(0) - 1, blocks).long()
        picked = torch.zeros(blocks + 1, dtype=torch.int32, device=DEVICE).scatter_(
            0, order, torch.arange(blocks, dtype=torch.int32, device=DEVICE))
        fresh = (self.column >= begin.view(-1, 1)) & (self.column < (begin + need).view(-1, 1)) & ok
        pick = (rank.view(-1, 1) + self.column - begin.view(-1, 1)).clamp(0, blocks)
        table = torch.where(fresh, picked[pick], self.table)
        self._count(table, fresh.int())
        copy = copy & ok
        self._count(torch.where(copy, tail, -1), -copy.int())
        to = table.gather(1, column.view(-1, 1)).view(-1)
        copies = torch.stack([torch.where(copy, tail, -1), torch.where(copy, to, -1), torch.where(copy, inside, 0)], dim=1)
        self.table = table
        self.lengths = torch.where(ok, ends, old)
        seen = torch.where(ok & (new > 0), ends, 0)
        starts = torch.nn.functional.pad(new.cumsum(0), (1, 0)).to(torch.int32)
        return seen.to(torch.int32), starts, copies.to(torch.int32), lacks.to(torch.int32).view(1)

    def slots(self, seen: torch.Tensor, starts: torch.Tensor, rows: int):
        row = torch.arange(rows, dtype=torch.int32, device=DEVICE)
        seq = torch.searchsorted(starts[1:].contiguous(), row, right=True).clamp(max=seen.shape[0] - 1)
        at = seen[seq] - (starts[seq + 1] - row)
        page = self.table[seq, (at // self.block).clamp(0, self.table.shape[1] - 1).long()].long()
        slot = torch.where((at >= 0) & (page >= 0), page * self.block + at % self.block, -1)
        return at.clamp(min=0).to(torch.int32), slot


def _plain_pages(state: dict) -> tuple:
    pool = state["pool"]
    pool.trim(state["before"])
    if "parents" in state:
        pool.reorder(state["parents"])
    seen, starts, copies, lacks = pool.assign(state["new"])
    positions, slots = pool.slots(seen, starts, state["rows"])
    out = (pool.table, pool.lengths, pool.refs[:pool.blocks], seen, copies, lacks, positions, slots)
    if "k" not in state:
        return out
    source, target = copies[:, 0].clamp(min=0).long(), torch.where(copies[:, 1] < 0, pool.blocks, copies[:, 1]).long()
    there = torch.arange(pool.block, device=DEVICE).view(1, 1, -1, 1) < copies[:, 2].view(-1, 1, 1, 1)
    for codes in (state["k"], state["v"]):
        codes[target] = torch.where(there, codes[source], codes[target])
    state["scales"][target] = state["scales"][source]
    return out + tuple(state[n][:pool.blocks] for n in ("k", "v", "scales"))


def _plain_select(state: dict) -> tuple:
    c = state["case"]
    requests, beams, size, k = c["requests"], c["beams"], c["vocabulary"], c["k"]
    logits = state["logits"].double()
    score = state["scores"].double().unsqueeze(2) + (logits - logits.logsumexp(dim=2, keepdim=True))
    if c["finished"]:
        ended = state["finished"].unsqueeze(2)
        score = torch.where(ended, -math.inf, score)
        score[:, :, c["vocabulary"] - 1] = torch.where(state["finished"], state["scores"].double(), score[:, :, c["vocabulary"] - 1])
    # the best of each beam in the order of its logits, then of the request
    most = min(k, size)
    order = (torch.where(ended, score, logits) if c["finished"] else logits).sort(dim=2, descending=True, stable=True)[1][:, :, :most]
    best = score.gather(2, order).view(requests, beams * most)
    top, at = best.sort(dim=1, descending=True, stable=True)
    top, at = top[:, :k], at[:, :k]
    tokens = order.reshape(requests, beams * most).gather(1, at).to(torch.int32)
    parents = (at // most + torch.arange(requests, device=DEVICE).view(-1, 1) * beams).to(torch.int32)
    return top.float(), tokens, parents


# ---------------------------------------------------------------------------
# What a program has in hand, and the calls it makes
# ---------------------------------------------------------------------------
def _backend():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    package = os.path.join(root, "rns-llm_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from rns_llm_amd import HipRNSBackend

    return HipRNSBackend()


def prepare(case: dict, seed: int) -> dict:
    raw = _inputs(case, seed)
    state = {"case": case, **raw}
    backend = _backend() if own else None
    if own:
        state["backend"] = backend
    if case["op"] == "rotate":
        if own:
            scaling = {"scaling": case["scaling"], "factor": case["factor"]} if case["scaling"] else {}
            if case["scaling"] == "bands":
                scaling.update(original_length=ORIGINAL, low_turns=LOW, high_turns=HIGH)
            state["rotary"] = backend.create_rotary(device=torch.device(DEVICE), rotary_dim=case["part"], base=BASE,
                                                    layout=case["layout"], **scaling)
            if case["grad"]:
                state["q"], state["k"] = (state[n].detach().requires_grad_() for n in ("q", "k"))
        else:
            state["frequencies"] = _frequencies(case).to(DEVICE)
        return state
    if case["op"] == "select":
        return state
    lengths, news, block = _lengths(case, seed), _news(case, seed), case["block"]
    seqs, width, blocks = len(lengths), _width(case), _blocks(case)
    state.update(new=_ints(news), before=_ints([n - m for n, m in zip(lengths, news)]), rows=sum(news))
    if case["op"] == "fork":
        state["parents"] = _ints(_parents(case, 0.5698402910))
    if own:
        pool = backend.create_kv_pool(device=torch.device(DEVICE), blocks=blocks, block_size=block, sequences=seqs, width=width)
        for call, numbers in _history(case, seed):
            if call == "assign":
                step = backend.kv_step(pool, rows=sum(numbers), max_query=max(numbers))
                backend.kv_assign(pool, step, _ints(numbers))
            else:
                (backend.kv_trim if call == "trim" else backend.kv_reorder)(pool, _ints(numbers))
        state.update(pool=pool, step=backend.kv_step(pool, rows=sum(news), max_query=max(news)))
        if case["op"] == "fork":
            cache = backend.create_kv_cache(device=torch.device(DEVICE), blocks=blocks, block_size=block,
                                            kv_heads=case["heads"], head_dim=case["dim"])
            for to, name in ((cache.k_codes, "k"), (cache.v_codes, "v"), (cache.scales, "scales")):
                to.copy_(state.pop(name))
            state["cache"] = cache
        return state
    pool = _Pool(blocks, block, seqs, width)
    for call, numbers in _history(case, seed):
        getattr(pool, call)(_ints(numbers))
    state["pool"] = pool
    for name in ("k", "v", "scales"):
        if name in state:  # a page more, which what copies nothing is written to
            state[name] = torch.cat([state[name], state[name][:1]])
    return state


def run(state: dict):
    case = state["case"]
    op = case["op"]
    if not own:
        return (_plain_rotate if op == "rotate" else _plain_select if op == "select" else _plain_pages)(state)
    backend = state["backend"]
    if op == "rotate":
        q, k = backend.rotate(state["rotary"], state["positions"], state["q"], state["k"])
        if not case["grad"]:
            return q, k
        return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))
    if op == "select":
        ended = {"finished": state["finished"], "end_token": case["vocabulary"] - 1} if case["finished"] else {}
        return backend.beam_select(state["logits"], state["scores"], case["k"], **ended)
    pool, step = state["pool"], state["step"]
    backend.kv_trim(pool, state["before"])
    if op == "fork":
        backend.kv_reorder(pool, state["parents"])
    backend.kv_assign(pool, step, state["new"])
    positions, slots = backend.kv_slots(pool, step.batch)
    out = (pool.table, pool.lengths, pool.refs, step.lengths, step.copies, step.missing, positions, slots)
    if op == "pages":
        return out
    cache = state["cache"]
    backend.kv_copy(cache, step)
    return out + (cache.k_codes, cache.v_codes, cache.scales)


def work(case: dict) -> dict:
    if case["op"] == "rotate":
        values = case["rows"] * (case["q_heads"] + case["heads"])
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * values * case["dim"] * FLOATS[case["dtype"]].itemsize + 4 * case["rows"]),
                "flops": passes * 3 * values * case["part"]}
    if case["op"] == "select":
        rows = case["requests"] * case["beams"]
        return {"bytes": rows * case["vocabulary"] * FLOATS[case["dtype"]].itemsize + 4 * rows + 12 * case["requests"] * case["k"],
                "flops": 4 * rows * case["vocabulary"]}
    lengths, news, block = _lengths(case), _news(case), case["block"]
    fresh = sum(_pages(n, block) - _pages(n - m, block) for n, m in zip(lengths, news))
    seqs, rows = len(lengths), sum(news)
    # lengths and counts in and out, entries taken back and given, a bit a page, positions and slots
    size = seqs * 4 * 8 + fresh * 4 * 4 + _blocks(case) // 8 + rows * 12
    if case["op"] == "fork":
        size += seqs * 4 + sum(_pages(n, block) for n in lengths) * 4
        children = {}
        for s, p in enumerate(_parents(case, 0.5698402910)):
            children.setdefault(p, []).append(s)
        for p, all_of in children.items():
            size += (len(all_of) - 1) * case["heads"] * (((lengths[p] - 1) % block) * _row_bytes(case["dim"]) * 4 + 16)
    return {"bytes": size, "flops": rows * 8}


# ---------------------------------------------------------------------------
# The definitions, in 64 bits and one after the other
# ---------------------------------------------------------------------------
def _exact_rotate(case: dict, raw: dict) -> tuple:
    part, half = case["part"], case["part"] // 2
    # turns of a token to 2^-100 of one: whole numbers
    unit = 1 << 100
    pi = (4 * (4 * _arctan(5, unit) - _arctan(239, unit)))
    steps = [int(f * (1 << 64)) * (unit >> 64) * unit // (2 * pi) for f in _frequencies(case).tolist()]
    at = raw["positions"].tolist()
    turn = torch.empty((len(at), half), dtype=torch.float64)
    for i, step in enumerate(steps):
        fine = step >> 36  # 64 bits of a turn
        turn[:, i] = torch.tensor([((p * fine) & ((1 << 64) - 1)) / (1 << 64) for p in at], dtype=torch.float64)
    angle = (turn * (2 * math.pi)).to(DEVICE).unsqueeze(1)
    out = []
    for name, sign in (("q", 1), ("k", 1), ("dq", -1), ("dk", -1)):
        if name not in raw:
            continue
        x = raw[name].double()
        y = x.clone()
        ia = torch.arange(half, device=DEVICE) * (1 if case["layout"] == "half" else 2)
        ib = ia + (half if case["layout"] == "half" else 1)
        y[..., ia] = x[..., ia] * angle.cos() - sign * x[..., ib] * angle.sin()
        y[..., ib] = x[..., ib] * angle.cos() + sign * x[..., ia] * angle.sin()
        out.append(y)
    return tuple(out)


def _arctan(n: int, unit: int) -> int:
    """arctan(1 / n) in units of 1 / unit, by its series."""
    total, term, k = 0, unit // n, 1
    while term:
        total += term // k if k % 4 == 1 else -(term // k)
        term //= n * n
        k += 2
    return total


class _Book:
    """Pages one at a time."""

    def __init__(self, blocks: int, block: int, seqs: int, width: int):
        self.block, self.width = block, width
        self.refs = [0] * blocks
        self.rows = [[] for _ in range(seqs)]
        self.lengths = [0] * seqs

    def _drop(self, page: int) -> None:
        self.refs[page] -= 1

    def trim(self, to) -> None:
        for s, n in enumerate(to):
            self.lengths[s] = min(self.lengths[s], max(n, 0))
            while len(self.rows[s]) > _pages(self.lengths[s], self.block):
                self._drop(self.rows[s].pop())

    def reorder(self, parents) -> None:
        rows = [list(self.rows[p]) for p in parents]
        for row in rows:
            for page in row:
                self.refs[page] += 1
        for row in self.rows:
            for page in row:
                self._drop(page)
        self.rows, self.lengths = rows, [self.lengths[p] for p in parents]

    def assign(self, new):
        block, copies, holders = self.block, [], {}
        for s, n in enumerate(new):
            if n and self.lengths[s] % block:
                holders.setdefault(self.rows[s][-1], []).append(s)
        free = (p for p, r in enumerate(list(self.refs)) if r == 0)
        held = list(self.refs)
        for s, n in enumerate(new):
            inside, copied = self.lengths[s] % block, (-1, -1, 0)
            if n and inside:
                page = self.rows[s][-1]
                if held[page] > 1 and not (len(holders[page]) == held[page] and holders[page][0] == s):
                    copied = (page, next(free), inside)
                    self.rows[s][-1] = copied[1]
                    self.refs[copied[1]] += 1
                    self._drop(page)
            copies.append(copied)
            self.lengths[s] += n
            while len(self.rows[s]) < _pages(self.lengths[s], block):
                self.rows[s].append(next(free))
                self.refs[self.rows[s][-1]] += 1
        return copies


def _exact_pages(case: dict, raw: dict, seed: int):
    lengths, news, block = _lengths(case, seed), _news(case, seed), case["block"]
    book = _Book(_blocks(case), block, len(lengths), _width(case))
    for call, numbers in _history(case, seed):
        getattr(book, call)(numbers)
    book.trim([n - m for n, m in zip(lengths, news)])
    if case["op"] == "fork":
        book.reorder(_parents(case, 0.5698402910))
    copies = book.assign(news)
    table = [row + [-1] * (book.width - len(row)) for row in book.rows]
    seen = [n if m else 0 for n, m in zip(book.lengths, news)]
    positions = [p for n, m in zip(book.lengths, news) for p in range(n - m, n)]
    slots = [row[p // block] * block + p % block for row, n, m in zip(book.rows, book.lengths, news) for p in range(n - m, n)]
    out = (_ints(table), _ints(book.lengths), _ints(book.refs), _ints(seen), _ints(copies), _ints([0]), _ints(positions),
           torch.tensor(slots, dtype=torch.int64, device=DEVICE))
    if case["op"] == "pages":
        return out
    k, v, scales = raw["k"].clone(), raw["v"].clone(), raw["scales"].clone()
    for source, target, tokens in copies:
        if target >= 0:
            k[target, :, :tokens] = raw["k"][source, :, :tokens]
            v[target, :, :tokens] = raw["v"][source, :, :tokens]
            scales[target] = raw["scales"][source]
    return out + (k, v, scales.double())


def _exact_select(case: dict, raw: dict) -> tuple:
    scores, tokens, parents = [], [], []
    for r in range(case["requests"]):
        found = []
        for b in range(case["beams"]):
            own_score = raw["scores"][r, b].double()
            if case["finished"] and raw["finished"][r, b]:
                found.append((-float(own_score), b, 0.0, case["vocabulary"] - 1))
                continue
            x = raw["logits"][r, b].double()
            total = torch.log(torch.exp(x - x.max()).sum()) + x.max()
            least = x.topk(min(case["k"], x.numel()))[0][-1]
            for v in (x >= least).nonzero().view(-1).tolist():
                found.append((-float(own_score + (x[v] - total)), b, -float(x[v]), v))
        found.sort()
        found = found[:case["k"]]
        scores.append([-f[0] for f in found])
        tokens.append([f[3] for f in found])
        parents.append([r * case["beams"] + f[1] for f in found])
    return torch.tensor(scores, dtype=torch.float64, device=DEVICE), _ints(tokens), _ints(parents)


def exact(case: dict, seed: int):
    raw = _inputs(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(case, raw)
    return _exact_select(case, raw) if case["op"] == "select" else _exact_pages(case, raw, seed)
