"""The oracle of the decoding loop's operators, pinned by cases worked out by hand and by
slow definitions."""
import math

import pytest
import torch

from oracle import decode_oracle as do
from rns_llm_amd.backends.rotary import RotaryOps


def test_pages_by_hand():
    book = do.PageBook(blocks=8, page=16, seqs=3, width=3)
    assert book.assign([17, 0, 5], 64, 64, 48) == ([17, 0, 5], [0, 17, 17, 22], [(-1, -1, 0)] * 3, 0)
    assert book.pages == [[0, 1], [], [2]] and book.refs == [1, 1, 1, 0, 0, 0, 0, 0]
    book.reorder([0, 0, 0])  # three hold 0 and 1, 2 is free
    assert book.refs == [3, 3, 0, 0, 0, 0, 0, 0] and book.lengths == [17, 17, 17]
    # two of three go on: both copy; the third still holds the page
    assert book.assign([1, 1, 0], 64, 64, 48)[2:] == ([(1, 2, 1), (1, 3, 1), (-1, -1, 0)], 0)
    assert book.refs == [3, 1, 1, 1, 0, 0, 0, 0]
    book.reorder([0, 0, 0])
    # all three go on: the first keeps the page
    assert book.assign([1, 1, 1], 64, 64, 48)[2:] == ([(-1, -1, 0), (2, 1, 2), (2, 3, 2)], 0)
    book.trim([16, 0, 99])
    assert book.pages == [[0], [], [0, 3]] and book.refs == [2, 0, 0, 1, 0, 0, 0, 0] and book.lengths == [16, 0, 19]
    before = (book.pages, list(book.refs), list(book.lengths))
    assert book.assign([33, 0, 0], 64, 64, 48)[3] == -1
    assert book.assign([32, 33, 29], 64, 64, 48)[3] == -2
    assert do.PageBook(2, 16, 1, 3).assign([48], 64, 64, 48)[3] == 1
    assert (book.pages, book.refs, book.lengths) == before


def test_slots_by_hand():
    positions, places = do.slots([[4, 1], [9, -1], [0, 2]], [18, 17, 3], [0, 3, 5, 6], 7, 16, 9, 2, 32)
    assert positions.tolist() == [15, 16, 17, 15, 16, 2, 0]
    assert places.tolist() == [4 * 16 + 15, 16, -1, -1, -1, 2, -1]  # a row past two, a page past nine, none, no sequence


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_a_complex_product(interleaved):
    freq, positions = [1.0, 0.01], [0, 1, -7, 10 ** 6]
    x = torch.randn((4, 3, 5), dtype=torch.float64)
    y = do.rotate(x, *do.rotary_angles(freq, positions), interleaved, 2.0)
    for r, p in enumerate(positions):
        for i, f in enumerate(freq):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 2)
            z = torch.complex(x[r, :, a], x[r, :, b]) * 2 * complex(math.cos(p * f), math.sin(p * f))
            assert torch.allclose(torch.complex(y[r, :, a], y[r, :, b]), z, atol=1e-9)
    assert torch.equal(y[..., 4], x[..., 4])


def test_selection_by_hand():
    ln = math.log
    logits = torch.tensor([[[ln(1.0), ln(2.0), ln(1.0)], [ln(8.0), -math.inf, ln(8.0)], [1.0, math.nan, 0.0], [5.0, 5.0, 5.0]]])
    scores = torch.tensor([[0.0, 0.0, 9.0, ln(0.25)]])
    got = do.beam_select(logits, scores, 7, torch.tensor([[False, False, False, True]]), 2)
    assert torch.allclose(got[0], torch.tensor([[0.5, 0.5, 0.5, 0.25, 0.25, 0.25, 0.0]], dtype=torch.float64).log())
    # the scores of 0.5 are ln(2) - ln(4) and ln(8) - ln(16), which differ in 64 bits; tokens of a beam are in order
    assert sorted(zip(got[2][0, :3].tolist(), got[1][0, :3].tolist())) == [(0, 1), (1, 0), (1, 2)]
    assert got[1][0, 6] == 2 and got[2][0, 6] == 6 % 4


def frequencies(dim, base=10000.0, scaling=None, factor=1.0, original=None, low=1.0, high=32.0):
    return RotaryOps._frequencies(dim, base, scaling, factor, original, low, high)


def test_frequencies():
    plain = frequencies(8)
    assert plain == pytest.approx([1.0, 0.1, 0.01, 0.001])
    assert frequencies(8, scaling="linear", factor=4.0) == pytest.approx([f / 4 for f in plain])
    based = frequencies(8, scaling="base", factor=16.0)
    assert based[0] == 1.0 and based[3] == pytest.approx(plain[3] / 16)
    # 1000 tokens: 159 turns of the first, 15.9, 1.59 and 0.159 of the others
    bands = frequencies(8, scaling="bands", factor=8.0, original=1000, low=1.0, high=32.0)
    part = [1.0, (1000 * 0.1 / (2 * math.pi) - 1) / 31, (1000 * 0.01 / (2 * math.pi) - 1) / 31, 0.0]
    assert bands == pytest.approx([f * s + f / 8 * (1 - s) for f, s in zip(plain, part)])
