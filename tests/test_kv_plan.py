"""The rules by which attention over the 8-bit cache takes a kernel, its waves and
its splits, pinned at both sides of each; and what the GPU tests run by them."""
import ctypes

import pytest
import torch

from kv_plans import plan
from rns_llm_amd import _native

MANY = 170  # idle sequences of the GPU tests


# sizes (sequences, heads, query heads, rows, tokens, head dim), options ->
# tile_rows, row_tiles, waves, splits, chunk, stream
@pytest.mark.parametrize("sizes,options,want", [
    # single tokens: eight waves past 128 tokens while tasks are under 512 or tokens 4096 and more
    ((1, 12, 12, 1, 128, 64), {}, (16, 1, 4, 1, 128, 0)),
    ((1, 12, 12, 1, 144, 64), {}, (16, 1, 8, 1, 256, 0)),
    ((256, 12, 12, 1, 512, 64), {}, (16, 1, 4, 1, 512, 1)),
    ((511, 1, 1, 1, 512, 64), {}, (16, 1, 8, 1, 512, 0)),
    ((512, 1, 1, 1, 512, 64), {}, (16, 1, 4, 1, 512, 0)),
    ((62, 32, 32, 1, 4080, 128), {}, (16, 1, 4, 1, 4096, 1)),
    ((62, 32, 32, 1, 4096, 128), {}, (16, 1, 8, 1, 4096, 1)),
    ((1, 16, 16, 1, 1024, 192), {}, (16, 1, 4, 1, 1024, 0)),  # wide rows: four waves
    # splits: up to 256 workgroups, 1024 tokens and more each
    ((1, 8, 32, 1, 131072, 128), {}, (16, 1, 8, 32, 4096, 1)),
    ((1, 1, 16, 1, 2032, 128), {}, (16, 1, 8, 1, 2048, 0)),
    ((1, 1, 16, 1, 2048, 128), {}, (16, 1, 8, 2, 1024, 0)),
    ((128, 1, 1, 1, 4096, 64), {}, (16, 1, 8, 2, 2048, 0)),
    ((129, 1, 1, 1, 4096, 64), {}, (16, 1, 8, 1, 4096, 0)),
    # past the caches from 128 MB of codes on, whole rows, no mask, one tile of rows
    ((16, 8, 8, 1, 4096, 128), {}, (16, 1, 8, 2, 2048, 1)),
    ((16, 8, 8, 1, 4080, 128), {}, (16, 1, 8, 2, 2048, 0)),
    ((16, 8, 8, 1, 4096, 128), {"masked": True}, (16, 1, 8, 2, 2048, 0)),
    ((64, 8, 8, 1, 4096, 96), {}, (16, 1, 8, 1, 4096, 0)),
    ((16, 8, 8, 17, 4096, 128), {}, (16, 2, 8, 1, 4096, 0)),
    # a window's tokens decide
    ((24, 8, 40, 1, 3008, 80), {"window": 1023, "dtype": torch.float32}, (16, 1, 8, 1, 1280, 0)),
    ((1, 8, 32, 1, 131072, 128), {"window": 500}, (16, 1, 8, 1, 768, 0)),
    # 16 rows to a workgroup up to 32 rows, and past them up to 1280 workgroups (640 of wide rows) of few tokens
    ((16, 4, 16, 5, 800, 96), {"page": 32}, (16, 2, 8, 1, 1024, 0)),
    ((1000, 8, 8, 32, 512, 128), {}, (16, 2, 4, 1, 512, 0)),
    ((1000, 8, 8, 33, 512, 128), {}, (128, 1, 4, 1, 512, 0)),
    ((80, 1, 1, 256, 256, 128), {}, (16, 16, 4, 1, 256, 0)),
    ((81, 1, 1, 256, 256, 128), {}, (128, 2, 8, 1, 256, 0)),
    ((40, 1, 1, 256, 256, 256), {}, (16, 16, 4, 1, 256, 0)),
    ((41, 1, 1, 256, 256, 256), {}, (128, 2, 4, 1, 256, 0)),
    ((1, 8, 8, 128, 8000, 128), {}, (16, 8, 8, 4, 2048, 0)),
    ((1, 8, 8, 512, 8000, 128), {}, (128, 4, 8, 8, 1024, 0)),
    # prompts: eight waves up to 384 tiles, or 512 of 4096 tokens and more; rows of 160 bytes and up four
    ((1, 32, 32, 2048, 2048, 128), {"page": 64}, (128, 16, 4, 1, 2048, 0)),
    ((6, 12, 12, 511, 2512, 64), {}, (128, 4, 8, 1, 2560, 0)),
    ((1, 8, 8, 8192, 8192, 128), {}, (128, 64, 8, 1, 8192, 0)),
    ((1, 32, 32, 8192, 8192, 128), {}, (128, 64, 4, 1, 8192, 0)),
    ((1, 24, 24, 2048, 2048, 64), {}, (128, 16, 8, 1, 2048, 0)),
    ((1, 25, 25, 2048, 2048, 64), {}, (128, 16, 4, 1, 2048, 0)),
    # their tokens split up to 256 workgroups of 512 tokens and more
    ((1, 16, 16, 1024, 1024, 256), {}, (128, 8, 4, 2, 512, 0)),
    ((1, 17, 17, 1024, 1024, 256), {}, (128, 8, 4, 1, 1024, 0)),
])
def test_rules(sizes, options, want):
    assert plan(*sizes, **options) == want


# what the tests of the prompts' kernel with few real sequences rest on: 128 rows, and
# more than one split where that is their point
@pytest.mark.parametrize("sizes,options,split", [
    ((6 + MANY, 2, 2, 70, 208, 64), {}, False), ((6 + MANY, 2, 6, 70, 224, 128), {"page": 32}, False),
    ((6 + MANY, 2, 8, 70, 256, 80), {"page": 64}, False), ((6 + MANY, 2, 2, 70, 208, 64), {"window": 1}, False),
    ((8 + MANY, 2, 2, 100, 320, 64), {"window": 1}, False), ((8 + MANY, 2, 2, 100, 320, 128), {"window": 93}, False),
    ((5 + MANY, 1, 1, 129, 192, 1), {}, False), ((5 + MANY, 1, 1, 129, 192, 160), {}, False),
    ((5 + MANY, 1, 1, 129, 256, 192), {"page": 128}, False), ((5 + MANY, 1, 1, 129, 192, 256), {"page": 32}, False),
    ((20, 1, 1, 640, 3008, 64), {}, True), ((10, 2, 4, 300, 2624, 40), {"page": 64}, True),
    ((7, 1, 3, 600, 3008, 128), {"page": 32}, True), ((20, 1, 1, 640, 3008, 160), {}, True),
    ((10, 1, 2, 640, 3008, 250), {"page": 64}, True), ((150, 8, 8, 68, 160, 64), {"page": 32}, False),
    ((4 + MANY, 2, 4, 77, 160, 64), {"page": 32, "masked": True}, False),
    ((4 + MANY, 2, 4, 40, 160, 128), {"masked": True}, False), ((4 + MANY, 2, 4, 40, 160, 128), {"window": 30}, False),
    ((3 + MANY, 2, 4, 33, 144, 64), {"masked": True}, False), ((2 + MANY, 2, 4, 60, 208, 72), {"masked": True}, False),
    ((2 + MANY, 2, 2, 50, 112, 64), {"masked": True}, False), ((2 + MANY, 2, 8, 17, 64, 64), {"masked": True}, False),
    ((701, 1, 1, 40, 48, 64), {"masked": True}, False),
])
def test_tests_of_prompts_run_their_kernel(sizes, options, split):
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        got = plan(*sizes, dtype=dtype, **options)
        assert got[0] == 128 and (got[3] > 1) == split


@pytest.mark.parametrize("seqs,heads", [(2 ** 22, 2 ** 8), (2 ** 15, 2 ** 15), (2 ** 25, 1)])
def test_plans_of_more_bytes_than_64_bits_count(seqs, heads):
    """2^69 and 2^64 bytes of codes in the widest tables that the checks take."""
    assert plan(seqs, heads, heads, 1, 2 ** 30, 256, page=128)[5] == 1


def test_plans_follow_the_refusals():
    with pytest.raises(ValueError):
        plan(1, 3, 4, 1, 16, 64)
    with pytest.raises(ValueError):
        plan(1, 3, 3, 1, 16, 64, window=5, causal=0)
    assert _native.lib().rnsmx_kv_attention_plan(None, None, None, 0, None) == _native.EINVAL
    assert _native.lib().rnsmx_kv_attention_plan(None, None, None, 0, ctypes.addressof(_native.KVPlan())) == _native.EINVAL
