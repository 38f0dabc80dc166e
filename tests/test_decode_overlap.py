"""Rotations in place whose tensors lie among each other, refused before anything reaches the GPU."""
import ctypes

import pytest

from rns_llm_amd import _native

AT, ELSEWHERE, STEPS = 1 << 20, 1 << 30, 4096  # addresses that are never read


def turn(q, k, q_out, k_out, **changes):
    values = dict(rows=4, q_row_stride=64, q_head_stride=8, k_row_stride=64, k_head_stride=8, q_out_row_stride=64, q_out_head_stride=8,
                  k_out_row_stride=64, k_out_head_stride=8, q_heads=3, k_heads=2, head_dim=8, dtype=_native.FLOAT16,
                  positions_dtype=_native.INT32, back=0)
    values.update(changes)
    rotary, rows = _native.RotaryStruct(STEPS, 4, 0, 1.0), _native.RotaryRowsStruct(**values)
    rc = _native.lib().rnsmx_rotate(ctypes.byref(rotary), ctypes.byref(rows), STEPS, q, k, q_out, k_out, None)
    return rc, _native.lib().rnsmx_last_error().decode()


@pytest.mark.parametrize("moved", [0, 16, 3 * 128, -16])
@pytest.mark.parametrize("strides", [{}, {"row": 80}, {"head": 16}])
def test_one_in_place_the_other_read_from_its_memory(moved, strides):
    """Workgroups would read the one while others write it."""
    for mine, other in (("q", "k"), ("k", "q")):
        changes = {f"{other}_row_stride": strides.get("row", 64), f"{other}_head_stride": strides.get("head", 8)}
        args = {mine: AT, mine + "_out": AT, other: AT + moved, other + "_out": ELSEWHERE}
        rc, message = turn(args["q"], args["k"], args["q_out"], args["k_out"], **changes)
        assert rc == _native.EINVAL and "lie over queries or keys" in message


@pytest.mark.parametrize("changes", [
    {"q_row_stride": 2 ** 61, "q_out_row_stride": 2 ** 61, "rows": 9}, {"k_row_stride": 2 ** 62, "k_out_row_stride": 2 ** 62},
    {"q_head_stride": 2 ** 62, "q_out_head_stride": 2 ** 62}, {"k_out_head_stride": 2 ** 63 - 1},
])
def test_strides_past_the_address_space(changes):
    """Extents that pass 64 bits would not tell what lies over what."""
    rc, message = turn(AT, AT + (1 << 40), AT, AT + (1 << 40), **changes)
    assert rc == _native.EINVAL and "address space" in message
