"""Arguments of the decoding loop's entry points (pages, rotary positions, beam
selection), checked before anything reaches the GPU: through the C ABI with addresses
that are never read, and through the backend's methods on tensors in host memory."""
import ctypes
import math

import pytest
import torch
from torch import nn

from rns_llm_amd import HipRNSBackend, RNSCachedAttention, RNSLinear, RNSQKVProjection, _native

CPU = torch.device("cpu")
ADDRESS = 4096  # aligned to anything, never read


def backend():
    b = object.__new__(HipRNSBackend)  # no GPU here
    b._lib = _native.lib()
    b._beam_checked = {}
    return b


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def pool(**changes):
    sizes = dict(device=CPU, blocks=37, block_size=16, sequences=3, width=4)
    sizes.update(changes)
    return backend().create_kv_pool(**sizes)


# ---- pools -------------------------------------------------------------------
def test_an_empty_pool():
    p = pool()
    assert (p.table == -1).all() and p.table.shape == (3, 4) and (p.refs == 0).all() and (p.lengths == 0).all()
    assert p.free.shape == (48,) and p.free[:37].all() and not p.free[37:].any()
    words = _native.lib().rnsmx_kv_pool_scratch_words(37, 3, 4)
    assert words == 3 * 37 + 3 * 4 + 3 and p._scratch.shape == (words,)
    assert not p._scratch[:37].any() and (p._scratch[37:74] == 2 ** 31 - 1).all()
    assert _native.lib().rnsmx_kv_pool_scratch_words(0, 3, 4) == -1


@pytest.mark.parametrize("changes", [{"block_size": 8}, {"blocks": 0}, {"sequences": 0}, {"width": 0}, {"width": 2 ** 26 + 1},
                                     {"blocks": 2 ** 31}])
def test_pools_that_are_none(changes):
    with pytest.raises(ValueError):
        pool(**changes)


def test_steps_bind_their_rows():
    p = pool()
    s = backend().kv_step(p)
    assert s.starts is None and s.batch.rows == 3 and s.batch.max_query == 1 and s.batch.block_table is p.table
    s = backend().kv_step(p, rows=7, max_query=5, max_length=40)
    assert s.starts.shape == (4,) and (s.batch.rows, s.batch.max_query, s.batch.max_length) == (7, 5, 40)
    assert s.copies.tolist() == [[-1, -1, 0]] * 3 and s.missing.tolist() == [0]
    assert backend().kv_step(p, rows=7).batch.max_query == 7 and backend().kv_step(p, rows=0).batch.rows == 0


@pytest.mark.parametrize("options,match", [({"max_query": 2}, "goes with rows"), ({"rows": -1}, "rows"), ({"max_length": 65}, "max_length"),
                                           ({"rows": 2, "max_query": -1}, "max_query"), ({"rows": 2 ** 31}, "too many rows")])
def test_steps_that_are_none(options, match):
    with pytest.raises(ValueError, match=match):
        backend().kv_step(pool(), **options)


def test_numbers_of_all_sequences():
    p, b = pool(), backend()
    s = b.kv_step(p)
    for call in (lambda x: b.kv_trim(p, x), lambda x: b.kv_reorder(p, x), lambda x: b.kv_assign(p, s, x)):
        for bad, match in ((ints(1, 2), "3 elements"), (torch.zeros(3), "int32"), (torch.zeros(3, dtype=torch.int64), "int32"),
                           (torch.zeros((3, 1), dtype=torch.int32), "1-dimensional"), (ints(1, 1, 2, 2, 3, 3)[::2], "contiguous"),
                           (torch.zeros(3, dtype=torch.int32, device="meta"), "on cpu"), (ints(1, 2, 3), "on the GPU")):
            with pytest.raises(ValueError, match=match):
                call(bad)
    with pytest.raises(ValueError, match="on the GPU"):
        b.kv_assign(p, s)
    with pytest.raises(ValueError, match="another pool"):
        b.kv_assign(pool(), s)


def test_copies_and_slots_refuse():
    p, b = pool(), backend()
    s = b.kv_step(p)
    for sizes, match in (({"blocks": 36}, "37 pages"), ({"block_size": 32}, "of 16 tokens"), ({}, "on the GPU")):
        options = dict(device=CPU, blocks=37, block_size=16, kv_heads=2, head_dim=40)
        options.update(sizes)
        with pytest.raises(ValueError, match=match):
            b.kv_copy(b.create_kv_cache(**options), s)
    with pytest.raises(ValueError, match="on the GPU"):
        b.kv_slots(p, s.batch)


# ---- rotary ------------------------------------------------------------------
def rotary(**changes):
    options = dict(device=CPU, rotary_dim=8)
    options.update(changes)
    return backend().create_rotary(**options)


def test_steps_of_frequencies():
    r = rotary(frequencies=[0.0, 2 * math.pi, math.pi, -math.pi / 2])
    got = [int(v) % 2 ** 64 for v in r.steps]
    for g, turn in zip(got, (0.0, 1.0, 0.5, -0.25)):  # float64 pi is off by 2^-53 of itself at most
        off = (g - round(turn * 2 ** 64)) % 2 ** 64
        assert min(off, 2 ** 64 - off) < 2 ** 12
    assert rotary(layout="interleaved").interleaved and not rotary().interleaved


@pytest.mark.parametrize("options", [
    {"rotary_dim": 7}, {"rotary_dim": 0}, {"rotary_dim": 1026}, {"layout": "both"}, {"scaling": "other"}, {"factor": 2.0},
    {"scaling": "linear", "factor": 0.0}, {"scaling": "linear", "factor": math.inf}, {"scaling": "base", "rotary_dim": 2, "factor": 2.0},
    {"scaling": "bands", "factor": 2.0}, {"scaling": "bands", "factor": 2.0, "original_length": 100, "low_turns": 4.0, "high_turns": 4.0},
    {"base": 0.0}, {"base": math.nan}, {"magnitude": math.inf}, {"frequencies": [1.0] * 3}, {"frequencies": [1.0, 1.0, 1.0, math.nan]},
    {"frequencies": [1.0] * 4, "scaling": "linear"},
])
def test_rotaries_that_are_none(options):
    with pytest.raises(ValueError):
        rotary(**options)


def heads(n=2, h=3, dim=10, dtype=torch.float16):
    return torch.zeros((n, h, dim), dtype=dtype)


@pytest.mark.parametrize("positions,q,k,options,match", [
    (ints(1, 2), heads(dtype=torch.float64), None, {}, "q must be float32"),
    (ints(1, 2), heads(), heads(dtype=torch.float32), {}, "one dtype"),
    (ints(1, 2), heads(dim=7), None, {}, "q must be"),
    (ints(1, 2), heads()[0], None, {}, "q must be"),
    (ints(1, 2), heads(dim=1026), None, {}, "q must be"),
    (ints(1, 2), heads(), heads(n=3), {}, "one number of rows"),
    (ints(1, 2), heads(), heads(dim=12), {}, "one head dimension"),
    (ints(1, 2, 3), heads(), None, {}, "one number of rows"),
    (torch.zeros(2), heads(), None, {}, "positions must be"),
    (torch.zeros((2, 1), dtype=torch.int32), heads(), None, {}, "positions must be"),
    (torch.zeros(2, dtype=torch.int32, device="meta"), heads(), None, {}, "positions must be"),
    (ints(1, 2), torch.zeros((2, 3, 10), device="meta"), None, {}, "on cpu"),
    (ints(1, 2), heads(h=1).expand(2, 3, 10), None, {"inplace": True}, "lie apart"),
    (ints(1, 2), heads(n=1).expand(2, 3, 10), None, {"inplace": True}, "lie apart"),
    (ints(1, 2), torch.zeros((2, 10, 3), dtype=torch.float16).transpose(1, 2), None, {"inplace": True}, "lie apart"),
    (ints(1, 2), torch.zeros(80, dtype=torch.float16).as_strided((2, 3, 10), (20, 10, 1)), None, {"inplace": True}, "lie apart"),
    (ints(1, 2), heads().requires_grad_(), None, {"inplace": True}, "no gradient"),
    (ints(1, 2), heads(), None, {}, "on the GPU"),
])
def test_rotations_that_are_none(positions, q, k, options, match):
    with pytest.raises(ValueError, match=match):
        backend().rotate(rotary(), positions, q, k, **options)


def test_the_layer_takes_rotary_positions_that_fit():
    projection = RNSQKVProjection(RNSLinear(8, 24, mode="torch"), (8, 8, 8))
    make = lambda r: RNSCachedAttention(projection, nn.Identity(), backend=None, num_heads=2, rotary=r)  # noqa: E731
    assert make(rotary(rotary_dim=4)).rotary.rotary_dim == 4
    with pytest.raises(ValueError, match="do not fit"):
        make(rotary(rotary_dim=6))


# ---- beams -------------------------------------------------------------------
def logits(r=2, b=3, v=5, dtype=torch.float32):
    return torch.zeros((r, b, v), dtype=dtype)


@pytest.mark.parametrize("x,scores,k,options,match", [
    (logits(dtype=torch.float64), torch.zeros(2, 3), 2, {}, "logits must be"),
    (logits()[0], torch.zeros(2, 3), 2, {}, "logits must be"),
    (logits(), torch.zeros(2, 2), 2, {}, "scores must be"),
    (logits(), torch.zeros(2, 3, dtype=torch.float16), 2, {}, "scores must be"),
    (logits(), torch.zeros(2, 3, device="meta"), 2, {}, "scores must be"),
    (logits(), torch.zeros(2, 3), 0, {}, "1 to 64"),
    (logits(), torch.zeros(2, 3), 65, {}, "1 to 64"),
    (logits(b=0), torch.zeros(2, 0), 2, {}, "1 to 64"),
    (logits(b=65), torch.zeros(2, 65), 2, {}, "1 to 64"),
    (logits(v=0), torch.zeros(2, 3), 2, {}, "at least one token"),
    (logits(), torch.zeros(2, 3), 2, {"finished": torch.zeros(2, 3)}, "finished must be"),
    (logits(), torch.zeros(2, 3), 2, {"finished": torch.zeros(2, 2, dtype=torch.bool)}, "finished must be"),
    (logits(), torch.zeros(2, 3), 2, {"finished": torch.zeros(2, 3, dtype=torch.bool)}, "need an end_token"),
    (logits(), torch.zeros(2, 3), 2, {"end_token": 5}, "of the vocabulary"),
    (logits(), torch.zeros(2, 3), 2, {"end_token": -1}, "of the vocabulary"),
    (logits(), torch.zeros(2, 3), 2, {}, "on the GPU"),
])
def test_selections_that_are_none(x, scores, k, options, match):
    with pytest.raises(ValueError, match=match):
        backend().beam_select(x, scores, k, **options)
    with pytest.raises(TypeError):
        backend().beam_select(x, scores, 1.5)
    with pytest.raises(TypeError):
        backend().beam_select(x, scores, 1, end_token=0.5)


# ---- the C ABI ---------------------------------------------------------------
def refused(rc, match, code=_native.EINVAL):
    assert rc == code and match in _native.lib().rnsmx_last_error().decode()


def pool_struct(**changes):
    values = dict(table_dev=ADDRESS, lengths_dev=ADDRESS, refs_dev=ADDRESS, free_dev=ADDRESS, scratch_dev=ADDRESS, blocks=9, page=16,
                  seqs=2, width=3)
    values.update(changes)
    return _native.KVPoolStruct(**values)


def step_struct(**changes):
    values = dict(lengths_dev=ADDRESS, starts_dev=None, copies_dev=ADDRESS, missing_dev=ADDRESS, rows=2, max_rows=1, max_length=48)
    values.update(changes)
    return _native.KVStepStruct(**values)


@pytest.mark.parametrize("changes,match", [
    ({"page": 48}, "16, 32, 64 or 128"), ({"blocks": 0}, "a pool has"), ({"seqs": 0}, "a pool has"), ({"width": 0}, "a pool has"),
    ({"width": 2 ** 27}, "2^30"), ({"table_dev": None}, "null"), ({"lengths_dev": 4098}, "boundary"), ({"refs_dev": None}, "null"),
    ({"free_dev": 4104}, "16-byte"), ({"scratch_dev": None}, "null"),
])
def test_pools_the_library_refuses(changes, match):
    lib, p, s = _native.lib(), pool_struct(**changes), step_struct()
    refused(lib.rnsmx_kv_assign(ctypes.byref(p), ctypes.byref(s), ADDRESS, None), match)
    refused(lib.rnsmx_kv_trim(ctypes.byref(p), ADDRESS, None), match)
    refused(lib.rnsmx_kv_reorder(ctypes.byref(p), ADDRESS, None), match)


def test_steps_the_library_refuses():
    lib, p = _native.lib(), pool_struct()
    ref = ctypes.byref(p)
    refused(lib.rnsmx_kv_assign(None, ctypes.byref(step_struct()), None, None), "null pool")
    refused(lib.rnsmx_kv_assign(ref, None, None, None), "null step")
    for changes in ({"lengths_dev": None}, {"copies_dev": None}, {"missing_dev": None}, {"starts_dev": 4098}, {"lengths_dev": 4098}):
        refused(lib.rnsmx_kv_assign(ref, ctypes.byref(step_struct(**changes)), None, None), "null or not on")
    for changes in ({"rows": -1}, {"max_rows": -1}, {"max_length": -1}):
        refused(lib.rnsmx_kv_assign(ref, ctypes.byref(step_struct(**changes)), None, None), "bad step")
    refused(lib.rnsmx_kv_assign(ref, ctypes.byref(step_struct()), 4098, None), "null or not on")
    refused(lib.rnsmx_kv_trim(ref, None, None), "lengths null")
    refused(lib.rnsmx_kv_reorder(ref, 4098, None), "parents null")


def test_slots_and_copies_the_library_refuses():
    lib = _native.lib()
    make = lambda **c: _native.KVBatchStruct(**{**dict(table_dev=ADDRESS, table_stride=3, lengths_dev=ADDRESS, starts_dev=ADDRESS, seqs=2,  # noqa: E731
                                                       table_width=3, rows=5, max_rows=4, max_length=48), **c})
    call = lambda b, blocks=9, page=16, p=ADDRESS, s=ADDRESS: lib.rnsmx_kv_slots(ctypes.byref(b), blocks, page, p, s, None)  # noqa: E731
    refused(lib.rnsmx_kv_slots(None, 9, 16, ADDRESS, ADDRESS, None), "null batch")
    refused(call(make(), page=20), "16, 32, 64 or 128")
    for changes in ({"seqs": -1}, {"rows": -1}, {"max_rows": -1}, {"table_width": 0}, {"table_stride": -1}, {"max_length": -1}):
        refused(call(make(**changes)), "bad batch")
    refused(call(make(), blocks=0), "bad batch")
    refused(call(make(max_length=49)), "past the block table")
    refused(call(make(starts_dev=None)), "one row a sequence")
    refused(call(make(table_dev=None)), "null")
    refused(call(make(), p=None), "null")
    refused(call(make(), s=4100), "aligned")
    assert call(make(rows=0)) == _native.OK

    cache = lambda **c: _native.KVCacheStruct(**{**dict(k_dev=ADDRESS, v_dev=ADDRESS, scales_dev=ADDRESS, blocks=9, page=16, heads=2,  # noqa: E731
                                                        head_dim=40, row_bytes=64), **c})
    copy = lambda c, at=ADDRESS, n=3: lib.rnsmx_kv_copy(ctypes.byref(c), at, n, None)  # noqa: E731
    refused(lib.rnsmx_kv_copy(None, ADDRESS, 1, None), "null cache")
    for changes in ({"page": 8}, {"blocks": 0}, {"heads": 0}, {"row_bytes": 40}, {"head_dim": 300, "row_bytes": -1}):
        refused(copy(cache(**changes)), "bad cache")
    for changes in ({"k_dev": None}, {"v_dev": 4104}, {"scales_dev": 4100}):
        refused(copy(cache(**changes)), "boundaries")
    refused(copy(cache(), n=-1), "too many copies")
    refused(copy(cache(heads=2 ** 20), n=2 ** 12), "too many copies")
    refused(copy(cache(), at=None), "copies null")
    assert copy(cache(), at=None, n=0) == _native.OK


def rows_struct(**changes):
    values = dict(rows=2, q_row_stride=24, q_head_stride=8, k_row_stride=16, k_head_stride=8, q_out_row_stride=24, q_out_head_stride=8,
                  k_out_row_stride=16, k_out_head_stride=8, q_heads=3, k_heads=2, head_dim=8, dtype=_native.FLOAT16,
                  positions_dtype=_native.INT32, back=0)
    values.update(changes)
    return _native.RotaryRowsStruct(**values)


def turn(rows=None, positions=ADDRESS, q=1 << 20, k=2 << 20, qo=3 << 20, ko=4 << 20, **changes):
    values = dict(steps_dev=ADDRESS, pairs=4, interleaved=0, magnitude=1.0)
    values.update(changes)
    r, s = _native.RotaryStruct(**values), rows_struct() if rows is None else rows
    return _native.lib().rnsmx_rotate(ctypes.byref(r), ctypes.byref(s), positions, q, k, qo, ko, None)


def test_rotations_the_library_refuses():
    lib = _native.lib()
    refused(lib.rnsmx_rotate(None, ctypes.byref(rows_struct()), None, None, None, None, None, None), "null rotary")
    for changes, match in (({"pairs": 0}, "pairs"), ({"pairs": 5}, "pairs"), ({"magnitude": math.nan}, "magnitude"),
                           ({"steps_dev": None}, "steps"), ({"steps_dev": 4100}, "steps")):
        refused(turn(**changes), match)
    for changes, match in (({"dtype": _native.INT8}, "float32"), ({"positions_dtype": _native.INT16}, "int32 or int64"),
                           ({"rows": -1}, "row sizes"), ({"head_dim": 1025}, "row sizes"), ({"q_heads": -1}, "row sizes"),
                           ({"q_heads": 4096}, "row sizes"), ({"k_row_stride": -16}, "negative"), ({"rows": 2 ** 31}, "too many rows")):
        refused(turn(rows_struct(**changes)), match)
    refused(turn(positions=None), "positions")
    refused(turn(q=None), "null")
    refused(turn(ko=4097), "aligned")
    # outputs over inputs, their own apart: q's over k, and q's over its own rows moved on
    refused(turn(qo=2 << 20), "lie over")
    refused(turn(qo=(1 << 20) + 16), "lie over")
    # queries and keys that share values, in place: the same, some heads, rows moved on, other strides
    at = 1 << 20
    for k, changes in ((at, {}), (at + 16, {}), (at + 2 * 24 * 2, {}), (at + 2 * 20, {}), (at + 2 * 16, {"k_row_stride": 20})):
        both = {"rows": 4, "k_row_stride": 24}
        both.update(changes)
        both.update(k_out_row_stride=both["k_row_stride"])
        refused(turn(rows_struct(**both), q=at, qo=at, k=k, ko=k), "share values")
    assert turn(rows_struct(rows=0)) == _native.OK and turn(rows_struct(q_heads=0, k_heads=0)) == _native.OK


def beams_struct(**changes):
    values = dict(request_stride=15, beam_stride=5, dtype=_native.FLOAT32, requests=2, beams=3, vocabulary=5, k=4, end_token=-1)
    values.update(changes)
    return _native.BeamsStruct(**values)


def select(b=None, x=ADDRESS, s=ADDRESS, f=None, space=ADDRESS, size=1 << 30, o=ADDRESS, t=ADDRESS, p=ADDRESS):
    b = beams_struct() if b is None else b
    return _native.lib().rnsmx_beam_select(ctypes.byref(b), x, s, f, space, size, o, t, p, None)


def test_selections_the_library_refuses():
    lib = _native.lib()
    refused(lib.rnsmx_beam_select(None, None, None, None, None, 0, None, None, None, None), "null beams")
    for changes, match in (({"dtype": _native.INT8}, "float32"), ({"requests": -1}, "1 to 64"), ({"beams": 0}, "1 to 64"),
                           ({"beams": 65}, "1 to 64"), ({"vocabulary": 0}, "1 to 64"), ({"k": 0}, "1 to 64"), ({"k": 65}, "1 to 64"),
                           ({"beam_stride": -1}, "negative"), ({"beams": 64, "vocabulary": 2 ** 18 + 1}, "too many tokens"),
                           ({"requests": 2 ** 30, "beams": 3}, "too many requests")):
        refused(select(beams_struct(**changes)), match)
        assert lib.rnsmx_beam_workspace_bytes(ctypes.byref(beams_struct(**changes))) == -1
    assert lib.rnsmx_beam_workspace_bytes(ctypes.byref(beams_struct(beams=64, vocabulary=2 ** 18))) > 0
    for changes in ({"x": None}, {"x": 4098}, {"s": None}):
        refused(select(**changes), "logits or scores")
    for changes in ({"o": None}, {"t": 4098}, {"p": None}):
        refused(select(**changes), "output")
    refused(select(f=ADDRESS), "end token")
    refused(select(beams_struct(end_token=5), f=ADDRESS), "end token")
    refused(select(space=None), "workspace")
    refused(select(size=16), "too small", _native.ESPACE)
    assert select(beams_struct(requests=0)) == _native.OK
