"""Arguments of the key/value cache's entry points, checked before anything
reaches the GPU: through the C ABI with host addresses that are never read, and
through the backend's methods on a cache that lies in host memory."""
import ctypes
import math

import pytest
import torch

from rns_llm_amd import HipRNSBackend, _native

CPU = torch.device("cpu")


def backend():
    b = object.__new__(HipRNSBackend)  # no GPU here
    b._lib = _native.lib()
    return b


def cache(**changes):
    sizes = dict(device=CPU, blocks=4, block_size=16, kv_heads=2, head_dim=40)
    sizes.update(changes)
    return backend().create_kv_cache(**sizes)


def batch(c=None, **options):
    c = cache() if c is None else c
    return backend().kv_batch(c, torch.zeros((2, 2), dtype=torch.int32), [20, 7], **options)


def test_row_sizes():
    lib = _native.lib()
    sizes = [64, 96, 128, 160, 192, 256]
    for dim in range(1, 257):
        assert lib.rnsmx_kv_row_bytes(dim) == min(s for s in sizes if s >= dim)
    assert lib.rnsmx_kv_row_bytes(0) == lib.rnsmx_kv_row_bytes(257) == lib.rnsmx_kv_row_bytes(-3) == -1


def test_an_empty_cache_reads_as_zero():
    c = cache()
    assert c.k_codes.shape == c.v_codes.shape == (4, 2, 16, 64) and c.scales.shape == (4, 2, 2)
    assert (c.k_codes == 128).all() and c.scales.isfinite().all()
    assert c.nbytes == 2 * 4 * 2 * 16 * 64 + 4 * 4 * 2 * 2


@pytest.mark.parametrize("changes", [{"block_size": 8}, {"block_size": 48}, {"blocks": 0}, {"kv_heads": 0}, {"head_dim": 0},
                                     {"head_dim": 257}])
def test_caches_that_are_none(changes):
    with pytest.raises(ValueError):
        cache(**changes)


@pytest.mark.parametrize("table,lengths,options,match", [
    (torch.zeros((2, 2), dtype=torch.int64), [1, 2], {}, "int32"),
    (torch.zeros(2, dtype=torch.int32), [1, 2], {}, "2-dimensional"),
    (torch.zeros((2, 4), dtype=torch.int32).t()[:2], [1, 2], {}, "contiguous"),
    (torch.zeros((2, 0), dtype=torch.int32), [0, 0], {}, "column"),
    (torch.zeros((2, 2), dtype=torch.int32), [1, 2, 3], {}, "sequences"),
    (torch.zeros((2, 2), dtype=torch.int32), [1, 33], {}, "max_length"),
    (torch.zeros((2, 2), dtype=torch.int32), [1, 20], {"max_length": 19}, "max_length"),
    (torch.zeros((2, 2), dtype=torch.int32), [1, 20], {"max_length": 33}, "max_length"),
    (torch.zeros((2, 2), dtype=torch.int32), [1, -1], {}, "negative"),
    (torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2), {}, "int32"),
    (torch.zeros((2, 2), dtype=torch.int32), [1, 2], {"query_lengths": [1]}, "query_lengths"),
    (torch.zeros((2, 2), dtype=torch.int32), [1, 2], {"query_lengths": [1, -2]}, "negative"),
    (torch.zeros((2, 2), dtype=torch.int32), [1, 2], {"query_starts": torch.zeros(3, dtype=torch.int32)}, "max_query"),
    (torch.zeros((2, 2), dtype=torch.int32), [1, 2],
     {"query_starts": torch.zeros(2, dtype=torch.int32), "rows": 2, "max_query": 1}, "3 elements"),
    (torch.zeros((2, 2), dtype=torch.int32), [1, 2],
     {"query_starts": torch.zeros(3, dtype=torch.int32), "query_lengths": [1, 1]}, "both"),
])
def test_batches_that_are_none(table, lengths, options, match):
    with pytest.raises(ValueError, match=match):
        backend().kv_batch(cache(), table, lengths, **options)


@pytest.mark.parametrize("options,match", [
    ({"rows": 2}, "go with"), ({"max_query": 1}, "go with"), ({"query_lengths": [1, 1], "rows": 2}, "go with"),
    ({"query_lengths": [2 ** 30, 2 ** 30]}, "too many rows"),
    ({"query_starts": torch.zeros(3, dtype=torch.int32), "rows": 2 ** 32, "max_query": 1}, "too many rows"),
])
def test_rows_that_a_batch_does_not_take(options, match):
    with pytest.raises(ValueError, match=match):
        batch(**options)


def test_most_rows_of_a_sequence_are_no_more_than_there_are():
    starts = torch.zeros(3, dtype=torch.int32)
    assert batch(query_starts=starts, rows=2, max_query=2 ** 32).max_query == 2


def test_batches_of_another_device():
    c = cache()
    b = object.__new__(type(batch(c)))
    for name, value in vars(batch(c)).items():
        object.__setattr__(b, name, value)
    object.__setattr__(b, "lengths", torch.empty(2, dtype=torch.int32, device="meta"))
    for call in (lambda: backend().kv_append(c, b, rows(), rows()), lambda: backend().kv_read(c, b, dtype=torch.float16),
                 lambda: backend().kv_attention(rows(heads=4), c, b)):
        with pytest.raises(ValueError, match="batch must be on"):
            call()


def test_scales_and_windows_are_taken_by_value():
    """Numbers of any kind: a tensor's value, not which tensor it is."""
    c = cache()
    with pytest.raises(ValueError, match="scale"):
        backend().kv_attention(rows(heads=4), c, batch(c), scale=torch.tensor(-1.0))
    with pytest.raises(ValueError, match="window"):
        backend().kv_attention(rows(heads=4), c, batch(c), window=torch.tensor(0))
    with pytest.raises(TypeError):
        backend().kv_attention(rows(heads=4), c, batch(c), window=1.5)


def test_batches_bind_their_rows():
    b = batch()
    assert (b.rows, b.max_query, b.max_length, b.query_starts, b.sequences) == (2, 1, 32, None, 2)
    b = batch(query_lengths=[3, 0], max_length=20)
    assert (b.rows, b.max_query, b.max_length) == (3, 3, 20) and b.query_starts.tolist() == [0, 3, 3]
    assert batch(query_lengths=[1, 1]).query_starts is None


def rows(n=2, heads=2, dim=40, dtype=torch.float16):
    return torch.zeros((n, heads, dim), dtype=dtype)


@pytest.mark.parametrize("k,v,match", [
    (rows(3), rows(), "k must be"), (rows(), rows(heads=4), "v must be"), (rows(dim=64), rows(), "k must be"),
    (rows()[0], rows(), "k must be"), (rows(dtype=torch.float64), rows(), "float32"), (rows(), rows(dtype=torch.float32), "one dtype"),
])
def test_rows_that_do_not_fit(k, v, match):
    c = cache()
    with pytest.raises(ValueError, match=match):
        backend().kv_append(c, batch(c), k, v)


def test_read_types():
    c = cache()
    with pytest.raises(ValueError, match="dtype"):
        backend().kv_read(c, batch(c), dtype=torch.int8)


@pytest.mark.parametrize("options,match", [
    ({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"), ({"scale": math.nan}, "scale"), ({"scale": math.inf}, "scale"),
    ({"window": 0}, "window"), ({"window": 4, "causal": False}, "window"),
    ({"mask": torch.zeros((2, 1, 32), dtype=torch.int32)}, "mask"), ({"mask": torch.zeros((2, 32))}, "mask"),
    ({"mask": torch.zeros((3, 1, 32))}, "mask"), ({"mask": torch.zeros((2, 3, 32))}, "mask"),
    ({"mask": torch.zeros((2, 1, 19))}, "19 tokens"), ({"out": torch.zeros((2, 4, 40))}, "out"),
    ({"out": torch.zeros((4, 2, 40), dtype=torch.float16).transpose(0, 1)}, "out"),
])
def test_attention_arguments(options, match):
    c = cache()
    with pytest.raises(ValueError, match=match):
        backend().kv_attention(rows(heads=4), c, batch(c), **options)


@pytest.mark.parametrize("q", [rows(heads=3), rows(3, heads=4), rows(heads=4, dim=39), rows(heads=4, dtype=torch.int8), rows(heads=0)])
def test_queries_that_do_not_fit(q):
    c = cache()
    with pytest.raises(ValueError, match="q "):
        backend().kv_attention(q, c, batch(c))


def call(cache_changes=(), batch_changes=(), query_changes=(), q_dev=4096, mask_dev=None, out_dev=4096):
    """rnsmx_kv_attention with valid sizes but for the changes, on zero
    sequences, so that nothing is launched."""
    c = _native.KVCacheStruct(4096, 8192, 4096, 4, 16, 2, 40, 64)
    b = _native.KVBatchStruct(4096, 2, 4096, 4096, 0, 2, 0, 1, 32)
    q = _native.KVQueryStruct(80, 40, 0, 0, 0, _native.FLOAT16, 4, 0, 0, 1, 0, 0.5)
    for struct, changes in ((c, cache_changes), (b, batch_changes), (q, query_changes)):
        for name, value in dict(changes).items():
            setattr(struct, name, value)
    return _native.lib().rnsmx_kv_attention(ctypes.addressof(c), ctypes.addressof(b), ctypes.addressof(q), q_dev, mask_dev,
                                             None, 0, out_dev, None)


def test_c_abi_accepts_no_sequences():
    assert call() == _native.OK


WITH_ROWS = {"seqs": 1, "rows": 1}  # past the call of zero sequences; refused before a launch


@pytest.mark.parametrize("changes", [
    {"cache_changes": {"page": 24}}, {"cache_changes": {"blocks": 0}}, {"cache_changes": {"heads": 0}},
    {"cache_changes": {"head_dim": 300}}, {"cache_changes": {"row_bytes": 96}}, {"cache_changes": {"k_dev": None}},
    {"cache_changes": {"v_dev": 8200}}, {"cache_changes": {"scales_dev": 4100}}, {"batch_changes": {"seqs": -1}},
    {"batch_changes": {"rows": -1}}, {"batch_changes": {"table_width": 0}}, {"batch_changes": {"max_length": 33}},
    {"batch_changes": {"seqs": 65536}, "cache_changes": {"heads": 65536}, "query_changes": {"q_heads": 65536}},
    {"batch_changes": {"seqs": 2 ** 31 - 1}, "cache_changes": {"heads": 2 ** 30}, "query_changes": {"q_heads": 2 ** 30}},
    {"batch_changes": {"rows": 2 ** 30, "max_rows": 2 ** 30}, "query_changes": {"q_heads": 8}},
    {"batch_changes": {"lengths_dev": 4098}}, {"batch_changes": {"table_dev": 4097}}, {"batch_changes": {"starts_dev": 4099}},
    {"batch_changes": {"seqs": 2, "lengths_dev": None}}, {"batch_changes": {"seqs": 2, "starts_dev": None, "rows": 3}},
    {"query_changes": {"dtype": _native.INT8}}, {"query_changes": {"q_heads": 3}}, {"query_changes": {"q_heads": 0}},
    {"query_changes": {"scale": 0.0}}, {"query_changes": {"scale": math.inf}}, {"query_changes": {"window": -1}},
    {"query_changes": {"window": 5, "causal": 0}},
    {"batch_changes": WITH_ROWS, "query_changes": {"mask_dtype": _native.INT32}, "mask_dev": 4096},
    {"batch_changes": WITH_ROWS, "query_changes": {"mask_dtype": _native.FLOAT16}, "mask_dev": 4097},
    {"batch_changes": WITH_ROWS, "query_changes": {"mask_dtype": _native.INT8, "mask_len": -1}, "mask_dev": 4096},
    {"batch_changes": WITH_ROWS, "q_dev": None}, {"batch_changes": WITH_ROWS, "q_dev": 4097},
    {"batch_changes": WITH_ROWS, "out_dev": None}, {"batch_changes": WITH_ROWS, "out_dev": 4099},
])
def test_c_abi_refuses(changes):
    assert call(**changes) == _native.EINVAL
    assert _native.lib().rnsmx_last_error()
    with pytest.raises(ValueError):
        _native.check(_native.EINVAL)
