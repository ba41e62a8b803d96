"""The cache in pages and trees without a device: the restatement against itself, the layout's size,
and every refusal of the entry points (before any device access)."""
import ctypes

import numpy as np
import pytest

from oracle import paged_ref


def _cache(**change):
    from kotensor_amd import _lib
    c = _lib.PagedCache()
    c.keys, c.values, c.format, c.layers, c.pages, c.kv_heads, c.page_tokens, c.head_dim = 4096, 4096, 0, 2, 10, 2, 32, 64
    for name, value in change.items():
        setattr(c, name, value)
    return ctypes.byref(c)


def _batch(**change):
    from kotensor_amd import _lib
    b = _lib.PagedBatch()
    b.tables, b.lengths, b.starts, b.table_stride, b.sequences, b.rows, b.most_rows, b.key_bound = 4096, 4096, 4096, 4, 3, 8, 5, 100
    for name, value in change.items():
        setattr(b, name, value)
    return ctypes.byref(b)


TREE = {"depths": 4096, "masks": 4096, "mask_words": 1}


def test_roundings():
    x = np.array([1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 1 + 2.0 ** -8 + 2.0 ** -20, -3.0e38, 65519.0, 65520.0, 1e-40, np.nan, np.inf], np.float32)
    assert paged_ref.stored(x, "bfloat16")[:4].tolist() == [1.0, 1.0, 1 + 2.0 ** -6, 1 + 2.0 ** -7]
    half = paged_ref.stored(x, "float16")
    assert half[5] == 65504.0 and np.isinf(half[6]) and np.isnan(half[8]) and np.isinf(half[9])
    assert np.array_equal(paged_ref.stored(x, "float32"), x, equal_nan=True)


def test_trees_by_hand():
    #       0
    #     1   2
    #    3   4 5
    #           6       7: another root
    parents = [-1, 0, 0, 1, 2, 2, 5, 9]
    depths, bits = paged_ref.masks(parents, 2)
    assert depths.tolist() == [0, 1, 1, 2, 2, 2, 3, 0]
    assert bits[:, 0].tolist() == [1, 3, 5, 11, 21, 37, 101, 128] and not bits[:, 1].any()
    assert paged_ref.accept(parents, [9, 4, 5, 1, 2, 2, 3, 5], [5, 0, 2, 0, 0, 8, 0, 0]) == [0, 2, 4]
    assert paged_ref.accept(parents, [9, 4, 5, 1, 1, 2, 3, 5], [5, 0, 2, 0, 0, 3, 0, 0]) == [0, 2, 5, 6]
    assert paged_ref.accept([], [], []) == []


def test_attention_by_hand():
    q = np.zeros((2, 2, 4))
    q[0, 0] = [2, 0, 0, 0]
    keys, values = np.zeros((1, 3, 4)), np.arange(12.0).reshape(1, 3, 4)
    keys[0, 0, 0] = 1
    see = np.array([[True, True, False], [False, False, False]])
    out, bound = paged_ref.attend(q, keys, values, see)
    w = np.exp(1.0) / (np.exp(1.0) + 1)
    assert np.allclose(out[0, 0], w * values[0, 0] + (1 - w) * values[0, 1]) and np.allclose(out[0, 1], values[0, :2].mean(0))
    assert not out[1].any() and not bound[1].any() and (bound[0] < 1e-3).all()


@pytest.mark.parametrize("fmt,size", [(0, 4), (1, 2), (2, 2)])
def test_layout(fmt, size):
    from kotensor_amd import _lib
    out = ctypes.c_int64()
    assert _lib.lib().kt_paged_layout(_cache(format=fmt, layers=80, pages=1 << 16, kv_heads=8, page_tokens=256, head_dim=128), ctypes.byref(out)) == _lib.KT_OK
    assert out.value == size * 80 * (1 << 16) * 8 * 256 * 128
    assert _lib.lib().kt_paged_layout(_cache(), None) == _lib.KT_ERR_ARGUMENT


CALLS = {
    "kt_rope_paged": lambda lib, c, b: lib.kt_rope_paged(16, 16, 16, 4, 16, c, 0, b, 16, None),
    "kt_attention_paged": lambda lib, c, b: lib.kt_attention_paged(16, 4, c, 0, b, 16, None),
    "kt_rope_attention_paged": lambda lib, c, b: lib.kt_rope_attention_paged(16, 16, 16, 16, 4, c, 0, b, 16, None),
    "kt_paged_keep": lambda lib, c, b: lib.kt_paged_keep(c, b, 16, 5, 16, 16, None),
}


@pytest.mark.parametrize("change,want,message", [
    ({"format": 3}, "arg", "cache format 3"), ({"format": -1}, "arg", "cache format -1"), ({"layers": 0}, "arg", "must be positive"), ({"pages": 0}, "arg", "must be positive"),
    ({"kv_heads": -1}, "arg", "must be positive"), ({"head_dim": 96}, "arg", "head dimension 96"), ({"head_dim": 16}, "arg", "head dimension 16"),
    ({"page_tokens": 8}, "arg", "8 tokens to a page"), ({"page_tokens": 48}, "arg", "48 tokens to a page"), ({"page_tokens": 512}, "arg", "512 tokens to a page"),
    ({"kv_heads": 70000}, "shape", "at most 65535"), ({"pages": 2**31 - 1, "kv_heads": 65535, "layers": 65535}, "shape", "too large"),
])
def test_shapes_refused(change, want, message):
    from kotensor_amd import _lib
    lib, out = _lib.lib(), ctypes.c_int64()
    want = {"arg": _lib.KT_ERR_ARGUMENT, "shape": _lib.KT_ERR_SHAPE}[want]
    for status in [lib.kt_paged_layout(_cache(**change), ctypes.byref(out)), lib.kt_paged_read(_cache(**change), 0, 16, 4, 0, 1, 16, 16, None)] + \
            [f(lib, _cache(**change), _batch()) for f in CALLS.values()]:
        assert status == want and message in _lib.last_error()


@pytest.mark.parametrize("change,want,message", [
    ({"tables": None}, "arg", "NULL"), ({"lengths": None}, "arg", "NULL"), ({"starts": None}, "arg", "NULL"), ({"sequences": -1}, "arg", "-1 sequences"),
    ({"sequences": 65536}, "arg", "65536 sequences"), ({"rows": -1}, "arg", "rows"), ({"most_rows": 9}, "arg", "at most 9 rows"), ({"most_rows": -1}, "arg", "rows"), ({"rows": 1 << 24}, "shape", "at most 16777215"),
    ({"depths": 16}, "arg", "masks and depths"), ({"masks": 16, "mask_words": 1}, "arg", "masks and depths"), ({**TREE, "mask_words": 0}, "shape", "0 mask words"),
    ({**TREE, "rows": 40, "most_rows": 33}, "shape", "do not hold 33"), ({**TREE, "mask_words": 2**31 - 1}, "shape", "mask words"),
    ({"table_stride": 0}, "arg", "table_stride"), ({"key_bound": 4}, "arg", "key bound 4"), ({"key_bound": 129}, "arg", "128 tokens"), ({"key_bound": (1 << 30) + 1, "table_stride": 1 << 30}, "shape", "key bound 1073741825"),
])
def test_batches_refused(change, want, message):
    from kotensor_amd import _lib
    lib = _lib.lib()
    want = {"arg": _lib.KT_ERR_ARGUMENT, "shape": _lib.KT_ERR_SHAPE}[want]
    for name, f in CALLS.items():
        assert f(lib, _cache(), _batch(**change)) == want and message in _lib.last_error(), (name, _lib.last_error())
        assert f(lib, _cache(), None) == _lib.KT_ERR_ARGUMENT and "batch is NULL" in _lib.last_error()
        assert f(lib, None, _batch()) == _lib.KT_ERR_ARGUMENT and "cache is NULL" in _lib.last_error()


def test_calls_refused():
    from kotensor_amd import _lib
    lib = _lib.lib()

    def refused(status, want, message):
        assert status == want and message in _lib.last_error(), (status, _lib.last_error())
    arg, shape, rng = _lib.KT_ERR_ARGUMENT, _lib.KT_ERR_SHAPE, _lib.KT_ERR_RANGE
    c, b, t = _cache(), _batch(), _batch(**TREE)
    for missing in ("keys", "values"):
        refused(lib.kt_attention_paged(16, 4, _cache(**{missing: None}), 0, b, 16, None), arg, "NULL")
        refused(lib.kt_attention_paged(16, 4, _cache(**{missing: 4104}), 0, b, 16, None), arg, "16-byte aligned")
    for layer in (-1, 2):
        refused(lib.kt_attention_paged(16, 4, c, layer, b, 16, None), rng, f"layer {layer} out of bounds 2")
        refused(lib.kt_rope_paged(16, 16, 16, 4, 16, c, layer, b, 16, None), rng, f"layer {layer}")
        refused(lib.kt_paged_read(c, layer, 16, 4, 0, 1, 16, 16, None), rng, f"layer {layer}")
    for heads in (0, 3, -2):
        refused(lib.kt_attention_paged(16, heads, c, 0, b, 16, None), arg, "multiple of numKeyValueHeads")
        refused(lib.kt_rope_paged(16, 16, 16, heads, 16, c, 0, b, 16, None), arg, "multiple of numKeyValueHeads")
        refused(lib.kt_rope_attention_paged(16, 16, 16, 16, heads, c, 0, b, 16, None), arg, "multiple of numKeyValueHeads")
    # the append
    refused(lib.kt_rope_paged(16, None, 16, 4, 16, c, 0, b, 16, None), arg, "NULL")
    refused(lib.kt_rope_paged(16, 16, None, 4, 16, c, 0, b, 16, None), arg, "NULL")
    refused(lib.kt_rope_paged(16, 16, 16, 4, None, c, 0, b, 16, None), arg, "NULL")
    refused(lib.kt_rope_paged(None, 16, 16, 4, 16, c, 0, b, 16, None), arg, "NULL")
    refused(lib.kt_rope_paged(16, 16, 16, 4, 16, c, 0, b, None, None), arg, "NULL")
    # the attention
    refused(lib.kt_attention_paged(None, 4, c, 0, b, 16, None), arg, "NULL")
    refused(lib.kt_attention_paged(16, 4, c, 0, b, None, None), arg, "NULL")
    refused(lib.kt_attention_paged(20, 4, c, 0, b, 16, None), arg, "16-byte aligned")
    refused(lib.kt_attention_paged(16, 4, c, 0, b, 24, None), arg, "16-byte aligned")
    for i in range(4):
        args = [16, 16, 16, 16]
        args[i] = None
        refused(lib.kt_rope_attention_paged(*args, 4, c, 0, b, 16, None), arg, "NULL")
    refused(lib.kt_rope_attention_paged(16, 16, 16, 16, 4, c, 0, b, None, None), arg, "NULL")
    refused(lib.kt_rope_attention_paged(20, 16, 16, 16, 4, c, 0, b, 16, None), arg, "16-byte aligned")
    # trees
    refused(lib.kt_tree_masks(None, t, 16, 16, None), arg, "NULL")
    refused(lib.kt_tree_masks(16, t, None, 16, None), arg, "NULL")
    refused(lib.kt_tree_masks(16, t, 16, None, None), arg, "NULL")
    refused(lib.kt_tree_masks(16, b, 16, 16, None), arg, "no masks")
    refused(lib.kt_tree_masks(16, None, 16, 16, None), arg, "batch is NULL")
    for i in range(6):
        args = [16] * 6
        args[i] = None
        refused(lib.kt_tree_accept(*args[:3], t, args[3], 5, *args[4:], None), arg, "NULL")
    refused(lib.kt_tree_accept(16, 16, 16, t, 16, 4, 16, 16, None), shape, "kept_stride 4 does not hold 5")
    refused(lib.kt_tree_accept(16, 16, 16, _batch(rows=0, most_rows=0), 16, 0, 16, 16, None), shape, "kept_stride 0")
    # what is kept
    refused(lib.kt_paged_keep(c, t, None, 5, 16, 16, None), arg, "NULL")
    refused(lib.kt_paged_keep(c, t, 16, 5, None, 16, None), arg, "NULL")
    refused(lib.kt_paged_keep(c, t, 16, 5, 16, None, None), arg, "NULL")
    refused(lib.kt_paged_keep(c, t, 16, 0, 16, 16, None), shape, "kept_stride")
    refused(lib.kt_paged_advance(None, b, None), arg, "NULL")
    refused(lib.kt_paged_advance(16, None, None), arg, "batch is NULL")
    # rows
    refused(lib.kt_paged_read(c, 0, None, 4, 0, 1, 16, 16, None), arg, "NULL")
    for entries, first, count in ((0, 0, 0), (-1, 0, 1), (4, -1, 1), (4, 0, 129), (4, 128, 1), (4, 3, -1), (4, 2**31 - 1, 2**31 - 1)):
        refused(lib.kt_paged_read(c, 0, 16, entries, first, count, 16, 16, None), rng, "out of bounds")


def test_calls_of_nothing():
    """No rows, or no sequences: nothing is enqueued."""
    from kotensor_amd import _lib
    lib = _lib.lib()
    for empty in (_batch(rows=0, most_rows=0), _batch(sequences=0)):
        assert lib.kt_rope_paged(16, 16, 16, 4, 16, _cache(), 0, empty, 16, None) == _lib.KT_OK
        assert lib.kt_attention_paged(16, 4, _cache(), 0, empty, 16, None) == _lib.KT_OK
        assert lib.kt_rope_attention_paged(16, 16, 16, 16, 4, _cache(), 0, empty, 16, None) == _lib.KT_OK
    none = _batch(sequences=0, **TREE)
    assert lib.kt_tree_masks(16, none, 16, 16, None) == _lib.KT_OK and lib.kt_paged_keep(_cache(), none, 16, 5, 16, 16, None) == _lib.KT_OK
    assert lib.kt_tree_accept(16, 16, 16, none, 16, 5, 16, 16, None) == _lib.KT_OK and lib.kt_paged_advance(16, none, None) == _lib.KT_OK
    assert lib.kt_paged_read(_cache(), 0, 16, 4, 128, 0, 16, 16, None) == _lib.KT_OK and lib.kt_paged_read(_cache(), 0, 16, 4, 0, 5, None, None, None) == _lib.KT_OK


@pytest.mark.parametrize("tree", [{}, TREE])
def test_calls_without_a_row_of_a_sequence(tree):
    """Rows that belong to no sequence alone, as in a padded batch whose sequences are all empty: nothing is enqueued."""
    from kotensor_amd import _lib
    lib = _lib.lib()
    for bound in (0, 100):
        padding = _batch(most_rows=0, key_bound=bound, **tree)
        assert lib.kt_rope_paged(16, 16, 16, 4, 16, _cache(), 0, padding, 16, None) == _lib.KT_OK, _lib.last_error()
        assert lib.kt_attention_paged(16, 4, _cache(), 0, padding, 16, None) == _lib.KT_OK, _lib.last_error()
        assert lib.kt_rope_attention_paged(16, 16, 16, 16, 4, _cache(), 0, padding, 16, None) == _lib.KT_OK, _lib.last_error()


def test_launches_past_32_bits_of_threads_refused():
    """A launch has fewer than 2^32 threads: more rows and heads, or tokens to read, are refused as such, not by the device."""
    from kotensor_amd import _lib
    lib = _lib.lib()
    rows = (1 << 24) - 1
    many = dict(rows=rows, most_rows=rows, sequences=1, table_stride=1 << 20, key_bound=1 << 24)
    few_keys = dict(rows=1 << 20, most_rows=16, sequences=65535, table_stride=4, key_bound=128)
    for batch, kv, heads, dim in ((many, 1, 128, 32), (many, 2, 130, 64), (many, 8, 128, 128), (many, 4, 256, 256), (few_keys, 512, 512, 32)):
        for fmt in range(3):
            cache = _cache(kv_heads=kv, head_dim=dim, format=fmt)
            assert lib.kt_attention_paged(16, heads, cache, 0, _batch(**batch), 16, None) == _lib.KT_ERR_SHAPE, (kv, heads, dim, fmt, _lib.last_error())
            assert "too many rows and heads" in _lib.last_error()
    wide = _cache(kv_heads=64, head_dim=256)
    assert lib.kt_rope_paged(16, 16, 16, 256, 16, wide, 0, _batch(**many), 16, None) == _lib.KT_ERR_SHAPE and "too many rows and heads" in _lib.last_error()
    assert lib.kt_paged_read(wide, 0, 16, 1 << 20, 0, 1 << 18, 16, 16, None) == _lib.KT_ERR_SHAPE and "too many tokens and heads" in _lib.last_error()
