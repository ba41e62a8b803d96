"""The 8-bit KV cache and the logits controls without a device: the format's restatement against
itself, the layout's sizes, and every refusal of the entry points (before any device access)."""
import ctypes

import numpy as np
import pytest

from oracle import kv8_ref


def _cache(**change):
    from kotensor_amd import _lib
    c = _lib.KV8Cache()
    for name in ("keys", "values", "key_scales", "value_scales", "key_rows", "value_rows"):
        setattr(c, name, 4096)
    c.format, c.layers, c.kv_heads, c.max_seq, c.head_dim, c.block_tokens = _lib.KT_KV8_INT8, 2, 2, 100, 64, 64
    for name, value in change.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("max_seq,block,slots", [(1, 32, 64), (64, 64, 64), (65, 32, 128), (100, 128, 128), (129, 128, 256), (8192, 64, 8192)])
def test_layout(max_seq, block, slots):
    from kotensor_amd import _lib
    out = (ctypes.c_int64 * 3)()
    c = _cache(max_seq=max_seq, block_tokens=block, head_dim=128, layers=3, kv_heads=5)
    assert _lib.lib().kt_kv8_layout(ctypes.byref(c), out) == _lib.KT_OK
    assert list(out) == [15 * slots * 128, 15 * slots // block, 15 * block * 128]


def test_layout_passes_32_bits():
    from kotensor_amd import _lib
    out = (ctypes.c_int64 * 3)()
    c = _cache(max_seq=1 << 20, head_dim=128, layers=80, kv_heads=8)
    assert _lib.lib().kt_kv8_layout(ctypes.byref(c), out) == _lib.KT_OK
    assert out[0] == 80 * 8 * (1 << 20) * 128


@pytest.mark.parametrize("change,message", [
    ({"format": 2}, "cache format 2"), ({"layers": 0}, "must be positive"), ({"kv_heads": -1}, "must be positive"), ({"max_seq": 0}, "must be positive"),
    ({"max_seq": 2**31 - 1}, "too large"), ({"head_dim": 96}, "head dimension 96"), ({"head_dim": 16}, "head dimension 16"), ({"block_tokens": 16}, "16 tokens to a block"),
    ({"block_tokens": 48}, "48 tokens to a block"),
])
def test_shapes_refused(change, message):
    from kotensor_amd import _lib
    out = (ctypes.c_int64 * 3)()
    lib, c = _lib.lib(), _cache(**change)
    assert lib.kt_kv8_layout(ctypes.byref(c), out) == _lib.KT_ERR_ARGUMENT and message in _lib.last_error()
    for status in (lib.kt_rope_kv8(16, 16, 16, 1, 4, 16, 16, ctypes.byref(c), 0, 16, None),
                   lib.kt_attention_kv8(16, 1, 16, 1, ctypes.byref(c), 0, 4, 16, None),
                   lib.kt_rope_attention_kv8(16, 16, 16, 16, 1, 16, 1, ctypes.byref(c), 0, 4, 16, None),
                   lib.kt_kv8_read(ctypes.byref(c), 0, 0, 1, 16, 16, None),
                   lib.kt_kv8_copy(ctypes.byref(c), 1, ctypes.byref(_cache()), 1, None), lib.kt_kv8_copy(ctypes.byref(_cache()), 1, ctypes.byref(c), 1, None)):
        assert status == _lib.KT_ERR_ARGUMENT and message in _lib.last_error()


def test_calls_refused():
    from kotensor_amd import _lib
    lib, good = _lib.lib(), ctypes.byref(_cache())

    def refused(status, want, message):
        assert status == want and message in _lib.last_error(), (status, _lib.last_error())
    arg, shape, rng = _lib.KT_ERR_ARGUMENT, _lib.KT_ERR_SHAPE, _lib.KT_ERR_RANGE
    for missing in ("keys", "values", "key_scales", "value_scales", "key_rows", "value_rows"):
        refused(lib.kt_attention_kv8(16, 1, 16, 1, ctypes.byref(_cache(**{missing: None})), 0, 4, 16, None), arg, "NULL")
    refused(lib.kt_attention_kv8(16, 1, 16, 1, ctypes.byref(_cache(values=4104)), 0, 4, 16, None), arg, "16-byte aligned")
    refused(lib.kt_attention_kv8(16, 1, 16, 1, None, 0, 4, 16, None), arg, "cache is NULL")
    # the append
    refused(lib.kt_rope_kv8(16, None, 16, 1, 4, 16, 16, good, 0, 16, None), arg, "NULL")
    refused(lib.kt_rope_kv8(16, 16, 16, 1, 4, 16, None, good, 0, 16, None), arg, "NULL")
    refused(lib.kt_rope_kv8(16, 16, 16, 1, 4, 16, 16, good, 0, None, None), arg, "NULL")
    refused(lib.kt_rope_kv8(None, 16, 16, 1, 4, 16, 16, good, 0, 16, None), arg, "NULL")
    refused(lib.kt_rope_kv8(16, 16, 16, 1, 5, 16, 16, good, 0, 16, None), arg, "multiple of numKeyValueHeads")
    refused(lib.kt_rope_kv8(16, 16, 16, 1, 0, 16, 16, good, 0, 16, None), arg, "multiple of numKeyValueHeads")
    refused(lib.kt_rope_kv8(16, 16, 16, -1, 4, 16, 16, good, 0, 16, None), arg, "do not fit")
    refused(lib.kt_rope_kv8(16, 16, 16, 101, 4, 16, 16, good, 0, 16, None), arg, "do not fit")
    refused(lib.kt_rope_kv8(16, 16, 16, 1, 4, 16, 16, good, 2, 16, None), rng, "layer 2 out of bounds 2")
    assert lib.kt_rope_kv8(16, 16, 16, 0, 4, 16, 16, good, 1, 16, None) == _lib.KT_OK
    # the attention
    refused(lib.kt_attention_kv8(None, 1, 16, 1, good, 0, 4, 16, None), arg, "NULL")
    refused(lib.kt_attention_kv8(16, 1, 16, 1, good, 0, 4, None, None), arg, "NULL")
    refused(lib.kt_attention_kv8(16, 1, 16, 0, good, 0, 4, 16, None), arg, "key bound 0")
    refused(lib.kt_attention_kv8(16, 1, 16, 101, good, 0, 4, 16, None), arg, "key bound 101")
    refused(lib.kt_attention_kv8(16, -1, 16, 1, good, 0, 4, 16, None), arg, "key bound")
    refused(lib.kt_attention_kv8(20, 1, 16, 1, good, 0, 4, 16, None), arg, "16-byte aligned")
    refused(lib.kt_attention_kv8(16, 1, 16, 1, good, 0, 4, 24, None), arg, "16-byte aligned")
    refused(lib.kt_attention_kv8(16, 1, 16, 1, good, -1, 4, 16, None), rng, "layer -1")
    wide = ctypes.byref(_cache(max_seq=2_000_000))
    refused(lib.kt_attention_kv8(16, 524_281, 16, 524_281, wide, 0, 4, 16, None), shape, "at most 1048560 rows")
    refused(lib.kt_rope_attention_kv8(16, 16, 16, 16, 2_000_000, 16, 2_000_000, wide, 0, 4000, 16, None), shape, "at most 1048560 rows")
    assert lib.kt_attention_kv8(16, 0, 16, 0, good, 0, 4, 16, None) == _lib.KT_OK
    refused(lib.kt_rope_attention_kv8(None, 16, 16, 16, 1, 16, 1, good, 0, 4, 16, None), arg, "NULL")
    refused(lib.kt_rope_attention_kv8(16, 16, 16, None, 1, 16, 1, good, 0, 4, 16, None), arg, "NULL")
    refused(lib.kt_rope_attention_kv8(16, 16, 16, 16, 1, 16, 0, good, 0, 4, 16, None), arg, "key bound 0")
    refused(lib.kt_rope_attention_kv8(16, 16, 16, 16, 2, 16, 101, good, 0, 4, 16, None), arg, "key bound 101")
    refused(lib.kt_rope_attention_kv8(20, 16, 16, 16, 2, 16, 2, good, 0, 4, 16, None), arg, "16-byte aligned")
    refused(lib.kt_rope_attention_kv8(16, 16, 16, 16, 1, 16, 1, good, 0, 3, 16, None), arg, "multiple of numKeyValueHeads")
    # rows and copies
    for first, count in ((-1, 1), (0, 101), (100, 1), (50, -1), (2**31 - 1, 1)):
        refused(lib.kt_kv8_read(good, 0, first, count, 16, 16, None), rng, "out of bounds 100")
    refused(lib.kt_kv8_read(good, 0, 0, 1, 20, 16, None), arg, "16-byte aligned")
    assert lib.kt_kv8_read(good, 0, 100, 0, 16, 16, None) == _lib.KT_OK and lib.kt_kv8_read(good, 0, 0, 5, None, None, None) == _lib.KT_OK
    refused(lib.kt_kv8_copy(good, 101, good, 1, None), rng, "from a cache holding 101")
    refused(lib.kt_kv8_copy(good, 5, good, 6, None), rng, "Cannot copy 6")
    refused(lib.kt_kv8_copy(ctypes.byref(_cache(max_seq=200)), 150, good, 120, None), rng, "into a cache of 100")
    for change in ({"layers": 1}, {"kv_heads": 1}, {"head_dim": 32}, {"format": 1}, {"block_tokens": 32}):
        refused(lib.kt_kv8_copy(ctypes.byref(_cache(**change)), 5, good, 5, None), shape, "differ")
    assert lib.kt_kv8_copy(good, 5, good, 0, None) == _lib.KT_OK


def _controls(**change):
    from kotensor_amd import _lib
    c = _lib.LogitsControls()
    c.history, c.history_length, c.history_stride, c.history_capacity, c.repetition = 16, 16, 8, 8, 1.5
    for name, value in change.items():
        setattr(c, name, value)
    return ctypes.byref(c)


@pytest.mark.parametrize("change,want,message", [
    ({"repetition": 0.0}, -1, "repetition"), ({"repetition": -1.0}, -1, "repetition"), ({"repetition": float("nan")}, -1, "repetition"),
    ({"repetition": float("inf")}, -1, "repetition"), ({"frequency": float("nan")}, -1, "finite"), ({"presence": float("inf")}, -1, "finite"),
    ({"history": None}, -1, "history"), ({"history_length": None}, -1, "history"), ({"history_capacity": -1}, -2, "history"),
    ({"history_stride": 7}, -2, "history"), ({"bias_count": -1}, -2, "bias"), ({"bias_count": 2}, -1, "bias_tokens"),
    ({"bias_count": 2, "bias_tokens": 16, "bias_values": 16, "bias_stride": 1}, -2, "biases"), ({"allowed": 16, "allowed_stride": 3}, -2, "mask"),
])
def test_logits_refused(change, want, message):
    from kotensor_amd import _lib
    lib = _lib.lib()
    assert lib.kt_process_logits(16, 2, 100, 100, _controls(**change), 16, 100, None) == want and message in _lib.last_error()


def test_logits_shapes_refused():
    from kotensor_amd import _lib
    lib = _lib.lib()
    for args, want in (((None, 2, 100, 100, _controls(), 16, 100), -1), ((16, 2, 100, 100, _controls(), None, 100), -1), ((16, 2, 100, 100, None, 16, 100), -1),
                       ((16, -1, 100, 100, _controls(), 16, 100), -2), ((16, 2, 0, 100, _controls(), 16, 100), -2), ((16, 2, 100, 99, _controls(), 16, 100), -2),
                       ((16, 2, 100, 100, _controls(), 16, 99), -2), ((16, 65536, 100, 100, _controls(), 16, 100), -2)):
        assert lib.kt_process_logits(*args, None) == want, args
    assert lib.kt_process_logits(16, 0, 100, 100, _controls(), 16, 100, None) == _lib.KT_OK


def test_formats_restated():
    """Every code is its own nearest; ties go to even; the packed order is a permutation."""
    finite = kv8_ref.E4M3[np.isfinite(kv8_ref.E4M3)]
    assert np.array_equal(kv8_ref._nearest_e4m3(finite.astype(np.float32)), finite)
    assert list(kv8_ref._nearest_e4m3(np.array([1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 500.0], np.float32))) == [1.0, 1.25, 0.0, 2.0 ** -8, 448.0]
    codes, s = kv8_ref.hold_block(np.array([[127.0, 0.5, 1.5, -2.5]], np.float32), "int8")
    assert s == 1.0 and codes.tolist() == [[127.0, 0.0, 2.0, -2.0]]
    assert kv8_ref.hold_block(np.zeros((3, 4), np.float32), "e4m3")[1] == np.float32(2.0 ** -120)
    assert sorted(kv8_ref.VALUE_ORDER) == list(range(64))
    for fmt, step in (("int8", 0.5 / 127), ("e4m3", 2.0 ** -4)):
        x = np.random.default_rng(0).standard_normal((2, 70, 8)).astype(np.float32)
        held = kv8_ref.hold(x, fmt, 32)
        for g in range(2):
            for b in range(0, 70, 32):
                top = np.abs(x[g, b:b + 32]).max()
                off = np.abs(held[g, b:b + 32] - x[g, b:b + 32])
                # half a step, of the largest value (int8) or of each (e4m3, not below its least normal number)
                bound = step * top if fmt == "int8" else step * np.maximum(np.abs(x[g, b:b + 32]), top / 448 * 2.0 ** -6)
                assert np.all(off <= bound * (1 + 1e-5))


def test_controls_refused():
    import kotensor_amd as kt
    for args in ({"repetition_penalty": 0.0}, {"repetition_penalty": float("inf")}, {"frequency_penalty": float("nan")}, {"presence_penalty": float("inf")}):
        with pytest.raises(kt.IllegalArgumentException):
            kt.LogitsControls(**args)
    with pytest.raises(kt.IllegalArgumentException, match="cache format"):
        kt.QuantizedKVCache(1, 1, 8, 64, "int4")
    with pytest.raises(kt.IllegalArgumentException, match="head dimension 48"):
        kt.QuantizedKVCache(1, 1, 8, 48)
    with pytest.raises(kt.IllegalArgumentException, match="33 tokens to a block"):
        kt.QuantizedKVCache(1, 1, 8, 64, "int8", 33)
