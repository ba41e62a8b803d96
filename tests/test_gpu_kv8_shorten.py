"""Dropped tokens leave nothing behind: a copy that ends in the source's open block goes on, from its first
append on, as a cache that never held them."""
import ctypes

import numpy as np
import pytest

from conftest import normwise_rel
from gpu_helpers import banner, same_bits
from oracle import kv8_ref
from test_gpu_kv8 import _append, _attend, _dev, _inv_freq, _rows, _tolerance

pytestmark = pytest.mark.gpu

FORMS = [("int8", 64, 64, 2), ("e4m3", 32, 128, 2), ("int8", 128, 32, 1), ("e4m3", 128, 64, 3), ("int8", 32, 256, 1)]


def _state(cache, kv, n):
    """Everything a cache holds of n tokens, as bytes: codes, scales, the open block's rows."""
    block, d = cache.block_tokens, cache.head_dim
    slots = cache.keys.nbytes // (cache.num_layers * kv * d)
    keys = cache.keys.download(np.uint8).reshape(-1, kv, slots, d)[:, :, :n]
    values = cache.values.download(np.uint8).reshape(-1, kv, slots // 64, d, 64)[..., kv8_ref.VALUE_ORDER].transpose(0, 1, 2, 4, 3).reshape(-1, kv, slots, d)[:, :, :n]
    blocks = (n + block - 1) // block
    scales = [b.download(np.float32).reshape(-1, kv, slots // block)[:, :, :blocks] for b in (cache.key_scales, cache.value_scales)]
    rows = [b.download(np.float32).reshape(-1, kv, block, d)[:, :, :n % block] for b in (cache.key_rows, cache.value_rows)]
    return [keys, values, *scales, *rows]


def _assert_same(one, two, kv, n):
    for a, b in zip(_state(one, kv, n), _state(two, kv, n)):
        assert same_bits(a, b)


def _step(kt, cache, layer, q, k, v, at, heads):
    """kt_rope_attention_kv8 of the rows; its context."""
    from kotensor_amd import _lib
    dq, dk, dv, freq = (_dev(kt, a) for a in (q, k, v, _inv_freq(cache.head_dim)))
    pos, out = _dev(kt, np.array([at], np.int32)), kt.DeviceBuffer(q.nbytes)
    _lib.call("kt_rope_attention_kv8", dq.ptr, dk.ptr, dv.ptr, freq.ptr, q.shape[0], pos.ptr, cache.max_sequence_length, ctypes.byref(cache.cache), layer, heads,
              out.ptr, None)
    kt.synchronize()
    return out.download(np.float32).reshape(q.shape)


def _drafted(rng, fmt, kind, kv, d, length, dropped, more):
    """Rows of `length` tokens that stay, `dropped` that set the open block's scale, `more` that follow."""
    parts = [[_rows(rng, n, kv, d) for n in (length, dropped, more)] for _ in range(2)]
    for p in parts:
        p[1] *= {"loud": 500.0, "infinite": 500.0, "nan": 500.0, "quiet": 1e-3}[kind]
        if kind == "nan":
            p[1][:, ::7] = np.nan
        if kind == "infinite":
            p[1][0, ::d] = -np.inf
    return parts


@pytest.mark.parametrize("fmt,block,d,kv", FORMS)
@pytest.mark.parametrize("kind", ["loud", "infinite", "nan", "quiet"])
@pytest.mark.parametrize("how", ["copy", "in place", "copy of a copy"])
def test_what_follows_a_drop(kt, fmt, block, d, kv, kind, how):
    rng = np.random.default_rng(d + block)
    for length, dropped, calls in ((2 * block + 5, 3, [1, 1]), (2 * block + 1, block - 2, [4]), (block + block - 3, 2, [7, 1, block]), (1, 6, [2]), (5, 1, [block - 5, 3])):
        banner("kv8-drop", fmt, block, d, kind, how, length, dropped, calls)
        (k0, k1, k2), (v0, v1, v2) = _drafted(rng, fmt, kind, kv, d, length, dropped, sum(calls))
        size = length + max(dropped, sum(calls)) + 3
        source, fresh = (kt.QuantizedKVCache(2, kv, size, d, fmt, block) for _ in range(2))
        for layer in range(2):
            _append(kt, source, layer, np.concatenate([k0, k1]), np.concatenate([v0, v1]), 0)
            _append(kt, fresh, layer, k0, v0, 0)
        source.advance(length + dropped)
        cache = source
        if how == "copy of a copy":
            between = kt.QuantizedKVCache(2, kv, size, d, fmt, block)
            between.copy_from(source, length)
            source = between
        if how != "in place":
            cache = kt.QuantizedKVCache(2, kv, size + 100, d, fmt, block)
        cache.copy_from(source, length)
        at = length
        for count in calls:
            for layer in range(2):
                for c in (cache, fresh):
                    _append(kt, c, layer, k2[at - length:at - length + count], v2[at - length:at - length + count], at)
            at += count
            _assert_same(cache, fresh, kv, at)


@pytest.mark.parametrize("fmt,block,d,kv,heads", [("int8", 64, 64, 2, 8), ("e4m3", 32, 128, 2, 4), ("int8", 128, 32, 3, 3), ("e4m3", 128, 64, 1, 20), ("int8", 64, 256, 1, 2)])
@pytest.mark.parametrize("kind", ["loud", "nan"])
@pytest.mark.parametrize("length", [9, 197, 2900])
def test_a_step_after_a_drop(kt, oracle_lib, fmt, block, d, kv, heads, kind, length):
    """The append inside a step's attention launch, and one of several tokens with its attention."""
    rng = np.random.default_rng(length + d)
    (k0, k1, k2), (v0, v1, v2) = _drafted(rng, fmt, kind, kv, d, length, 3, 8)
    q = rng.standard_normal((8, heads * d)).astype(np.float32)
    source, cache, fresh = (kt.QuantizedKVCache(1, kv, length + 20, d, fmt, block) for _ in range(3))
    _append(kt, source, 0, np.concatenate([k0, k1]), np.concatenate([v0, v1]), 0)
    _append(kt, fresh, 0, k0, v0, 0)
    source.advance(length + 3)
    cache.copy_from(source, length)
    at = 0
    for count in (1, 1, 5, 1):
        banner("kv8-drop-step", fmt, block, d, heads, kind, length, at, count)
        rows = slice(at, at + count)
        got, want = (_step(kt, c, 0, q[rows], k2[rows], v2[rows], length + at, heads) for c in (cache, fresh))
        at += count
        _assert_same(cache, fresh, kv, length + at)
        assert same_bits(got, want)
        held = cache.rows_numpy(0, 0, length + at)
        turned = oracle_lib.rope_rows(q[rows], d, _inv_freq(d), length + at - count)
        assert normwise_rel(got, kv8_ref.attend(turned, *held, length + at - count, heads)) <= _tolerance(turned, held[0], heads)


@pytest.mark.parametrize("fmt,block,d,kv", FORMS)
def test_a_copy_before_its_first_append(kt, fmt, block, d, kv):
    """Until then it holds what the source holds of its tokens; a copy of the whole is the source, in every bit."""
    banner("kv8-drop-read", fmt, block, d)
    rng = np.random.default_rng(3 * d)
    length = block + 7
    (k0, k1, _), (v0, v1, _) = _drafted(rng, fmt, "loud", kv, d, length, 3, 1)
    source, part, again, whole = (kt.QuantizedKVCache(1, kv, 3 * block, d, fmt, block) for _ in range(4))
    _append(kt, source, 0, np.concatenate([k0, k1]), np.concatenate([v0, v1]), 0)
    source.advance(length + 3)
    part.copy_from(source, length)
    again.copy_from(part, length)
    whole.copy_from(source, length + 3)
    _assert_same(whole, source, kv, length + 3)
    held = [r[:, :length] for r in source.rows_numpy(0)]
    q = rng.standard_normal((3, 2 * kv * d)).astype(np.float32)
    want = kv8_ref.attend(q, *held, length - 3, 2 * kv)
    for cache in (part, again):
        for a, b in zip(cache.rows_numpy(0), held):
            assert same_bits(a, b)
        assert normwise_rel(_attend(kt, cache, 0, q, length - 3, 2 * kv), want) <= _tolerance(q, held[0], 2 * kv)
    # a block that the source has gone past: its rows are gone, the codes stay with their scale
    early = kt.QuantizedKVCache(1, kv, 3 * block, d, fmt, block)
    early.copy_from(source, block - 2)
    for a, b in zip(early.rows_numpy(0), held):
        assert same_bits(a, b[:, :block - 2])
