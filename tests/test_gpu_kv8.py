"""The KV cache held in 8 bits (kt_kv8.hip) against its restatement: the append's bits, the
attention in 64 bits over what the cache holds, reads, copies, and their use together.

The append's arithmetic is the format's definition (fp32 quotients, products and roundings), so what
the cache holds of given rows is compared bit for bit; rotated keys come from cosines whose last
bit may be a library's, and are read back from the call's own open rows or compared within 2 ulp.

Attention: a rounding to fp32 is off by at most 2^-24, and by 0.41 of that rms over mantissas. A
score s passes about six of them (the query's parts, to 2^-22 of its row's largest element, are one; the
products' sums, two scales, the difference to the maximum), which moves its weight by sqrt(6) * 0.41 *
2^-24 |s| = 2^-24 |s| relative; the exponential and the weight's parts add 2^-23. A weighted sum of
values of random sign is as large as the sum of its terms' errors is small: their ratio is the terms'
own relative error. A chain of N fp32 additions and rescalings adds 0.41 * 2^-24 * sqrt(2 N): 16 * 2^-24 for
750 (a lane adds 32 keys at a time, then their sums). So 2^-24 (S + 24) normwise, S the case's largest score."""
import ctypes

import numpy as np
import pytest

from conftest import normwise_rel
from gpu_helpers import banner, same_bits
from oracle import kv8_ref

pytestmark = pytest.mark.gpu


def _tolerance(q, keys, heads):
    return 2.0 ** -24 * (kv8_ref.largest_score(q, keys, heads) + 24.0)


def _dev(kt, a):
    return kt.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


def _inv_freq(d, theta=10000.0):
    from kotensor_amd.transformer import rope_inv_freq
    return rope_inv_freq(d, theta)


def _append(kt, cache, layer, k, v, start, q=None, heads=None, stream=None, in_place=False):
    """kt_rope_kv8 of rows [tokens x kv * d] at `start`; returns the rotated q."""
    from kotensor_amd import _lib
    heads = heads or cache.num_heads
    dk, dv, dq = _dev(kt, k), _dev(kt, v), None if q is None else _dev(kt, q)
    out = dq if in_place else None if q is None else kt.DeviceBuffer(q.nbytes)
    freq, pos = _dev(kt, _inv_freq(cache.head_dim)), _dev(kt, np.array([start], np.int32))
    _lib.call("kt_rope_kv8", dq.ptr if dq else None, dk.ptr, dv.ptr, k.shape[0], heads, freq.ptr, pos.ptr, ctypes.byref(cache.cache), layer,
              out.ptr if out else None, stream)
    kt.synchronize()
    return None if out is None else out.download(np.float32).reshape(q.shape)


def _rows(rng, tokens, kv, d):
    x = rng.standard_normal((tokens, kv, d)) * np.exp(rng.standard_normal((1, kv, d))) * np.exp(0.5 * rng.standard_normal((tokens, kv, 1)))
    return x.reshape(tokens, kv * d).astype(np.float32)


def _heads_first(rows, kv):
    return rows.reshape(rows.shape[0], kv, -1).transpose(1, 0, 2)


def _rotated(oracle_lib, k, d, start):
    return oracle_lib.rope_rows(k, d, _inv_freq(d), start)


SHAPES = [("int8", 64, 64, 2), ("e4m3", 64, 64, 3), ("int8", 32, 128, 2), ("e4m3", 32, 32, 1), ("int8", 128, 32, 2), ("e4m3", 128, 256, 1), ("int8", 128, 256, 1)]


@pytest.mark.parametrize("fmt,block,d,kv", SHAPES)
@pytest.mark.parametrize("calls", [[1], [5], [200], [64, 64], [1, 1, 1, 1], [31, 2, 33, 1], [63, 130, 7, 1], [100, 1, 155, 3, 5]])
def test_append_holds_the_rows(kt, oracle_lib, fmt, block, d, kv, calls):
    """Whatever calls the rows come in, the cache holds their restatement, bit for bit: blocks that
    begin, end or stay open inside a call, the second layer, the memory around untouched."""
    banner("kv8-append", fmt, block, d, kv, calls)
    rng = np.random.default_rng(sum(calls) + d)
    n = sum(calls)
    k, v = _rows(rng, n, kv, d), _rows(rng, n, kv, d)
    cache = kt.QuantizedKVCache(2, kv, n + 3, d, fmt, block)
    cache.keys.upload(np.full(cache.keys.nbytes, 0x7F, np.uint8))  # (a NaN in e4m3)
    cache.values.upload(np.full(cache.values.nbytes, 0x7F, np.uint8))
    at = 0
    for c in calls:
        _append(kt, cache, 1, k[at:at + c], v[at:at + c], at)
        at += c
    got_k, got_v = cache.rows_numpy(1, 0, n)
    assert same_bits(got_v, kv8_ref.hold(_heads_first(v, kv), fmt, block))
    rotated = _heads_first(_rotated(oracle_lib, k, d, 0), kv)
    want = kv8_ref.hold(rotated, fmt, block)
    # a last bit of a cosine may move a rotated value by 2 ulp, and, rarely, a code by one step
    assert np.mean(got_k == want) > 0.999 and normwise_rel(got_k, want) < 2e-3
    # one call holds the same bits
    whole = kt.QuantizedKVCache(2, kv, n + 3, d, fmt, block)
    _append(kt, whole, 1, k, v, 0)
    assert all(same_bits(a, b) for a, b in zip(whole.rows_numpy(1, 0, n), (got_k, got_v)))
    # slots of tokens not held, and the other layer, as they were
    raw = cache.keys.download(np.uint8).reshape(2, kv, -1, d)
    assert np.all(raw[0] == 0x7F) and np.all(raw[1, :, n:] == 0x7F)
    raw = cache.values.download(np.uint8).reshape(2, kv, -1, d, 64)
    assert np.all(raw[0] == 0x7F)
    behind = np.concatenate([raw[1][..., kv8_ref.VALUE_ORDER].transpose(0, 1, 3, 2).reshape(kv, -1, d)[:, n:]])
    assert np.all(behind == 0x7F)
    # the open block's rows
    if n % block:
        rows = cache.value_rows.download(np.float32).reshape(2, kv, block, d)[1][:, :n % block]
        assert same_bits(rows, _heads_first(v, kv)[:, n // block * block:])


def test_rotated_queries(kt, oracle_lib):
    for d, heads, kv, tokens, start in [(64, 8, 2, 1, 0), (64, 14, 2, 70, 1000), (128, 4, 4, 9, 131000), (32, 6, 6, 33, 5), (256, 2, 1, 3, 77)]:
        banner("kv8-rope", d, heads, kv, tokens, start)
        rng = np.random.default_rng(d)
        cache = kt.QuantizedKVCache(1, kv, start + tokens, d)
        q, k = (rng.standard_normal((tokens, h * d)).astype(np.float32) for h in (heads, kv))
        got = _append(kt, cache, 0, k, k, start, q, heads)
        want = _rotated(oracle_lib, q, d, start)
        np.testing.assert_allclose(got, want, rtol=0, atol=2 * np.spacing(np.abs(want).max()))
        assert same_bits(_append(kt, cache, 0, k, k, start, q, heads, in_place=True), got)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_extreme_rows(kt, fmt):
    """Zeros, one loud value, values below the smallest scale, a block that is not finite."""
    banner("kv8-extreme", fmt)
    d, kv, block = 64, 1, 32
    v = np.zeros((160, d), np.float32)
    v[32:64] = 1e-3
    v[40, 7] = 3e38
    v[64:96] = 1e-42
    v[100, 3] = np.inf
    v[130, 5] = np.nan
    cache = kt.QuantizedKVCache(1, kv, 160, d, fmt, block)
    for at in (0, 50, 51, 120):
        end = {0: 50, 50: 51, 51: 120, 120: 160}[at]
        _append(kt, cache, 0, v[at:end], v[at:end], at)
    got = cache.rows_numpy(0, 0, 160)[1][0]
    assert np.all(got[:32] == 0) and np.all(got[64:96] == 0)
    assert same_bits(got[32:64], kv8_ref.hold(v[None, 32:64], fmt, block)[0])
    assert np.all(np.isnan(got[96:160]))


def test_reads(kt):
    rng = np.random.default_rng(5)
    for fmt, d, block in (("int8", 64, 64), ("e4m3", 256, 32), ("int8", 32, 128)):
        cache = kt.QuantizedKVCache(1, 2, 300, d, fmt, block)
        k, v = _rows(rng, 290, 2, d), _rows(rng, 290, 2, d)
        _append(kt, cache, 0, k, v, 0)
        whole = cache.rows_numpy(0, 0, 290)
        for first, count in ((0, 1), (63, 2), (64, 64), (5, 280), (289, 1), (128, 0)):
            banner("kv8-read", fmt, d, first, count)
            for a, b in zip(cache.rows_numpy(0, first, count), whole):
                assert same_bits(a, b[:, first:first + count])


@pytest.mark.parametrize("fmt,block,d", [("int8", 64, 64), ("e4m3", 32, 128), ("int8", 128, 32)])
def test_copies_and_what_follows(kt, fmt, block, d):
    """A prefix copied, in the source's open block, at a block's end, inside an earlier block, and
    a cache shortened; then both go on."""
    rng = np.random.default_rng(6)
    kv, n = 2, 201
    source = kt.QuantizedKVCache(2, kv, 400, d, fmt, block)
    k, v = _rows(rng, n + 40, kv, d), _rows(rng, n + 40, kv, d)
    for layer in range(2):
        _append(kt, source, layer, k[:n], v[:n], 0)
    source.advance(n)
    before = [source.rows_numpy(layer) for layer in range(2)]
    for length in (0, 1, n, n - 1, block, 100, 128):
        banner("kv8-copy", fmt, block, length)
        copy = kt.QuantizedKVCache(2, kv, 300, d, fmt, block)
        copy.copy_from(source, length)
        assert copy.length == length and copy.position.download(np.int32)[0] == length
        for layer in range(2):
            for a, b in zip(copy.rows_numpy(layer), before[layer]):
                assert same_bits(a, b[:, :length])
            _append(kt, copy, layer, k[length:length + 40], v[length:length + 40], length)
        copy.advance(40)
        rows = copy.rows_numpy(1)[1]
        whole = kv8_ref.hold(_heads_first(v[:length + 40], kv), fmt, block)
        if length // block == n // block or length % block == 0:  # the source's own rows: as if appended
            assert same_bits(rows[:, length // block * block:], whole[:, length // block * block:])
        else:  # a code's rounding once more
            assert normwise_rel(rows, whole) < 0.1
    source.copy_from(source, 70)  # shortened in place
    assert source.length == 70
    for a, b in zip(source.rows_numpy(0), before[0]):
        assert same_bits(a, b[:, :70])
    _append(kt, source, 0, k[70:75], v[70:75], 70)
    assert normwise_rel(source.rows_numpy(0, 0, 75)[1], kv8_ref.hold(_heads_first(v[:75], kv), fmt, block)) < 0.1


# ---- attention ---------------------------------------------------------------------------------

def _filled(kt, rng, fmt, block, d, kv, n, max_seq, layers=1, layer=0, loud=None):
    """A cache holding n tokens, written as bytes; (cache, keys, values it holds as fp64)."""
    cache = kt.QuantizedKVCache(layers, kv, max_seq, d, fmt, block)
    slots = cache.keys.nbytes // (layers * kv * d)
    held = []
    for name, scales in (("keys", "key_scales"), ("values", "value_scales")):
        if fmt == "int8":
            stored = rng.integers(1, 256, (kv, slots, d)).astype(np.uint8)
        else:
            stored = rng.integers(0, 0x7F, (kv, slots, d)).astype(np.uint8) | (rng.integers(0, 2, (kv, slots, d)) * 0x80).astype(np.uint8)
        stored[:, n:] = 0x7F  # not held: a NaN in e4m3
        top = 127.0 if fmt == "int8" else 448.0
        s = ((0.3 + rng.random((kv, slots // block))) / top * (3.0 if fmt == "int8" else 9.0)).astype(np.float32)
        if loud is not None and name == "values":
            s *= np.exp2(rng.integers(-loud, loud, s.shape)).astype(np.float32)
        s[:, (n + block - 1) // block:] = np.nan
        x = kv8_ref.code_values(stored, fmt) * np.repeat(s, block, 1)[..., None].astype(np.float64)
        held.append(x[:, :n])
        raw = np.full((layers, kv, slots * d), 0x7F, np.uint8)
        raw[layer] = (kv8_ref.pack_values(stored) if name == "values" else stored).reshape(kv, -1)
        getattr(cache, name).upload(raw)
        scale = np.full((layers, kv, slots // block), np.nan, np.float32)
        scale[layer] = s
        getattr(cache, scales).upload(scale)
    return cache, held[0], held[1]


def _attend(kt, cache, layer, q, start, heads, bound=None, stream=None):
    from kotensor_amd import _lib
    dq, pos, out = _dev(kt, q), _dev(kt, np.array([start], np.int32)), _dev(kt, np.full(q.shape, 7.0, np.float32))
    kt.synchronize()
    _lib.call("kt_attention_kv8", dq.ptr, q.shape[0], pos.ptr, bound or start + q.shape[0], ctypes.byref(cache.cache), layer, heads, out.ptr, stream)
    _lib.call("kt_stream_sync", stream)
    return out.download(np.float32).reshape(q.shape)


ATTENTION = [
    # one token: first, block and chunk ends, many splits; group sizes 1 to 16 and more
    (1, 0, 4, 4, 64), (1, 31, 8, 1, 64), (1, 32, 14, 2, 64), (1, 63, 32, 8, 64), (1, 64, 16, 1, 64), (1, 200, 6, 6, 32), (1, 511, 32, 8, 128), (1, 1000, 8, 2, 256),
    (1, 5000, 32, 8, 64), (1, 9000, 14, 2, 64), (1, 4097, 20, 1, 64), (1, 3000, 64, 2, 64), (1, 20000, 5, 5, 128),
    # drafted tokens
    (2, 0, 4, 4, 64), (7, 4000, 32, 8, 64), (15, 62, 14, 2, 64), (5, 700, 8, 1, 128), (9, 1500, 8, 2, 256), (3, 2500, 3, 3, 32), (15, 3000, 16, 1, 64),
    # prompts
    (16, 0, 4, 4, 64), (17, 47, 14, 2, 64), (64, 0, 32, 8, 64), (65, 63, 8, 1, 64), (100, 1500, 4, 1, 64), (300, 1, 8, 8, 64), (33, 95, 16, 2, 128), (130, 200, 7, 1, 128),
    (40, 3, 3, 1, 64), (191, 0, 6, 6, 32), (70, 1000, 8, 2, 256), (257, 64, 5, 5, 128), (150, 0, 20, 1, 64), (513, 0, 2, 1, 64), (48, 0, 1, 1, 256), (31, 129, 40, 2, 64),
]


@pytest.mark.parametrize("fmt,block", [("int8", 64), ("e4m3", 32), ("int8", 128), ("e4m3", 128), ("int8", 32)])
@pytest.mark.parametrize("tokens,start,heads,kv,d", ATTENTION)
def test_attention_against_64_bits(kt, fmt, block, tokens, start, heads, kv, d):
    banner("kv8-attention", fmt, block, tokens, start, heads, kv, d)
    rng = np.random.default_rng(tokens + start + d)
    n = start + tokens
    cache, keys, values = _filled(kt, rng, fmt, block, d, kv, n, n + 70, layers=2, layer=1)
    q = (1.5 * rng.standard_normal((tokens, heads * d))).astype(np.float32)
    want = kv8_ref.attend(q, keys, values, start, heads)
    got = _attend(kt, cache, 1, q, start, heads)
    err = normwise_rel(got, want)
    print(f"  error {err:.2e} of {_tolerance(q, keys, heads):.2e}", flush=True)
    assert err <= _tolerance(q, keys, heads)
    # the bits do not depend on the bound that sizes the launch
    assert same_bits(_attend(kt, cache, 1, q, start, heads, n + 70), got)


@pytest.mark.parametrize("tokens,start,heads,kv,d", [(1, 700, 8, 2, 64), (6, 3000, 8, 2, 64), (200, 300, 8, 2, 64), (100, 0, 4, 1, 128)])
def test_blocks_of_very_different_loudness(kt, tokens, start, heads, kv, d):
    """Value scales from 2^-20 to 2^20: each row to its own values' size."""
    banner("kv8-loud", tokens, start)
    rng = np.random.default_rng(9)
    n = start + tokens
    cache, keys, values = _filled(kt, rng, "int8", 32, d, kv, n, n, loud=20)
    q = rng.standard_normal((tokens, heads * d)).astype(np.float32)
    want = kv8_ref.attend(q, keys, values, start, heads).reshape(tokens * heads, d)
    got = _attend(kt, cache, 0, q, start, heads).reshape(tokens * heads, d).astype(np.float64)
    assert np.max(np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)) <= 4e-6


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 30.0, 1e4, 1e30])
@pytest.mark.parametrize("tokens,start", [(1, 900), (4, 900), (40, 100)])
def test_queries_of_any_size(kt, tokens, start, scale):
    """Flat and one-hot softmaxes. A score of magnitude s is off by at most 2^-21 s (q's parts, fp32
    sums), which is the relative error of its weight; rows whose largest scores are
    nearer than that to each other are left out."""
    banner("kv8-scale", tokens, scale)
    rng = np.random.default_rng(10)
    heads, kv, d, n = 4, 2, 64, start + tokens
    cache, keys, values = _filled(kt, rng, "int8", 64, d, kv, n, n)
    q = (scale * rng.standard_normal((tokens, heads * d))).astype(np.float32)
    want = kv8_ref.attend(q, keys, values, start, heads).reshape(tokens * heads, d)
    got = _attend(kt, cache, 0, q, start, heads).reshape(tokens * heads, d)
    assert np.all(np.isfinite(got))
    for r in range(tokens * heads):
        t, h = divmod(r, heads)
        s = keys[h // 2, :start + t + 1] @ q[t, h * d:(h + 1) * d].astype(np.float64) / 8.0
        top = np.sort(s)[-2:]
        off = 2.0 ** -21 * np.abs(s).max()
        if off > 1e-3 and top[1] - top[0] < 40 + 2 * off:
            continue
        assert normwise_rel(got[r], want[r]) <= 24 * 2.0 ** -24 + (2 * off if off <= 1e-3 else 0.0)


@pytest.mark.parametrize("tokens,start", [(1, 300), (5, 300), (80, 260)])
def test_not_finite(kt, tokens, start):
    """A block whose scale is NaN makes NaNs of the rows that see one of its tokens, and of no
    other; a query that is not finite, of its own row. (The other rows' bits may differ: a scale's exponent
    enters the exponentials' argument, whose rounding is one of those that _tolerance counts.)"""
    banner("kv8-nan", tokens)
    rng = np.random.default_rng(11)
    heads, kv, d, n, block = 4, 2, 64, start + tokens, 32
    cache, keys, values = _filled(kt, rng, "int8", block, d, kv, n, n)
    q = rng.standard_normal((tokens, heads * d)).astype(np.float32)
    tol = _tolerance(q, keys, heads)
    q[0, 3] = np.inf
    q[tokens - 1, 3 * d] = np.nan
    clean = _attend(kt, cache, 0, q, start, heads)
    bad = (start + tokens // 2) // block  # the block of a token in the middle of the call
    for name in ("key_scales", "value_scales"):
        buffer = getattr(cache, name)
        held = buffer.download(np.float32)
        changed = held.reshape(kv, -1).copy()
        changed[1, bad] = np.nan
        buffer.upload(changed)
        got = _attend(kt, cache, 0, q, start, heads)
        buffer.upload(held)
        for t in range(tokens):
            for h in range(heads):
                row, was = got[t, h * d:(h + 1) * d], clean[t, h * d:(h + 1) * d]
                if (t == 0 and h == 0) or (t == tokens - 1 and h == 3) or (h >= 2 and start + t >= bad * block):
                    assert np.all(np.isnan(row)), (name, t, h)
                else:
                    assert np.all(np.isfinite(row)) and normwise_rel(row, was) <= tol, (name, t, h)


@pytest.mark.parametrize("tokens", [1, 6, 20])
def test_positions_outside(kt, tokens):
    """Tokens that see no key get zeros; nothing past the cache is read."""
    banner("kv8-outside", tokens)
    rng = np.random.default_rng(12)
    cache, keys, values = _filled(kt, rng, "int8", 64, 64, 2, 100, 100)
    q = rng.standard_normal((tokens, 4 * 64)).astype(np.float32)
    assert np.all(_attend(kt, cache, 0, q, -tokens, 4, tokens) == 0.0)
    got = _attend(kt, cache, 0, q, -2, 4, tokens)
    assert np.all(got[:2] == 0.0)
    if tokens > 2:
        assert normwise_rel(got[2:], kv8_ref.attend(q[2:], keys, values, 0, 4)) <= _tolerance(q, keys, 4)
    assert normwise_rel(_attend(kt, cache, 0, q, 5000, 4, 100), kv8_ref.attend(q, keys, values, 5000, 4)) <= _tolerance(q, keys, 4)


def test_a_long_cache_passes_32_bits(kt):
    """The last layer of a cache of more than 4 GiB a side: offsets of codes past 32 bits."""
    banner("kv8-long")
    kv, d, layers, max_seq, start = 8, 128, 36, 131072, 4000
    rng = np.random.default_rng(13)
    cache = kt.QuantizedKVCache(layers, kv, max_seq, d, "int8", 64)
    assert cache.keys.nbytes > 2 ** 32
    k, v = _rows(rng, start, kv, d), _rows(rng, start, kv, d)
    _append(kt, cache, layers - 1, k, v, 0)
    rows = cache.rows_numpy(layers - 1, 0, start)
    assert same_bits(rows[1], kv8_ref.hold(_heads_first(v, kv), "int8", 64))
    q = rng.standard_normal((2, kv * d)).astype(np.float32)
    assert normwise_rel(_attend(kt, cache, layers - 1, q, start - 2, kv, max_seq), kv8_ref.attend(q, *rows, start - 2, kv)) <= _tolerance(q, rows[0], kv)
    assert not np.any(cache.keys.download(np.uint8, count=1 << 20))  # the first layer is untouched


# ---- a decode step in one call -------------------------------------------------------------------

@pytest.mark.parametrize("fmt,block", [("int8", 64), ("e4m3", 32), ("int8", 128)])
@pytest.mark.parametrize("start,heads,kv,d", [(0, 32, 8, 64), (1, 14, 2, 64), (63, 8, 1, 64), (64, 6, 6, 32), (500, 32, 8, 128), (1055, 8, 2, 256), (3000, 14, 2, 64), (127, 20, 1, 64)])
def test_step_equals_its_parts(kt, oracle_lib, fmt, block, start, heads, kv, d):
    """kt_rope_attention_kv8 of one token: the cache has the append's bits, q stays, the context is
    the attention's of the rotated q."""
    from kotensor_amd import _lib
    banner("kv8-step", fmt, block, start, heads, kv, d)
    rng = np.random.default_rng(start + d)
    k, v = _rows(rng, start + 2, kv, d), _rows(rng, start + 2, kv, d)
    k[start] *= 3.0  # raises the open block's scale
    k[start + 1] *= 0.1  # does not
    q = rng.standard_normal((2, heads * d)).astype(np.float32)
    one, two = (kt.QuantizedKVCache(2, kv, start + 2, d, fmt, block) for _ in range(2))
    if start:
        for c in (one, two):
            _append(kt, c, 1, k[:start], v[:start], 0)
    freq = _dev(kt, _inv_freq(d))
    for t in range(2):
        rotated = _append(kt, one, 1, k[start + t:start + t + 1], v[start + t:start + t + 1], start + t, q[t:t + 1], heads)
        want = _attend(kt, one, 1, rotated, start + t, heads)
        dq, dk, dv = _dev(kt, q[t]), _dev(kt, k[start + t]), _dev(kt, v[start + t])
        pos, out = _dev(kt, np.array([start + t], np.int32)), kt.DeviceBuffer(4 * heads * d)
        _lib.call("kt_rope_attention_kv8", dq.ptr, dk.ptr, dv.ptr, freq.ptr, 1, pos.ptr, start + 2, ctypes.byref(two.cache), 1, heads, out.ptr, None)
        kt.synchronize()
        assert same_bits(dq.download(np.float32), q[t]) and same_bits(dk.download(np.float32), k[start + t])
        for a, b in zip(one.rows_numpy(1, 0, start + t + 1), two.rows_numpy(1, 0, start + t + 1)):
            assert same_bits(a, b)
        for name in ("keys", "values", "key_scales", "value_scales", "key_rows", "value_rows"):
            assert same_bits(getattr(one, name).download(np.uint8), getattr(two, name).download(np.uint8)), name
        turned, held = _rotated(oracle_lib, q[t:t + 1], d, start + t), one.rows_numpy(1, 0, start + t + 1)
        tol = _tolerance(turned, held[0], heads)
        assert normwise_rel(out.download(np.float32), want.reshape(-1)) <= tol
        assert normwise_rel(want, kv8_ref.attend(turned, *held, start + t, heads)) <= tol


def test_after_a_call_that_leaves_the_workspace_at_an_odd_place(kt):
    """The fp32 cache's attention of an odd number of heads and splits sizes the stream's zeroed words, behind which
    the general area begins at any dword: the splits' pairs of words are placed at their own alignment."""
    from kotensor_amd import _lib
    banner("kv8-workspace")
    rng = np.random.default_rng(17)
    stream = kt.Stream.create()
    q, k = rng.standard_normal((1, 3 * 64)).astype(np.float32), rng.standard_normal((1, 700, 64)).astype(np.float32)
    dq, dk, pos, out = _dev(kt, q), _dev(kt, k), _dev(kt, np.array([699], np.int32)), kt.DeviceBuffer(q.nbytes)
    _lib.call("kt_attention", dq.ptr, 1, pos.ptr, 700, dk.ptr, dk.ptr, 0, 700, 3, 1, 64, out.ptr, stream.handle)
    stream.synchronize()
    cache, keys, values = _filled(kt, rng, "int8", 64, 64, 1, 3000, 3000)
    got = _attend(kt, cache, 0, q, 2999, 3, stream=stream.handle)
    assert normwise_rel(got, kv8_ref.attend(q, keys, values, 2999, 3)) <= _tolerance(q, keys, 3)
    stream.destroy()


def test_steps_of_two_streams_and_threads(kt):
    """Steps of two sequences enqueued on two streams by two threads at once: each its own result."""
    import threading

    from kotensor_amd import _lib
    banner("kv8-streams")
    rng = np.random.default_rng(14)
    heads, kv, d, start = 8, 2, 64, 2500
    runs = []
    for _ in range(2):
        cache, keys, values = _filled(kt, rng, "int8", 64, d, kv, start + 1, start + 1)
        q = rng.standard_normal((1, heads * d)).astype(np.float32)
        runs.append((cache, _dev(kt, q), _dev(kt, np.array([start], np.int32)), [kt.DeviceBuffer(q.nbytes) for _ in range(50)],
                     kt.Stream.create(), _attend(kt, cache, 0, q, start, heads)))

    def go(run):
        cache, q, pos, outs, stream, _ = run
        for out in outs:
            _lib.call("kt_attention_kv8", q.ptr, 1, pos.ptr, start + 1, ctypes.byref(cache.cache), 0, heads, out.ptr, stream.handle)
    threads = [threading.Thread(target=go, args=(r,)) for r in runs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for cache, _, _, outs, stream, want in runs:
        stream.synchronize()
        for out in outs:
            assert same_bits(out.download(np.float32), want.reshape(-1))
        stream.destroy()


@pytest.mark.parametrize("tokens", [1, 5, 40])
def test_recorded_calls(kt, tokens):
    """A recorded step follows the device position from replay to replay, with eager calls of
    other sizes on other streams in between; every replay equals the eager call."""
    from kotensor_amd import _lib
    banner("kv8-record", tokens)
    rng = np.random.default_rng(15)
    heads, kv, d, start, steps = 8, 2, 64, 700, 4
    n = start + tokens * steps
    k, v = _rows(rng, n, kv, d), _rows(rng, n, kv, d)
    caches = [kt.QuantizedKVCache(1, kv, n, d) for _ in range(2)]
    for c in caches:
        _append(kt, c, 0, k[:start], v[:start], 0)
        c.advance(start)
    q0 = rng.standard_normal((tokens, heads * d)).astype(np.float32)
    dq, dk, dv, out = _dev(kt, q0), kt.DeviceBuffer(4 * tokens * kv * d), kt.DeviceBuffer(4 * tokens * kv * d), kt.DeviceBuffer(q0.nbytes)
    freq, stream, graph = _dev(kt, _inv_freq(d)), kt.Stream.create(), ctypes.c_void_p()

    def step(cache, st):
        _lib.call("kt_rope_attention_kv8", dq.ptr, dk.ptr, dv.ptr, freq.ptr, tokens, cache.position.ptr, n, ctypes.byref(cache.cache), 0, heads, out.ptr, st)
        _lib.call("kt_position_add", cache.position.ptr, tokens, st)

    def load(i):
        dq.upload(q0)
        dk.upload(k[start + i * tokens:start + (i + 1) * tokens])
        dv.upload(v[start + i * tokens:start + (i + 1) * tokens])
        kt.synchronize()
    want = []
    for i in range(steps):  # eager, on the stream that records afterwards
        load(i)
        step(caches[0], stream.handle)
        stream.synchronize()
        want.append(out.download(np.float32))
    _lib.call("kt_graph_begin", stream.handle)
    try:
        step(caches[1], stream.handle)
    finally:
        _lib.call("kt_graph_end", stream.handle, ctypes.byref(graph))
    other, keys, values = _filled(kt, rng, "e4m3", 32, d, kv, 6000, 6000)
    try:
        for i in range(steps):
            load(i)
            out.fill_zero()
            kt.synchronize()
            _lib.call("kt_graph_launch", graph, stream.handle)
            stream.synchronize()
            assert same_bits(out.download(np.float32), want[i]), i
            for t in (1, 3, 30):
                q = rng.standard_normal((t, heads * d)).astype(np.float32)
                assert normwise_rel(_attend(kt, other, 0, q, 6000 - t, heads), kv8_ref.attend(q, keys, values, 6000 - t, heads)) <= _tolerance(q, keys, heads)
        for a, b in zip(caches[0].rows_numpy(0, 0, n), caches[1].rows_numpy(0, 0, n)):
            assert same_bits(a, b)
    finally:
        stream.synchronize()
        _lib.call("kt_graph_destroy", graph)
        stream.destroy()


# ---- a model on it ---------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt,block,dim,heads,kvh", [("int8", 64, 256, 4, 2), ("e4m3", 32, 256, 4, 1), ("int8", 32, 128, 4, 4)])
def test_a_model_decodes_on_it(kt, oracle_lib, fmt, block, dim, heads, kvh):
    """Prompts and decode steps on an 8-bit cache against the oracle's decoder with the same cache; and,
    bit for bit: graph replays and eager steps, copies that go on, a cache used again.

    The projections of one and two rows agree with the oracle's to fp32 roundings (logits to 1e-4), so a
    row's elements to some 1e-5 of its size: an int8 code (steps of 1/127 of the largest) is then another one
    in about 1e-3 of the elements, an e4m3 code (2^-4 of each) in 2e-4, which moves a row of 64 by about 1e-3
    of its size; the layers of the small model may make ten times that of it: 1e-2. Prompts through the
    prefill GEMM (2^-12 of a product) change one code in 50, 5e-3 of a row: 5e-2."""
    from oracle import decoder_ref
    from test_gpu_decoder import to_oracle
    banner("kv8-model", fmt, block)
    rng = np.random.default_rng(16)
    model = kt.Transformer(500, dim, 3, heads, 2 * dim, kvh, quantization=kt.Quantization(8, 32), seed=3, init_std=0.08)
    plain = to_oracle(kt, model)
    ref = kv8_ref.HeldTransformer(plain.config, plain.quantized, plain.norms)
    ref.fmt, ref.block = fmt, block
    prompt = rng.integers(0, 500, 75).tolist()
    full, held = model.new_cache(200), model.new_cache(200, cache_format=fmt, block_tokens=block)
    assert held.size_in_bytes < full.size_in_bytes * (0.4 + block / 200)
    buffers, cache = model.new_inference_buffers(200), ref.new_cache(200)
    got, want = model.prefill(prompt, held, buffers, chunk_rows=2).logits_numpy(), ref.prefill_chunks(prompt, cache, 2)
    print(f"  two rows at a time {normwise_rel(got, want):.2e}", flush=True)
    assert normwise_rel(got, want) < 1e-2
    for token in (3, 99, 7):
        got, want = model.decode(token, held, buffers).logits_numpy(), ref.decode(token, cache)
        print(f"  decode {normwise_rel(got, want):.2e}", flush=True)
        assert normwise_rel(got, want) < 1e-2
    one, cache = model.new_cache(200, cache_format=fmt, block_tokens=block), ref.new_cache(200)
    first = model.prefill(prompt, one, buffers).logits_numpy()
    want = ref.prefill_chunks(prompt, cache, 75)
    print(f"  whole prompt {normwise_rel(first, want):.2e}", flush=True)
    assert normwise_rel(first, want) < 5e-2
    copy = model.new_cache(150, cache_format=fmt, block_tokens=block)
    copy.copy_from(one, 75)
    assert same_bits(model.decode(5, one, buffers).logits_numpy(), model.decode(5, copy, buffers).logits_numpy())
    one.reset()
    assert same_bits(model.prefill(prompt, one, buffers).logits_numpy(), first)
    eager = model.generate(prompt, 70, use_graph=False, cache_format=fmt, block_tokens=block)
    assert model.generate(prompt, 70, cache_format=fmt, block_tokens=block) == eager
    assert model.generate(prompt, 70, cache_format=fmt, block_tokens=block) == eager


def test_cache_refusals(kt):
    model = kt.Transformer(100, 128, 2, 2, 128, 2, quantization=kt.Quantization(8, 32))
    cache, buffers = model.new_cache(20, cache_format="int8"), model.new_inference_buffers(20)
    with pytest.raises(kt.IllegalArgumentException, match="KV cache full"):
        model.prefill(list(range(21)), cache, buffers)
    with pytest.raises(kt.IllegalArgumentException, match="KV cache full"):
        cache.advance(21)
    with pytest.raises(kt.IllegalArgumentException, match="Cannot copy"):
        cache.copy_from(cache, 1)
    with pytest.raises(kt.IllegalArgumentException, match="Cannot copy a cache"):
        cache.copy_from(model.new_cache(20, cache_format="e4m3"), 0)
    small = kt.Transformer(100, 32, 1, 2, 64, 2, quantization=kt.Quantization(8, 32))
    with pytest.raises(kt.IllegalArgumentException, match="head dimension 16"):
        small.new_cache(20, cache_format="int8")
