"""How calls on an 8-bit cache are launched: captures that the library did not begin, and bounds on both sides of the
length at which the form of the attention changes; and where reads may go."""
import ctypes

import numpy as np
import pytest

from conftest import normwise_rel
from gpu_helpers import banner, same_bits
from oracle import kv8_ref
from test_gpu_kv8 import _append, _attend, _dev, _filled, _inv_freq, _rows, _tolerance
from test_gpu_recorded_scratch import _hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,d", [(2, 1, 256), (8, 4, 256), (20, 1, 64), (34, 2, 128)])
@pytest.mark.parametrize("start,bound", [(10, 64), (700, 4000)])
def test_a_callers_own_capture_of_a_step(kt, heads, kv, d, start, bound):
    """Steps whose append is a launch of its own: one eager call of the same shapes on the stream has sized what
    a capture begun with HIP itself needs, with and without key splits."""
    from kotensor_amd import _lib
    banner("kv8-own-capture", heads, kv, d, start, bound)
    rng = np.random.default_rng(heads + d)
    k, v = _rows(rng, start + 4, kv, d), _rows(rng, start + 4, kv, d)
    one, two = (kt.QuantizedKVCache(1, kv, bound, d, "int8", 64) for _ in range(2))
    for c in (one, two):
        _append(kt, c, 0, k[:start], v[:start], 0)
        c.advance(start)
    freq, stream, out = _dev(kt, _inv_freq(d)), kt.Stream.create(), kt.DeviceBuffer(4 * heads * d)
    dq, dk, dv = kt.DeviceBuffer(4 * heads * d), kt.DeviceBuffer(4 * kv * d), kt.DeviceBuffer(4 * kv * d)
    q = rng.standard_normal((4, heads * d)).astype(np.float32)

    def run(cache):
        _lib.call("kt_rope_attention_kv8", dq.ptr, dk.ptr, dv.ptr, freq.ptr, 1, cache.position.ptr, bound, ctypes.byref(cache.cache), 0, heads, out.ptr, stream.handle)
        _lib.call("kt_position_add", cache.position.ptr, 1, stream.handle)

    def load(i):
        dq.upload(q[i])
        dk.upload(k[start + i])
        dv.upload(v[start + i])
        out.fill_zero()
        kt.synchronize()
    want = []
    for i in range(4):
        load(i)
        run(one)
        stream.synchronize()
        want.append(out.download(np.float32))
    hip, handle, graph, exe = _hip(), ctypes.c_void_p(stream.handle), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(handle, 1) == 0  # thread-local
    try:
        run(two)
    finally:
        assert hip.hipStreamEndCapture(handle, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    assert hip.hipGraphDestroy(graph) == 0
    for i in range(4):
        load(i)
        _lib.call("kt_graph_launch", exe, stream.handle)
        stream.synchronize()
        assert same_bits(out.download(np.float32), want[i]), i
    for a, b in zip(one.rows_numpy(0, 0, start + 4), two.rows_numpy(0, 0, start + 4)):
        assert same_bits(a, b)
    assert hip.hipGraphExecDestroy(exe) == 0
    stream.destroy()


def test_a_recording_without_an_eager_call(kt):
    """A step of 256 dims without key splits needs nothing of its stream: it is recorded on a new one."""
    from kotensor_amd import _lib
    banner("kv8-record-first")
    rng = np.random.default_rng(3)
    heads, kv, d = 4, 2, 256
    k, v, q = _rows(rng, 11, kv, d), _rows(rng, 11, kv, d), rng.standard_normal(heads * d).astype(np.float32)
    one, two = (kt.QuantizedKVCache(1, kv, 64, d, "e4m3", 32) for _ in range(2))
    for c in (one, two):
        _append(kt, c, 0, k[:10], v[:10], 0)
        c.advance(10)
    dq, dk, dv, freq, out = _dev(kt, q), _dev(kt, k[10]), _dev(kt, v[10]), _dev(kt, _inv_freq(d)), [kt.DeviceBuffer(q.nbytes) for _ in range(2)]
    stream, graph = kt.Stream.create(), ctypes.c_void_p()

    def run(cache, out, st):
        _lib.call("kt_rope_attention_kv8", dq.ptr, dk.ptr, dv.ptr, freq.ptr, 1, cache.position.ptr, 64, ctypes.byref(cache.cache), 0, heads, out.ptr, st)
    kt.synchronize()
    _lib.call("kt_graph_begin", stream.handle)
    try:
        run(one, out[0], stream.handle)
    finally:
        _lib.call("kt_graph_end", stream.handle, ctypes.byref(graph))
    _lib.call("kt_graph_launch", graph, stream.handle)
    stream.synchronize()
    run(two, out[1], None)
    kt.synchronize()
    assert same_bits(out[0].download(np.float32), out[1].download(np.float32))
    _lib.call("kt_graph_destroy", graph)
    stream.destroy()


@pytest.mark.parametrize("fmt,block", [("int8", 64), ("e4m3", 128)])
@pytest.mark.parametrize("tokens,start,heads,kv,d,wide", [(1, 980, 32, 8, 64, 1060), (1, 600, 32, 8, 128, 700), (7, 1000, 14, 2, 64, 9000), (16, 500, 6, 6, 32, 1100), (3, 630, 8, 1, 128, 5000)])
def test_bounds_on_both_sides_of_a_form(kt, fmt, block, tokens, start, heads, kv, d, wide):
    """A bound of up to 1024 keys (640 of 128 dims) takes the keys in one workgroup, a larger one in splits: the
    sums' order differs, so the bits may; each is within the tolerance."""
    banner("kv8-bounds", fmt, block, tokens, start, heads, kv, d, wide)
    rng = np.random.default_rng(start)
    n = start + tokens
    cache, keys, values = _filled(kt, rng, fmt, block, d, kv, n, wide)
    q = (1.5 * rng.standard_normal((tokens, heads * d))).astype(np.float32)
    want = kv8_ref.attend(q, keys, values, start, heads)
    for bound in (n, wide):
        assert normwise_rel(_attend(kt, cache, 0, q, start, heads, bound), want) <= _tolerance(q, keys, heads)


@pytest.mark.parametrize("fmt,block,d", [("int8", 64, 64), ("e4m3", 32, 256), ("int8", 128, 32)])
def test_values_are_read_to_any_float(kt, fmt, block, d):
    """Keys at 16 bytes, values at any float; the floats around them stay."""
    from kotensor_amd import _lib
    rng = np.random.default_rng(d)
    cache = kt.QuantizedKVCache(1, 2, 150, d, fmt, block)
    k, v = _rows(rng, 140, 2, d), _rows(rng, 140, 2, d)
    _append(kt, cache, 0, k, v, 0)
    want, count = cache.rows_numpy(0, 3, 130), 2 * 130 * d
    for offset in (1, 2, 3):
        banner("kv8-read-offset", fmt, d, offset)
        keys, values = (_dev(kt, np.full(count + 8, 7.0, np.float32)) for _ in range(2))
        _lib.call("kt_kv8_read", ctypes.byref(cache.cache), 0, 3, 130, keys.ptr + 16, values.ptr + 4 * offset, None)
        kt.synchronize()
        for buffer, first, rows in ((keys, 4, want[0]), (values, offset, want[1])):
            got = buffer.download(np.float32)
            assert same_bits(got[first:first + count].reshape(rows.shape), rows)
            assert np.all(got[:first] == 7.0) and np.all(got[first + count:] == 7.0)
