"""Penalties, biases and masks on logits (kt_logits.hip) against 64 bits: at most four fp32 roundings of
values no larger than the result plus what was taken off, so 4 * 2^-24 of their sum; minus
infinities and untouched logits bit for bit."""
import ctypes

import numpy as np
import pytest

from gpu_helpers import banner, same_bits
from oracle import kv8_ref

pytestmark = pytest.mark.gpu


def _text(rng, rows, length, n):
    t = (n * rng.random((rows, length)) ** 5).astype(np.int32)
    t[rng.random((rows, length)) < 0.05] = -1
    t[rng.random((rows, length)) < 0.02] = n  # outside the vocabulary
    return t


def _check(got, logits, want, sizes):
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    fine = np.isfinite(want)
    off = np.abs(got[fine] - want[fine])
    assert np.all(off <= 4 * 2.0 ** -24 * (np.abs(want) + np.abs(logits) + sizes)[fine])


@pytest.mark.parametrize("rows,n,length", [(1, 1, 1), (1, 5, 0), (2, 31, 7), (3, 32, 100), (1, 4096, 300), (2, 4097, 4096), (5, 8191, 1000), (7, 32000, 2000), (1, 151936, 9000),
                                           (64, 1000, 33), (33, 49157, 500)])
@pytest.mark.parametrize("bias,mask", [(0, False), (3, True), (700, False), (0, True)])
def test_controls_against_64_bits(kt, rows, n, length, bias, mask):
    banner("logits", rows, n, length, bias, mask)
    rng = np.random.default_rng(rows + n + length)
    logits = (4.0 * rng.standard_normal((rows, n))).astype(np.float32)
    logits[0, 0] = 0.0
    text = _text(rng, rows, max(1, length), n)
    lengths, starts = rng.integers(0, length + 1, rows).astype(np.int32), rng.integers(-1, length + 1, rows).astype(np.int32)
    lengths[0] = length
    biases = {int(t): float(v) for t, v in zip(rng.permutation(n)[:min(bias, n)], rng.standard_normal(bias))}
    allowed = rng.random((rows, n)) < 0.4 if mask else None
    if mask and rows > 1:
        allowed[1] = False
    controls = kt.LogitsControls(1.3, 0.25, 0.5, biases, allowed)
    bufs = [kt.DeviceBuffer.from_numpy(a) for a in (text, lengths, starts)]
    dl = kt.DeviceTensor.from_numpy(logits)
    got = kt.process_logits(dl, controls, *bufs).numpy()
    want = kv8_ref.process_logits(logits, text, lengths, starts, 1.3, 0.25, 0.5, biases.items(), allowed)
    _check(got, logits, want, 0.25 * text.shape[1] + 3.0)
    kt.process_logits(dl, controls, *bufs, out=dl)  # in place: the same bits
    assert same_bits(dl.numpy(), got)


@pytest.mark.parametrize("rows,n,length", [(1100, 33, 9), (205, 4097, 100), (1025, 1000, 5)])
def test_segments_of_many_rows(kt, rows, n, length):
    test_controls_against_64_bits(kt, rows, n, length, 5, True)


@pytest.mark.parametrize("repetition,frequency,presence", [(1.0, 0.0, 0.0), (2.0, 0.0, 0.0), (1.0, 0.7, 0.0), (1.0, 0.0, -0.4), (0.5, -0.1, 0.3)])
def test_each_penalty(kt, repetition, frequency, presence):
    banner("logits-penalty", repetition, frequency, presence)
    rng = np.random.default_rng(2)
    logits, text, lengths = rng.standard_normal((2, 5000)).astype(np.float32), _text(rng, 2, 900, 5000), np.array([900, 3], np.int32)
    controls = kt.LogitsControls(repetition, frequency, presence)
    got = kt.process_logits(kt.DeviceTensor.from_numpy(logits), controls, kt.DeviceBuffer.from_numpy(text), kt.DeviceBuffer.from_numpy(lengths)).numpy()
    want = kv8_ref.process_logits(logits, text, lengths, None, repetition, frequency, presence)
    _check(got, logits, want, 900.0)
    untouched = want == logits
    assert same_bits(got[untouched], logits[untouched])


def test_values_that_are_not_finite(kt):
    """Infinities and NaNs stay, unless masked."""
    logits = np.array([[np.inf, -np.inf, np.nan, np.nan, 3.4e38, 1e-45, -0.0, 1.0]], np.float32)
    text = np.array([[0, 1, 2, 4, 4, 5, 6]], np.int32)
    allowed = np.array([True, True, True, False, True, True, True, False])
    got = kt.process_logits(kt.DeviceTensor.from_numpy(logits), kt.LogitsControls(1.5, 0.1, 0.0, None, allowed), kt.DeviceBuffer.from_numpy(text),
                            kt.DeviceBuffer.from_numpy(np.array([7], np.int32))).numpy()[0]
    assert np.isposinf(got[0]) and np.isneginf(got[1]) and np.isnan(got[2]) and np.isneginf(got[3]) and np.isneginf(got[7])
    assert abs(got[4] / np.float64(np.float32(3.4e38) / 1.5) - 1) < 1e-6 and got[6] == np.float32(-0.1)


def test_rows_with_strides_and_repeated_biases(kt):
    """The C entry: rows of a wider matrix, unaligned, one text and one mask for all rows, biases given
    twice (the later holds), ids outside; the columns between the rows stay."""
    from kotensor_amd import _lib
    rng = np.random.default_rng(4)
    rows, n, stride, cap = 3, 5003, 5010, 50
    for offset in (0, 1):
        banner("logits-strides", offset)
        wide = rng.standard_normal(rows * stride + 8).astype(np.float32)
        logits = np.stack([wide[offset + r * stride:offset + r * stride + n] for r in range(rows)])
        text, lengths = _text(rng, 1, cap, n), np.array([50, 0, 200], np.int32)
        tokens = np.array([5, 9, 5, 5, -1, n, 4999, 9], np.int32)
        values = rng.standard_normal(8).astype(np.float32)
        allowed = rng.random(n) < 0.5
        words = np.packbits(np.concatenate([allowed, np.zeros(-n % 32, bool)]), bitorder="little").view(np.uint32)
        bufs = [kt.DeviceBuffer.from_numpy(a) for a in (wide, text, lengths, tokens, values, words)]
        out = kt.DeviceBuffer.from_numpy(np.full(rows * (stride + 3), 7.0, np.float32))
        c = _lib.LogitsControls()
        c.history, c.history_length, c.history_stride, c.history_capacity, c.length_offset = bufs[1].ptr, bufs[2].ptr, 0, cap, -1
        c.repetition, c.frequency, c.presence = 1.2, 0.1, 0.0
        c.bias_count, c.bias_tokens, c.bias_values, c.allowed = 8, bufs[3].ptr, bufs[4].ptr, bufs[5].ptr
        _lib.call("kt_process_logits", bufs[0].ptr + 4 * offset, rows, n, stride, ctypes.byref(c), out.ptr, stride + 3, None)
        got = out.download(np.float32).reshape(rows, stride + 3)
        assert np.all(got[:, n:] == 7.0)
        want = kv8_ref.process_logits(logits, [text[0]] * rows, [49, -1, 50], None, 1.2, 0.1, 0.0, zip(tokens.tolist(), values.tolist()), allowed)
        _check(got[:, :n], logits, want, 10.0)


def test_a_recorded_step_follows_its_text(kt):
    from kotensor_amd import _lib
    banner("logits-record")
    rng = np.random.default_rng(5)
    n, cap = 7000, 40
    logits, text = rng.standard_normal((1, n)).astype(np.float32), _text(rng, 1, cap, n)
    dl, dt, pos, out = kt.DeviceTensor.from_numpy(logits), kt.DeviceBuffer.from_numpy(text), kt.DeviceBuffer.from_numpy(np.zeros(1, np.int32)), kt.DeviceBuffer(4 * n)
    controls = kt.LogitsControls(1.4, 0.2, 0.1, {3: 1.0}, np.ones(n, bool))
    c = controls.descriptor(1, n, dt, pos, None, cap, cap, 1)
    stream, graph = kt.Stream.create(), ctypes.c_void_p()
    _lib.call("kt_graph_begin", stream.handle)
    try:
        _lib.call("kt_process_logits", dl.ptr, 1, n, n, ctypes.byref(c), out.ptr, n, stream.handle)
        _lib.call("kt_position_add", pos.ptr, 1, stream.handle)
    finally:
        _lib.call("kt_graph_end", stream.handle, ctypes.byref(graph))
    try:
        for i in range(5):
            allowed = rng.random(n) < 0.7
            controls.set_allowed(allowed, stream)
            _lib.call("kt_graph_launch", graph, stream.handle)
            stream.synchronize()
            want = kv8_ref.process_logits(logits, text, [i + 1], None, 1.4, 0.2, 0.1, {3: 1.0}.items(), allowed)
            _check(out.download(np.float32).reshape(1, n), logits, want, 10.0)
    finally:
        stream.synchronize()
        _lib.call("kt_graph_destroy", graph)
        stream.destroy()


def _plain_generate(kt, model, prompt, count, controls, cache_format):
    """generate with the controls restated on the host, a step at a time."""
    cache, buffers = model.new_cache(len(prompt) + count, cache_format=cache_format), model.new_inference_buffers(len(prompt) + count)
    text = list(prompt)
    x = model.prefill(prompt, cache, buffers).logits_numpy()
    for i in range(count):
        y = kv8_ref.process_logits(x[None], [text], [len(text)], [len(prompt)], *controls)[0]
        order = np.sort(y)
        assert order[-1] - order[-2] > 1e-4  # no near tie: the choice is the same in fp32
        text.append(int(np.argmax(y)))
        if i + 1 < count:
            x = model.decode(text[-1], cache, buffers).logits_numpy()
    return text


@pytest.mark.parametrize("cache_format", [None, "int8"])
def test_generate_with_controls(kt, cache_format):
    """Prompt, cache, attention, logits and controls together: the tokens are those of the controls
    on the host, by graph replays and by eager steps; without controls as before."""
    banner("logits-generate", cache_format)
    rng = np.random.default_rng(7)
    n = 400
    model = kt.Transformer(n, 128, 2, 2, 256, 1, quantization=kt.Quantization(8, 32), seed=5, init_std=0.1)
    prompt = rng.integers(0, n, 40).tolist()
    plain = model.generate(prompt, 30, cache_format=cache_format)
    allowed = rng.random(n) < 0.8
    bias = {int(plain[-1]): -1.5, 17: 0.7}
    controls = kt.LogitsControls(1.2, 0.15, 0.3, bias, allowed)
    want = _plain_generate(kt, model, prompt, 30, (1.2, 0.15, 0.3, bias.items(), allowed), cache_format)
    for graph in (True, False):
        assert model.generate(prompt, 30, use_graph=graph, cache_format=cache_format, controls=controls) == want
    assert all(allowed[t] for t in want[40:])
    assert model.generate(prompt, 30, cache_format=cache_format) == plain


def test_penalties_need_the_text(kt):
    model = kt.Transformer(100, 128, 1, 2, 128, 1, quantization=kt.Quantization(8, 32))
    cache, buffers, controls = model.new_cache(60), model.new_inference_buffers(60), kt.LogitsControls(1.2)
    model.prefill([1, 2, 3], cache, buffers)
    with pytest.raises(kt.IllegalArgumentException, match="record_tokens"):
        model.greedy_decode(cache, buffers, 4, controls=controls)
    cache.reset()
    model.prefill([1, 2, 3], cache, buffers, record_tokens=True)
    model.greedy_decode(cache, buffers, 4, controls=controls)
    model.greedy_decode(cache, buffers, 4, controls=controls)  # goes on with its own text
    model.decode(5, cache, buffers)  # a token that is not recorded
    with pytest.raises(kt.IllegalArgumentException, match="record_tokens"):
        model.greedy_decode(cache, buffers, 4, controls=controls)
    with pytest.raises(kt.IllegalArgumentException, match="out of vocab"):
        kt.LogitsControls(bias={100: 1.0}).descriptor(1, 100)
    with pytest.raises(kt.IllegalArgumentException, match="mask of 4 words"):
        kt.LogitsControls(allowed=np.ones(100, bool)).descriptor(1, 200)
    with pytest.raises(kt.IllegalArgumentException, match="mask of 2 rows"):
        kt.LogitsControls(allowed=np.ones((2, 100), bool)).descriptor(1, 100)
    with pytest.raises(kt.IllegalArgumentException, match="history"):
        kt.process_logits(kt.DeviceTensor.zeros((1, 100)), controls)


def test_text_of_an_earlier_sequence_does_not_count(kt):
    model = kt.Transformer(100, 128, 1, 2, 128, 1, quantization=kt.Quantization(8, 32))
    cache, buffers, controls, stream = model.new_cache(60), model.new_inference_buffers(60), kt.LogitsControls(1.2), kt.Stream.create()
    model.prefill(list(range(20)), cache, buffers, stream, record_tokens=True)
    model.greedy_decode(cache, buffers, 4, stream, controls=controls)
    graph = model.capture_decode(cache, buffers, stream, controls)
    graph.replay(2)
    cache.reset(stream)
    for token in (7, 8, 9):
        model.decode(token, cache, buffers, stream)
    for call in (lambda: model.greedy_decode(cache, buffers, 4, stream, controls=controls), lambda: model.decode_step(cache, buffers, stream, controls), graph.replay):
        with pytest.raises(kt.IllegalArgumentException, match="record_tokens"):
            call()
    stream.synchronize()
    graph.destroy()
    stream.destroy()


def test_a_mask_keeps_its_shape(kt):
    controls = kt.LogitsControls(allowed=np.ones(100, bool))
    for shape in ((1, 100), (129,), (4, 100)):
        with pytest.raises(kt.IllegalArgumentException, match="cannot replace"):
            controls.set_allowed(np.ones(shape, bool))
    controls.set_allowed(np.zeros(128, bool))  # as many words
