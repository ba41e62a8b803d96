"""A mask has an entry for every token of the vocabulary."""
import numpy as np
import pytest

from gpu_helpers import banner

pytestmark = pytest.mark.gpu


def _model(kt):
    return kt.Transformer(100, 128, 1, 2, 128, 1, quantization=kt.Quantization(8, 32))


def _packed(allowed):
    return np.packbits(np.concatenate([allowed, np.zeros(-len(allowed) % 32, bool)]), bitorder="little").view(np.uint32)


@pytest.mark.parametrize("entries", [97, 99, 101, 128])
def test_a_mask_of_another_length(kt, entries):
    """As many words as the vocabulary's, but another number of tokens."""
    banner("controls-mask", entries)
    controls = kt.LogitsControls(allowed=np.ones(entries, bool))
    with pytest.raises(kt.IllegalArgumentException, match=f"mask of {entries} tokens .* 100"):
        controls.descriptor(1, 100)
    with pytest.raises(kt.IllegalArgumentException, match=f"mask of {entries} tokens"):
        _model(kt).generate([1, 2, 3], 4, controls=controls)
    rows = kt.LogitsControls(allowed=np.ones((2, entries), bool))
    with pytest.raises(kt.IllegalArgumentException, match=f"mask of {entries} tokens"):
        kt.process_logits(kt.DeviceTensor.zeros((2, 100)), rows)


def test_a_mask_replaced_by_one_of_another_length(kt):
    """What a recorded step reads next; packed words hold no length."""
    banner("controls-mask-replaced")
    controls = kt.LogitsControls(allowed=np.ones(100, bool))
    controls.descriptor(1, 100)
    for entries in (97, 128):
        with pytest.raises(kt.IllegalArgumentException, match=f"mask of {entries} tokens"):
            controls.set_allowed(np.ones(entries, bool))
    allowed = np.random.default_rng(1).random(100) < 0.5
    logits = kt.DeviceTensor.from_numpy(np.random.default_rng(2).standard_normal((1, 100)).astype(np.float32))
    for mask in (allowed, _packed(~allowed), np.ones(100, bool), _packed(allowed).view(np.int32)):
        controls.set_allowed(mask)
        want = mask if mask.dtype == bool else np.unpackbits(mask.view(np.uint8), bitorder="little")[:100] > 0
        assert np.array_equal(np.isfinite(kt.process_logits(logits, controls).numpy()[0]), want)


def _words_behind(count):
    words = np.zeros((count + 31) // 32, np.uint32)
    words[-1] = 0xFFFFFFFF << (count % 32) & 0xFFFFFFFF
    return words


DEAD = {"none": lambda: {"allowed": np.zeros(100, bool)}, "behind the vocabulary": lambda: {"allowed": _words_behind(100)},
        "all banned": lambda: {"bias": {t: -np.inf for t in range(100)}},
        "the allowed banned": lambda: {"allowed": np.arange(100) % 50 == 7, "bias": {7: -1e9, 57: -np.inf, 3: 2.0}}}


@pytest.mark.parametrize("kind", list(DEAD))
def test_nothing_may_follow(kt, kind):
    """A grammar at its end leaves no token to choose: every call that would choose one refuses."""
    banner("controls-mask-dead", kind)
    model, controls, stream = _model(kt), kt.LogitsControls(**DEAD[kind]()), kt.Stream.create()
    cache, buffers = model.new_cache(20), model.new_inference_buffers(20)
    model.prefill([1, 2, 3], cache, buffers, stream)
    for call in (lambda: model.greedy_decode(cache, buffers, 4, stream, controls=controls), lambda: model.generate([1, 2, 3], 4, controls=controls),
                 lambda: model.decode_step(cache, buffers, stream, controls)):
        with pytest.raises(kt.IllegalArgumentException, match="no token may follow"):
            call()
    assert cache.length == 3
    model.greedy_decode(cache, buffers, 0, stream)
    model.decode_step(cache, buffers, stream)
    graph = model.capture_decode(cache, buffers, stream, controls)  # (its mask may be another one when it is replayed)
    with pytest.raises(kt.IllegalArgumentException, match="no token may follow"):
        graph.replay()
    stream.synchronize()
    graph.destroy()
    logits = kt.DeviceTensor.zeros((1, 100))  # the logits themselves may be asked for
    assert np.all(kt.process_logits(logits, controls).numpy()[0] <= -1e9)
    stream.destroy()


def test_a_grammar_that_ends_between_replays(kt):
    banner("controls-mask-ends")
    model, stream = _model(kt), kt.Stream.create()
    controls = kt.LogitsControls(bias={40: 5.0}, allowed=np.ones(100, bool))
    cache, buffers = model.new_cache(20), model.new_inference_buffers(20)
    model.prefill([1, 2, 3], cache, buffers, stream)
    model.greedy_decode(cache, buffers, 2, stream, controls=controls)
    graph = model.capture_decode(cache, buffers, stream, controls)
    controls.set_allowed(np.zeros(100, bool), stream)
    with pytest.raises(kt.IllegalArgumentException, match="no token may follow"):
        graph.replay()
    for only in (61, 40):
        controls.set_allowed(np.arange(100) == only, stream)
        graph.replay()
        stream.synchronize()
        assert buffers.tokens.download(np.int32, count=1)[0] == only
    graph.destroy()
    stream.destroy()


def test_a_first_mask_after_the_recording(kt):
    """A step recorded without a mask addresses none: a replay does not pass over one that was set since."""
    banner("controls-mask-first")
    model, stream = _model(kt), kt.Stream.create()
    controls = kt.LogitsControls(bias={40: 5.0})
    cache, buffers = model.new_cache(20), model.new_inference_buffers(20)
    model.prefill([1, 2, 3], cache, buffers, stream)
    model.greedy_decode(cache, buffers, 2, stream, controls=controls)
    graph = model.capture_decode(cache, buffers, stream, controls)
    graph.replay()
    controls.set_allowed(np.arange(100) == 61, stream)
    length = cache.length
    with pytest.raises(kt.IllegalStateException, match="recorded without a mask"):
        graph.replay()
    assert cache.length == length
    again = model.capture_decode(cache, buffers, stream, controls)
    again.replay()
    stream.synchronize()
    assert buffers.tokens.download(np.int32, count=1)[0] == 61
    graph.destroy()
    again.destroy()
    stream.destroy()
