"""A controlled greedy decode made in pieces: whatever calls it is cut into, its tokens are those of
one call, since the controls act on the model's logits once and the output is one text."""
import numpy as np
import pytest

from gpu_helpers import banner, same_bits

pytestmark = pytest.mark.gpu

N, PROMPT = 64, 40  # (most of the vocabulary is in the text)


def _model(kt):
    return kt.Transformer(N, 128, 2, 2, 256, 1, quantization=kt.Quantization(8, 32), seed=5, init_std=0.1)


def _prompt(seed=7):
    return np.random.default_rng(seed).integers(0, N, PROMPT).tolist()


def _bias(scale=2.0):
    return {t: float(v) for t, v in enumerate(scale * np.random.default_rng(3).standard_normal(N))}


def _mask():
    return np.random.default_rng(4).random(N) < 0.5


def _start(kt, model, stream, seed=7):
    cache, buffers = model.new_cache(PROMPT + 60), model.new_inference_buffers(PROMPT + 60)
    model.prefill(_prompt(seed), cache, buffers, stream, record_tokens=True)
    return cache, buffers


def _pieces(kt, model, controls, graph, steps, seed):
    stream = kt.Stream.create()
    cache, buffers = _start(kt, model, stream, seed)
    out = []
    for count in steps:
        got = model.greedy_decode(cache, buffers, count, stream, graph, controls)
        assert not out or out[-1] == got[0]  # the token that the call before returned last
        out += got if not out else got[1:]
    stream.destroy()
    return out


def _steps_then_a_call(kt, model, controls, seed):
    """One token, single steps, replays, then a call that goes on."""
    stream = kt.Stream.create()
    cache, buffers = _start(kt, model, stream, seed)
    model.greedy_decode(cache, buffers, 0, stream, controls=controls)
    for _ in range(2):
        model.decode_step(cache, buffers, stream, controls)
    graph = model.capture_decode(cache, buffers, stream, controls)
    graph.replay(2)
    model.greedy_decode(cache, buffers, 4, stream, controls=controls)
    stream.synchronize()
    graph.destroy()
    stream.destroy()
    return buffers.generated.download(np.int32, count=9, offset=4 * PROMPT).tolist()


def _assert_pieces(kt, model, controls):
    for seed in (7, 8, 9):
        whole = model.generate(_prompt(seed), 9, controls=controls)[PROMPT:]
        for graph in (True, False):
            for steps in ((3, 1, 4), (0, 0, 8), (8, 0), (1,) * 8):
                assert _pieces(kt, model, controls, graph, steps, seed) == whole, (seed, graph, steps)
        assert _steps_then_a_call(kt, model, controls, seed) == whole, seed


ONCE = {"repetition": lambda: {"repetition_penalty": 1.3}, "a little repetition": lambda: {"repetition_penalty": 1.1}, "bias": lambda: {"bias": _bias(0.5)},
        "mask": lambda: {"bias": _bias(1.0), "allowed": _mask()}}


@pytest.mark.parametrize("kind", list(ONCE))
def test_pieces_are_one_call(kt, kind):
    """x / 1.3 and x + bias once, not once a call."""
    banner("controls-pieces", kind)
    _assert_pieces(kt, _model(kt), kt.LogitsControls(**ONCE[kind]()))


def test_logits_stay_the_models(kt):
    """buffers.logits are the model's own after controlled steps, as without controls."""
    banner("controls-logits")
    model, stream = _model(kt), kt.Stream.create()
    cache, buffers = _start(kt, model, stream)
    first = buffers.logits_numpy(stream)
    tokens = model.greedy_decode(cache, buffers, 3, stream, controls=kt.LogitsControls(1.5, bias=_bias()))
    got = buffers.logits_numpy(stream)
    cache, buffers = _start(kt, model, stream)
    assert same_bits(buffers.logits_numpy(stream), first)
    for token in tokens[:3]:
        model.decode(token, cache, buffers, stream)
    assert same_bits(buffers.logits_numpy(stream), got)
    stream.destroy()
