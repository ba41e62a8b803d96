"""Where the output of a controlled greedy decode starts: at the end of the last prefill, whatever
calls the tokens after it come from."""
import numpy as np
import pytest

from gpu_helpers import banner
from oracle import kv8_ref
from test_gpu_controls_pieces import PROMPT, _assert_pieces, _model, _prompt, _start

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,args", [("frequency", (1.0, 0.6, 0.0)), ("presence", (1.0, 0.0, 0.5)), ("all", (1.3, 0.3, 0.3))])
def test_pieces_are_one_call(kt, kind, args):
    """A later call's penalties count what the earlier ones generated."""
    banner("controls-output", kind)
    _assert_pieces(kt, _model(kt), kt.LogitsControls(*args))


def _plain_steps(model, text, start, count, args):
    """Tokens after text, whose output starts at start, with the controls restated on the host."""
    cache, buffers = model.new_cache(len(text) + count), model.new_inference_buffers(len(text) + count)
    x, text = model.prefill(text, cache, buffers).logits_numpy(), list(text)
    out = []
    for _ in range(count):
        y = kv8_ref.process_logits(x[None], [text], [len(text)], [start], *args)[0]
        order = np.sort(y)
        assert order[-1] - order[-2] > 1e-4  # no near tie: the choice is the same in fp32
        out.append(int(np.argmax(y)))
        text.append(out[-1])
        x = model.decode(out[-1], cache, buffers).logits_numpy()
    return out


@pytest.mark.parametrize("recorded", [False, True])
def test_steps_whose_first_token_had_no_controls(kt, recorded):
    """decode_step and replays with controls after a first token chosen without them: its position
    is the output's first."""
    banner("controls-output-step", recorded)
    args = (1.0, 0.7, 0.4)
    model, controls, stream = _model(kt), kt.LogitsControls(*args), kt.Stream.create()
    cache, buffers = _start(kt, model, stream)
    first = model.greedy_decode(cache, buffers, 0, stream)
    if recorded:
        model.decode_step(cache, buffers, stream)  # (sizes the workspaces; the second token has none either)
        graph = model.capture_decode(cache, buffers, stream, controls)
        graph.replay(5)
        stream.synchronize()
        graph.destroy()
        first = buffers.generated.download(np.int32, count=2, offset=4 * PROMPT).tolist()
    else:
        for _ in range(5):
            model.decode_step(cache, buffers, stream, controls)
        stream.synchronize()
    got = buffers.generated.download(np.int32, count=5, offset=4 * (PROMPT + len(first))).tolist()
    assert got == _plain_steps(model, _prompt() + first, PROMPT, 5, args)
    stream.destroy()


def test_a_later_prompt_starts_a_new_output(kt):
    """A second turn: its output starts behind its prompt, also for a graph recorded in the first."""
    banner("controls-output-turns")
    args = (1.0, 0.7, 0.4)
    model, controls, stream = _model(kt), kt.LogitsControls(*args), kt.Stream.create()
    cache, buffers = _start(kt, model, stream)
    model.greedy_decode(cache, buffers, 2, stream, controls=controls)
    graph = model.capture_decode(cache, buffers, stream, controls)
    graph.replay(2)
    stream.synchronize()
    said = buffers.generated.download(np.int32, count=4, offset=4 * PROMPT).tolist()  # (what the cache holds)
    turn = [5, 17, 30, 2]
    model.prefill(turn, cache, buffers, stream, record_tokens=True)
    text = _prompt() + said + turn
    assert cache.length == len(text)
    first = model.greedy_decode(cache, buffers, 0, stream, controls=controls)
    graph.replay(4)
    stream.synchronize()
    got = buffers.generated.download(np.int32, count=5, offset=4 * len(text)).tolist()
    assert got[:1] == first
    assert got == _plain_steps(model, text, len(text), 5, args)
    graph.destroy()
    stream.destroy()


def test_text_behind_the_buffers_end(kt):
    """A step whose own token has no place in the buffers' record is refused where penalties count it."""
    banner("controls-output-end")
    model, controls, stream = _model(kt), kt.LogitsControls(1.2), kt.Stream.create()
    cache, buffers = model.new_cache(20), model.new_inference_buffers(14)
    model.prefill(_prompt()[:10], cache, buffers, stream, record_tokens=True)
    model.greedy_decode(cache, buffers, 2, stream, controls=controls)
    graph = model.capture_decode(cache, buffers, stream, controls)
    with pytest.raises(kt.IllegalArgumentException, match="InferenceBuffers sized for 14"):
        graph.replay(3)
    graph.replay(1)
    model.decode_step(cache, buffers, stream, controls)  # takes the token at position 13; its own choice has no place
    for call in (lambda: model.decode_step(cache, buffers, stream, controls), graph.replay):
        with pytest.raises(kt.IllegalArgumentException, match="InferenceBuffers sized for 14"):
            call()
    assert cache.length == 14
    model.decode_step(cache, buffers, stream)  # without penalties as before
    stream.synchronize()
    graph.destroy()
    stream.destroy()
