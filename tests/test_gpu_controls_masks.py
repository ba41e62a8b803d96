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
