"""Several sequences over a cache in pages through Transformer: prompts and steps in one call, recorded steps,
trees of drafted tokens, against the oracle's decoder whose cache is held in the same format."""
import numpy as np
import pytest

from conftest import normwise_rel
from gpu_helpers import banner, same_bits
from oracle import decoder_ref, paged_ref

pytestmark = pytest.mark.gpu

# Logits, normwise. Projections of three rows and more round to fp16 (1e-2 through the small model's layers, as for prompts in
# one sequence). The cache rounds rows that differ by some 1e-3 of their size from the oracle's: as fp16 an element then
# differs by a step of 2^-10 at most, ten times that through the layers; as bf16 one element in five by a step
# of 2^-7 at most (mean square root 2^-8 of each), which is 2e-3 of a row, and ten times that.
TOLERANCE = {"float32": 1e-2, "float16": 2e-2, "bfloat16": 4e-2}


def held_oracle(model, fmt):
    """to_oracle of test_gpu_decoder.py with the cache's rows rounded to `fmt`."""
    from test_gpu_decoder import to_oracle
    plain = to_oracle(None, model)

    class Held(decoder_ref.RefTransformer):
        def _layer(self, x, cache, layer):
            c = self.config
            p, start, kv, d = f"block.{layer}.", cache.length, c.num_key_value_heads, c.head_dim
            import oracle
            normed = oracle.rmsnorm(x, self.norms[p + "norm1"], c.norm_eps)
            q, k, v = (self._project(normed, p + "attention." + w) for w in ("wQ", "wK", "wV"))
            q, k = (oracle.rope_rows(y, d, self.inv_freq, start) for y in (q, k))
            n = start + x.shape[0]
            rows = []
            for held, new in ((cache.keys, k), (cache.values, v)):
                held = held.reshape(c.num_layers, kv, -1, d)
                held[layer, :, start:n] = paged_ref.stored(np.ascontiguousarray(new.reshape(-1, kv, d).transpose(1, 0, 2)), fmt)
                rows.append(held[layer, :, :n].astype(np.float64))
            visible = np.arange(n)[None] <= start + np.arange(x.shape[0])[:, None]
            context = paged_ref.attend(q.reshape(-1, c.num_heads, d).astype(np.float64), *rows, visible)[0]
            x = (x + self._project(context.reshape(x.shape[0], -1).astype(np.float32), p + "attention.wOut")).astype(np.float32)
            normed = oracle.rmsnorm(x, self.norms[p + "norm2"], c.norm_eps)
            fused = oracle.silu_mul(self._project(normed, p + "ffn.wGate"), self._project(normed, p + "ffn.wUp"))
            return (x + self._project(fused, p + "ffn.wDown")).astype(np.float32)

    return Held(plain.config, plain.quantized, plain.norms, tied=model.tied)


def logits_of(ref, text):
    return ref.prefill(list(text), ref.new_cache(len(text)))


def small(kt, seed=5, layers=2, tied=False):
    model = kt.Transformer(300, 128, layers, 4, 192, 2, quantization=kt.Quantization(8, 32), seed=seed, init_std=0.12)
    if tied:
        model.tie_embedding_to_head()
    return model


@pytest.mark.parametrize("rows,n", [(1, 1), (1, 32000), (3, 1), (5, 1000), (64, 32000), (700, 4099), (3000, 61)])
def test_argmax_of_rows(kt, oracle_lib, rows, n):
    banner("argmax rows", rows, n)
    rng = np.random.default_rng(rows + n)
    x = rng.standard_normal((rows, n)).astype(np.float32)
    x[rows // 2, :] = -2e9                      # none is a candidate
    x[rows // 3, rng.integers(0, n, 4)] = 9.0   # a tie: the first
    x[rows // 4, rng.integers(0, n)] = np.nan
    x[rows // 5, rng.integers(0, n)] = np.inf
    want = [oracle_lib.argmax(row) for row in x]
    logits, tokens = kt.DeviceBuffer.from_numpy(x), kt.DeviceBuffer(4 * rows)
    from kotensor_amd import _lib
    positions = rng.integers(-2, 9, rows).astype(np.int32)
    before = np.full((rows, 7), -5, np.int32)
    place, generated = kt.DeviceBuffer.from_numpy(positions), kt.DeviceBuffer.from_numpy(before)
    for _ in range(2):  # (the counters are zero again)
        _lib.call("kt_argmax_rows", logits.ptr, rows, n, tokens.ptr, place.ptr, generated.ptr, 7, None)
        assert tokens.download(np.int32).tolist() == want
    for row, position in enumerate(positions):
        if 0 <= position < 7:
            before[row, position] = want[row]
    assert np.array_equal(generated.download(np.int32).reshape(rows, 7), before)
    assert np.array_equal(place.download(np.int32), positions)
    tokens.fill_zero()
    _lib.call("kt_argmax_rows", logits.ptr, rows, n, tokens.ptr, None, None, 0, None)
    assert tokens.download(np.int32).tolist() == want


@pytest.mark.parametrize("fmt", list(TOLERANCE))
@pytest.mark.parametrize("rows", [8, 64, 512])
def test_prompts_and_steps_in_one_call(kt, oracle_lib, fmt, rows):
    """extend: prompts of any length, in as many parts as the buffers ask for, beside single tokens of other sequences; sequences
    that leave and others that come take their pages."""
    model = small(kt)
    ref = held_oracle(model, fmt)
    rng = np.random.default_rng(3)
    cache = model.new_paged_cache(5, 150, fmt, 16, pages=24)
    buffers = model.new_batch_buffers(cache, rows)
    texts = {s: [] for s in range(5)}

    def call(new):
        banner("extend", fmt, rows, {s: len(t) for s, t in new.items()})
        chosen = model.extend(new, cache, buffers)
        logits = buffers.logits.download(np.float32, count=len(new) * 300).reshape(len(new), 300)
        for row, s in enumerate(sorted(new)):
            texts[s] += new[s]
            want = logits_of(ref, texts[s])
            print(f"  {normwise_rel(logits[row], want):.2e}", flush=True)
            assert normwise_rel(logits[row], want) <= TOLERANCE[fmt], s
            assert chosen[s] == oracle_lib.argmax(logits[row])
        assert cache.lengths == [len(texts[s]) for s in range(5)]
        assert cache.device_lengths.download(np.int32).tolist() == cache.lengths

    draw = lambda n: rng.integers(0, 300, n).tolist()
    call({0: draw(33), 1: draw(1), 3: draw(70), 4: draw(16)})
    call({0: draw(1), 3: draw(1), 1: draw(1)})
    call({2: draw(90), 1: draw(3), 0: draw(1)})
    for s in (3, 0):
        cache.release(s)
        texts[s] = []
    call({3: draw(17), 0: draw(100)})
    call({s: draw(1) for s in range(5)})
    held = cache.free_pages
    with pytest.raises(kt.IllegalArgumentException, match="free"):
        cache.reserve({s: 45 for s in range(5)})  # (none past maxSequenceLength)
    assert cache.free_pages == held


@pytest.mark.parametrize("fmt,tied", [("float32", False), ("float16", True), ("bfloat16", False)])
@pytest.mark.parametrize("n", [1, 3, 20])
def test_recorded_steps_equal_eager_ones_and_single_calls(kt, oracle_lib, fmt, tied, n):
    """generate_batch: eager and replayed steps give the same tokens as calls of one token a sequence, bit for bit, whose logits
    are the oracle's."""
    model = small(kt, tied=tied)
    ref = held_oracle(model, fmt)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 300, int(k)).tolist() for k in rng.integers(1, 60, n)]
    banner("generate batch", fmt, tied, n)
    eager = model.generate_batch(prompts, 9, use_graph=False, cache_format=fmt, page_tokens=16)
    assert eager == model.generate_batch(prompts, 9, cache_format=fmt, page_tokens=16)
    assert eager == model.generate_batch(prompts, 9, cache_format=fmt, page_tokens=16)
    cache = model.new_paged_cache(n, 70, fmt, 16)
    buffers = model.new_batch_buffers(cache)
    chosen = model.extend(dict(enumerate(prompts)), cache, buffers)
    for step in range(9):
        assert [chosen[s] for s in range(n)] == [eager[s][len(prompts[s]) + step] for s in range(n)]
        if step == 8:
            break
        chosen = model.extend({s: [chosen[s]] for s in range(n)}, cache, buffers)
        if step in (0, 7):
            logits = buffers.logits.download(np.float32, count=n * 300).reshape(n, 300)
            for s in range(0, n, 7):
                assert normwise_rel(logits[s], logits_of(ref, eager[s][:len(prompts[s]) + step + 1])) <= TOLERANCE[fmt]
    stop = eager[0][len(prompts[0]) + 4]
    stopped = model.generate_batch(prompts, 9, stop_tokens=[stop], cache_format=fmt, page_tokens=16)
    for s in range(n):
        out = eager[s][len(prompts[s]):]
        assert stopped[s] == prompts[s] + (out[:out.index(stop)] if stop in out else out)


def test_steps_go_on_and_several_recordings_share_a_stream(kt):
    """Two caches' steps on one stream in turn, each call from the last token of the one before."""
    model = small(kt)
    rng = np.random.default_rng(6)
    stream = kt.Stream.create()
    prompts = [rng.integers(0, 300, k).tolist() for k in (40, 5, 17)]
    want = model.generate_batch(prompts, 13, stream=stream)
    made = [{}, {}]
    sides = []
    for _ in made:
        cache = model.new_paged_cache(3, 70, stream=stream)
        sides.append((cache, model.new_batch_buffers(cache)))
    for side, (cache, buffers) in enumerate(sides):
        first = model.extend(dict(enumerate(prompts)), cache, buffers, stream)
        made[side] = [prompts[s] + [first[s]] for s in range(3)]
    for steps in (5, 1, 2, 4):
        for side, (cache, buffers) in enumerate(sides):
            more = model.greedy_decode_batch([t[-1] for t in made[side]], cache, buffers, steps, stream)
            made[side] = [t + m for t, m in zip(made[side], more)]
    assert made[0] == made[1] == want
    stream.destroy()


@pytest.mark.parametrize("fmt", list(TOLERANCE))
def test_drafted_tokens(kt, oracle_lib, fmt):
    """draft_step against the oracle: trees that hold what follows, beside what does not; the cache afterwards is that of the
    tokens kept."""
    model = small(kt)
    ref = held_oracle(model, fmt)
    rng = np.random.default_rng(7)
    prompts = {0: rng.integers(0, 300, 30).tolist(), 2: rng.integers(0, 300, 3).tolist(), 3: rng.integers(0, 300, 61).tolist()}
    plain = dict(zip(prompts, model.generate_batch(list(prompts.values()), 12, cache_format=fmt, page_tokens=16)))
    cache = model.new_paged_cache(4, 120, fmt, 16)
    buffers = model.new_batch_buffers(cache, 64)
    chosen = model.extend(prompts, cache, buffers)
    text = {s: prompts[s] + [chosen[s]] for s in prompts}
    taken = 0
    for step in range(3):
        drafts = {}
        for s in prompts:
            if s == 3 and step == 1:
                continue  # (a sequence that sits a call out)
            follow = plain[s][len(text[s]):len(text[s]) + 3] if plain[s][:len(text[s])] == text[s] else []
            tokens, parents = [text[s][-1]], [-1]
            for t in follow:  # each beside a wrong one, first
                parents += [len(tokens) - 1] * 2
                tokens += [(t + 1) % 300, t]
            tokens += rng.integers(0, 300, 4).tolist()
            parents += [0, len(tokens) - 4, len(tokens) - 3, 0]
            drafts[s] = (tokens, parents)
        banner("draft step", fmt, step, {s: len(t) for s, (t, _) in drafts.items()})
        before = {s: list(text[s]) for s in drafts}
        for s, out in model.draft_step(drafts, cache, buffers).items():
            text[s] += out
            taken += len(out) - 1
        for s in drafts:
            rc = ref.new_cache(len(text[s]))
            logits = ref.prefill(before[s], rc)
            for t in text[s][len(before[s]):]:
                # (an argmax over logits that differ by `tolerance` of the norm in all is as large but for twice that)
                assert logits[t] >= logits.max() - 2 * TOLERANCE[fmt] * np.linalg.norm(logits)
                if rc.length + 1 < len(text[s]):
                    logits = ref.decode(t, rc)
        assert cache.device_lengths.download(np.int32).tolist() == cache.lengths
        for s in prompts:
            assert cache.lengths[s] == len(text[s]) - 1
    assert taken >= 6  # (of up to 24 drafts that follow: a near tie may end a tree's use, not all of them)
    for s in prompts:  # the cache is that of the texts
        rc = ref.new_cache(len(text[s]))
        ref.prefill(text[s][:-1], rc)
        n = len(text[s]) - 1
        for layer in range(2):
            for got, want in zip(cache.rows_numpy(layer, s), (rc.keys, rc.values)):
                want = want.reshape(2, 2, -1, 32)[layer, :, :n]
                assert normwise_rel(got, want) <= TOLERANCE[fmt]
    after = model.extend({s: [text[s][-1]] for s in text}, cache, buffers)
    logits = buffers.logits.download(np.float32, count=3 * 300).reshape(3, 300)
    for row, s in enumerate(text):
        assert normwise_rel(logits[row], logits_of(ref, text[s])) <= TOLERANCE[fmt]
        assert after[s] == oracle_lib.argmax(logits[row])


def test_generate_with_drafts_from_the_text(kt, oracle_lib):
    """generate_batch with TextDraft, and with drafts that are never right, chooses tokens that the oracle would choose."""
    model = small(kt)
    ref = held_oracle(model, "float32")
    rng = np.random.default_rng(8)
    run = rng.integers(0, 300, 12).tolist()
    prompts = [run * 3, rng.integers(0, 300, 9).tolist(), run[:5] + run]
    never = lambda text: ([0] if text[-1] else [1], [-1])
    none = lambda text: ([], [])
    for draft in (kt.TextDraft(), kt.TextDraft(3, 1, 1), never, none):
        banner("generate with drafts", draft)
        made = model.generate_batch(prompts, 24, draft=draft, rows=64)
        for prompt, tokens in zip(prompts, made):
            assert tokens[:len(prompt)] == prompt and len(tokens) == len(prompt) + 24
            rc = ref.new_cache(len(tokens))
            logits = ref.prefill(prompt, rc)
            for t in tokens[len(prompt):]:
                assert logits[t] >= logits.max() - 2 * TOLERANCE["float32"] * np.linalg.norm(logits)
                logits = ref.decode(t, rc) if rc.length < len(tokens) - 1 else logits
        stop = made[0][len(prompts[0]) + 7]
        stopped = model.generate_batch(prompts, 24, stop_tokens=[stop], draft=draft, rows=64)
        assert stop not in [t for p, out in zip(prompts, stopped) for t in out[len(p):]]
        out = made[0][len(prompts[0]):]
        assert stopped[0][:len(prompts[0])] == prompts[0] and len(stopped[0]) <= len(made[0])


def test_shared_beginnings(kt):
    """share: pages of a common beginning serve two sequences, which go on apart; the first may leave."""
    model = small(kt)
    ref = held_oracle(model, "float16")
    rng = np.random.default_rng(9)
    cache = model.new_paged_cache(3, 100, "float16", 16, pages=10)
    buffers = model.new_batch_buffers(cache, 64)
    start = rng.integers(0, 300, 41).tolist()
    model.extend({0: start}, cache, buffers)
    assert cache.share(0, 1, 41) == 32 and cache.lengths[1] == 32 and cache.free_pages == 7
    assert cache.share(0, 2, 15) == 0 and cache.lengths[2] == 0
    with pytest.raises(kt.IllegalArgumentException, match="shared"):
        cache.set_length(0, 20)
    with pytest.raises(kt.IllegalArgumentException, match="not empty"):
        cache.share(0, 1, 16)
    cache.set_length(0, 33)
    texts = {0: start[:33] + rng.integers(0, 300, 7).tolist(), 1: start[:32] + rng.integers(0, 300, 20).tolist()}
    held = [a.copy() for a in cache.rows_numpy(1, 0, 0, 32)]
    for call in ({0: texts[0][33:], 1: texts[1][32:]},):
        model.extend(call, cache, buffers)
    logits = buffers.logits.download(np.float32, count=600).reshape(2, 300)
    for s in (0, 1):
        assert normwise_rel(logits[s], logits_of(ref, texts[s])) <= TOLERANCE["float16"]
        assert all(same_bits(a, b) for a, b in zip(held, cache.rows_numpy(1, s, 0, 32)))
    cache.release(0)
    assert cache.free_pages == 10 - 4
    model.extend({2: rng.integers(0, 300, 60).tolist()}, cache, buffers)
    model.extend({1: [5]}, cache, buffers)
    got = buffers.logits.download(np.float32, count=300)
    assert normwise_rel(got, logits_of(ref, texts[1] + [5])) <= TOLERANCE["float16"]
    cache.release(1)
    cache.release(2)
    assert cache.free_pages == 10


def test_refusals_of_calls(kt):
    model = small(kt)
    cache = model.new_paged_cache(2, 40, page_tokens=16)
    buffers = model.new_batch_buffers(cache, 8)
    other = kt.Transformer(300, 256, 2, 4, 192, 2, quantization=kt.Quantization(8, 32))
    E = kt.IllegalArgumentException
    for texts, message in (({}, "no sequence"), ({2: [1]}, "out of bounds"), ({0: []}, "empty"), ({0: [300]}, "vocab"), ({0: [1] * 41}, "full")):
        with pytest.raises(E, match=message):
            model.extend(texts, cache, buffers)
    with pytest.raises(E, match="Cache built"):
        other.extend({0: [1]}, cache, buffers)
    with pytest.raises(E, match="another cache"):
        model.extend({0: [1]}, model.new_paged_cache(3, 40), buffers)
    with pytest.raises(E, match="another model"):
        model.extend({0: [1]}, cache, other.new_batch_buffers(cache))
    for tokens, steps, message in (([1], 1, "1 tokens"), ([1, 2], -1, "negative"), ([1, 2], 41, "full"), ([1, 999], 1, "vocab")):
        with pytest.raises(E, match=message):
            model.greedy_decode_batch(tokens, cache, buffers, steps)
    assert model.greedy_decode_batch([1, 2], cache, buffers, 0) == [[], []]
    for draft, message in ((([1, 2], [-1]), "no tree"), (([1, 2], [-1, 1]), "no tree"), (([1], [0]), "no tree"), (([1, 2], [-1, -1]), "no tree"),
                           (([1] * 9, [-1] + [0] * 8), "rows"), (([], []), "empty")):
        with pytest.raises(E, match=message):
            model.draft_step({0: draft}, cache, buffers)
    assert cache.lengths == [0, 0] and cache.free_pages == cache.pages
    with pytest.raises(E, match="empty"):
        model.generate_batch([[1], []], 3)
    assert model.generate_batch([[1], [2]], 0) == [[1], [2]]
