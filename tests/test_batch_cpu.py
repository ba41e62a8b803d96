"""PagedKVCache's pages and TextDraft's trees without a device."""
import numpy as np
import pytest

import kotensor_amd as kt
from kotensor_amd import paged


class HostBuffer:
    """DeviceBuffer's calls on host memory."""

    def __init__(self, nbytes):
        self.nbytes, self.ptr = nbytes, 4096
        self.bytes = np.zeros(nbytes, np.uint8)

    @classmethod
    def from_numpy(cls, array, stream=None):
        buffer = cls(array.nbytes)
        buffer.upload(array)
        return buffer

    def upload(self, array, stream=None, offset=0):
        raw = np.ascontiguousarray(array).view(np.uint8).reshape(-1)
        assert offset + raw.size <= self.nbytes
        self.bytes[offset:offset + raw.size] = raw


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(paged, "DeviceBuffer", HostBuffer)
    return kt.PagedKVCache(2, 2, 4, 100, 32, "float16", 16, pages=12)


def tables(cache):
    return cache.tables.bytes.view(np.int32).reshape(cache.sequences, cache.table_stride)


def lengths(cache):
    return cache.device_lengths.bytes.view(np.int32).tolist()


def grow(cache, counts):
    cache.reserve(counts)
    for s, n in counts.items():
        cache.lengths[s] += n


def test_pages_go_to_sequences_and_back(cache):
    assert cache.size_in_bytes == 2 * 2 * 2 * 12 * 2 * 16 * 32 and cache.table_stride == 7
    grow(cache, {0: 1, 1: 16, 2: 17})
    assert cache.free_pages == 8
    grow(cache, {0: 15, 1: 1})
    assert cache.free_pages == 7
    held = [row[row >= 0].tolist() for row in tables(cache)]
    assert [len(h) for h in held] == [1, 2, 2, 0] and len({p for h in held for p in h}) == 5
    cache.release(1)
    assert cache.free_pages == 9 and cache.lengths[1] == 0 and lengths(cache)[1] == 0
    grow(cache, {3: 100})
    assert cache.free_pages == 2
    mine = tables(cache)[3].tolist()
    assert len(set(mine)) == 7 and not set(mine) & set(held[0] + held[2])


def test_a_reservation_is_whole_or_none(cache):
    grow(cache, {0: 90})
    with pytest.raises(kt.IllegalArgumentException, match="8 pages needed, 6 of 12 free"):
        cache.reserve({1: 64, 2: 64})
    with pytest.raises(kt.IllegalArgumentException, match="exceed maxSequenceLength 100"):
        cache.reserve({1: 1, 0: 11})
    assert cache.free_pages == 6
    cache.reserve({1: 64, 2: 32, 0: 0})
    assert cache.free_pages == 0


def test_shared_pages_are_freed_by_the_last_holder(cache):
    grow(cache, {0: 50})
    assert cache.share(0, 1, 50) == 48 and cache.share(1, 2, 40) == 32
    assert cache.free_pages == 8 and lengths(cache) == [0, 48, 32, 0]
    assert tables(cache)[1, :3].tolist() == tables(cache)[0, :3].tolist()
    grow(cache, {1: 1, 2: 1})
    assert cache.free_pages == 6 and tables(cache)[1, 3] != tables(cache)[0, 3]
    for keep, fine in ((50, True), (48, True), (47, False), (0, False)):
        if fine:
            cache.set_length(0, keep)
        else:
            with pytest.raises(kt.IllegalArgumentException, match="shared"):
                cache.set_length(0, keep)
    cache.release(0)
    assert cache.free_pages == 7  # its own last page
    cache.release(2)
    assert cache.free_pages == 8
    cache.set_length(1, 0)
    cache.release(1)
    assert cache.free_pages == 12 and sorted(cache._free) == list(range(12))


def test_refusals(cache):
    E = kt.IllegalArgumentException
    for change in ({"num_layers": 0}, {"num_heads": 0}, {"sequences": 0}, {"max_sequence_length": 0}, {"head_dim": 0}, {"page_tokens": 0},
                   {"format": "int8"}, {"head_dim": 48}, {"page_tokens": 24}, {"pages": -1}):
        with pytest.raises(E):
            kt.PagedKVCache(**{**dict(num_layers=1, num_heads=1, sequences=1, max_sequence_length=10, head_dim=32), **change})
    for call in (lambda: cache.reserve({4: 1}), lambda: cache.reserve({-1: 1}), lambda: cache.reserve({0: -1}), lambda: cache.release(4),
                 lambda: cache.set_length(0, 1), lambda: cache.set_length(0, -1), lambda: cache.share(0, 4, 0), lambda: cache.share(0, 1, 1),
                 lambda: kt.TextDraft(0), lambda: kt.TextDraft(1, 0), lambda: kt.TextDraft(1, 1, 0)):
        with pytest.raises(E):
            call()
    with pytest.raises(E):
        kt.BatchBuffers(8, 8, 8, 4, 10, 3, 8)


def test_drafts_from_the_text():
    draft = kt.TextDraft(tokens=3, branches=2, match=2)
    assert draft([1]) == ([], []) and draft([]) == ([], [])
    assert draft([1, 2, 3]) == ([], [])
    # the last two tokens occur twice before: the later place first; both go on with 9
    text = [5, 6, 9, 1, 2, 5, 6, 9, 4, 5, 6]
    tokens, parents = draft(text)
    assert tokens == [9, 4, 5, 1, 2] and parents == [-1, 0, 1, 0, 3]
    # only the last one occurs
    assert draft([7, 8, 3, 8]) == ([3, 8], [-1, 0])
    assert kt.TextDraft(4, 1, 3)([1, 1, 1]) == ([1], [-1])
    for run in range(50):
        rng = np.random.default_rng(run)
        text = rng.integers(0, 4, 40).tolist()
        tokens, parents = kt.TextDraft(5, 3, 3)(text)
        assert len(tokens) == len(parents) <= 15 and all(-1 <= p < i for i, p in enumerate(parents))


def test_argmax_of_rows_refused():
    from kotensor_amd import _lib
    lib = _lib.lib()
    call = lambda logits=16, rows=2, n=5, tokens=16, positions=16, generated=16, capacity=4: lib.kt_argmax_rows(
        logits, rows, n, tokens, positions, generated, capacity, None)
    for change, want, message in (({"logits": None}, _lib.KT_ERR_ARGUMENT, "NULL"), ({"tokens": None}, _lib.KT_ERR_ARGUMENT, "NULL"),
                                  ({"rows": -1}, _lib.KT_ERR_SHAPE, "argmax of -1 rows"), ({"rows": 15873}, _lib.KT_ERR_SHAPE, "0 to 15872"),
                                  ({"n": 0}, _lib.KT_ERR_SHAPE, "at least one logit"), ({"positions": None}, _lib.KT_ERR_ARGUMENT, "without positions"),
                                  ({"capacity": -1}, _lib.KT_ERR_SHAPE, "negative capacity")):
        assert call(**change) == want and message in _lib.last_error(), (change, _lib.last_error())
    assert call(rows=0, logits=None) == _lib.KT_OK


class Rows:
    """Of BatchBuffers what a batch of trees takes."""

    def __init__(self, rows):
        self.rows, self.depths, self.masks = rows, HostBuffer(4 * rows), HostBuffer(4 * rows * -(-rows // 32))


def test_batches_of_rows(cache):
    grow(cache, {0: 20, 2: 5})
    cache.reserve({0: 12, 1: 3, 2: 1})
    starts = HostBuffer(4 * 5)
    batch = kt.PagedBatch(cache, [12, 3, 0, 0], starts)
    assert starts.bytes.view(np.int32).tolist() == [0, 12, 15, 15, 15]
    assert (batch.batch.sequences, batch.batch.rows, batch.batch.most_rows, batch.batch.key_bound) == (4, 15, 12, 32)
    nothing = kt.PagedBatch(cache, [0] * 4, starts).batch
    assert (nothing.rows, nothing.most_rows, nothing.key_bound) == (0, 0, 0)
    tree = kt.PagedBatch(cache, [8, 3, 0, 0], starts, buffers=Rows(11)).batch
    assert tree.mask_words == 1 and tree.masks == tree.depths == 4096
    assert kt.PagedBatch(cache, np.array([1, 1, 1, 0]), starts, key_bound=100).batch.key_bound == 100


def test_batches_of_rows_refused(cache):
    grow(cache, {0: 20, 2: 5})
    cache.reserve({0: 12, 1: 3, 2: 1})
    starts = HostBuffer(4 * 5)
    for counts, change, message in (([1, 1, 1], {}, "3 counts for 4 sequences"), ([1] * 5, {}, "5 counts for 4 sequences"), ([], {}, "0 counts"),
                                    ([4, -1, 0, 0], {}, "must not be negative"), ([13, 0, 0, 0], {}, "no pages"), ([0, 0, 0, 1], {}, "no pages"), ([0, 17, 0, 0], {}, "no pages"),
                                    ([1, 1, 0, 0], {"key_bound": 20}, "key bound 20"), ([8, 3, 1, 0], {"buffers": Rows(11)}, "12 tokens exceed the buffers' 11 rows")):
        with pytest.raises(kt.IllegalArgumentException, match=message):
            kt.PagedBatch(cache, counts, starts, **change)
    assert not starts.bytes.any()


class Memory(HostBuffer):
    """Device memory by address, so that calls can find it."""
    at: dict = {}

    def __init__(self, nbytes):
        super().__init__(nbytes)
        self.ptr = 4096 * (len(Memory.at) + 1)
        Memory.at[self.ptr] = self

    def download(self, dtype, count=None, stream=None, offset=0):
        return self.bytes.view(dtype)[:count].copy()


@pytest.fixture
def decoder(monkeypatch):
    """(model, cache, buffers, calls): a decoder whose kernels do nothing but the lengths' advance; calls names what is to raise, and when."""
    from kotensor_amd import _lib, transformer
    for module in (paged, transformer):
        monkeypatch.setattr(module, "DeviceBuffer", Memory)
    monkeypatch.setattr(Memory, "at", {})
    model = object.__new__(kt.Transformer)
    model.num_layers, model.num_key_value_heads, model.head_dim, model.vocabulary_size = 2, 2, 32, 50
    model.dimension, model.hidden_dimension, model.kv_dimension = 64, 96, 64
    calls = {"made": [], "raise": None}
    plain = _lib.call

    def call(name, *args):
        if name == "kt_paged_layout":
            return plain(name, *args)
        calls["made"].append(name)
        if calls["raise"] and calls["raise"][0] == name and calls["made"].count(name) == calls["raise"][1]:
            raise kt.IllegalStateException("planted")
        if name == "kt_paged_advance":
            lengths = Memory.at[args[0]].bytes.view(np.int32)
            starts = Memory.at[args[1]._obj.starts].bytes.view(np.int32)
            lengths += starts[1:] - starts[:-1]

    monkeypatch.setattr(_lib, "call", call)
    for name in ("_embed", "_layers", "_head"):
        monkeypatch.setattr(kt.Transformer, name, lambda self, *args, name=name: call(name))
    cache = model.new_paged_cache(3, 60, "float16", 16)
    buffers = model.new_batch_buffers(cache, 8)
    return model, cache, buffers, calls


def test_a_call_that_fails_leaves_the_lengths_as_they_were(decoder):
    """Device and host agree after an error, whichever step of the call it comes from, and the next call goes on from there."""
    model, cache, buffers, calls = decoder

    def fails(at, call):
        before = list(cache.lengths)
        calls["made"], calls["raise"] = [], at
        with pytest.raises(kt.IllegalStateException, match="planted"):
            call()
        calls["raise"] = None
        assert cache.lengths == before == lengths(cache)

    assert set(model.extend({0: [1] * 5, 2: [2] * 9}, cache, buffers)) == {0, 2}
    assert cache.lengths == lengths(cache) == [5, 0, 9]
    texts = {0: [1] * 20, 1: [3] * 3}  # (three parts of eight rows)
    for at in (("_layers", 1), ("_layers", 3), ("kt_paged_advance", 2), ("kt_memcpy_d2d", 1), ("_head", 1), ("kt_argmax_rows", 1)):
        fails(at, lambda: model.extend(texts, cache, buffers))
    for at in (("_layers", 1), ("_layers", 3), ("_head", 2), ("kt_argmax_rows", 4), ("kt_paged_advance", 3)):
        fails(at, lambda: model.greedy_decode_batch([1, 2, 3], cache, buffers, 5, use_graph=False))
    drafts = {0: ([4, 5, 6], [-1, 0, 0])}
    for at in (("_layers", 1), ("kt_tree_accept", 1), ("kt_paged_keep", 1)):
        fails(at, lambda: model.draft_step(drafts, cache, buffers))
    model.extend(texts, cache, buffers)
    assert cache.lengths == lengths(cache) == [25, 3, 9]
    assert len(model.greedy_decode_batch([1, 2, 3], cache, buffers, 4, use_graph=False)) == 3
    assert cache.lengths == lengths(cache) == [29, 7, 13]


def test_a_recorded_replay_that_fails_leaves_the_lengths_as_they_were(decoder, monkeypatch):
    model, cache, buffers, calls = decoder
    from kotensor_amd import transformer

    class Stream:
        handle = 7

        def synchronize(self):
            calls["made"].append("synchronize")

    def record(st, step):  # (nothing of a recording runs)
        return "graph"

    monkeypatch.setattr(kt.Transformer, "_record", staticmethod(record))
    for at in (("kt_graph_launch", 1), ("kt_graph_launch", 3)):
        calls["made"], calls["raise"] = [], at
        with pytest.raises(kt.IllegalStateException, match="planted"):
            model.greedy_decode_batch([1, 2, 3], cache, buffers, 6, Stream())
        assert calls["made"].count("kt_graph_destroy") == 1 and "synchronize" in calls["made"]
        assert cache.lengths == lengths(cache) == [0, 0, 0]


def test_more_rows_than_an_argmax_takes(decoder, monkeypatch):
    model, cache, buffers, calls = decoder
    from kotensor_amd import _lib
    E = kt.IllegalArgumentException
    assert _lib.lib().kt_argmax_rows(16, _lib.KT_ARGMAX_MOST_ROWS + 1, 5, 16, None, None, 0, None) == _lib.KT_ERR_SHAPE
    with pytest.raises(E, match="at most 15872"):
        kt.BatchBuffers(8, 8, 8, 15873, 10, 15873, 8)
    kt.BatchBuffers(1, 1, 1, 1, 40000, 20000, 1)  # (parts of prompts may be larger)
    buffers.rows = 20000
    calls["made"] = []
    with pytest.raises(E, match="at most 15872"):
        model.draft_step({0: ([1] * 15873, [-1] + [0] * 15872)}, cache, buffers)
    assert not calls["made"] and not cache._held[0]
