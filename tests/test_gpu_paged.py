"""The cache in pages and trees of drafted tokens on the device, against the oracle in 64 bits."""
import ctypes

import numpy as np
import pytest

from gpu_helpers import banner
from oracle import paged_ref
from paged_helpers import Batch, random_parents

pytestmark = pytest.mark.gpu

FORMATS = ["float32", "float16", "bfloat16"]
SHAPES = [(8, 2, 64), (14, 2, 64), (6, 6, 32), (4, 2, 128), (4, 1, 256), (20, 1, 64), (3, 1, 32), (40, 2, 128)]
STEPS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 700]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_append_rotates_and_stores(kt, fmt, shape):
    b = Batch(kt, 1, [0, 5, 16, 100, 31], [1, 40, 0, 3, 17], shape, fmt, 16, layers=2, extra=3, lead=2)
    b.rope(1)
    b.append(1)
    b.check_pool()
    got, want = b.context(), b.rotated()
    inside = slice(int(b.starts[0]), int(b.starts[-1]))
    # fp32 steps on cosines and sines that are double-precision results rounded: one unit of either, of |x1| + |x2|
    assert np.abs(got[inside] - want[inside]).max() <= 2.0 ** -23 * 2 * np.abs(b.q).max() * 2
    assert np.isnan(got[:2]).all() and np.isnan(got[-3:]).all()


def test_append_in_place_and_alone(kt):
    b = Batch(kt, 2, [3, 64], [2, 5], (8, 2, 64), "float32", 32)
    b.rope(q=False)
    b.append()
    b.check_pool()
    assert np.isnan(b.context()).all()
    b.d["context"].upload(b.q)
    at = ctypes.byref
    b.lib.call("kt_rope_paged", b.d["context"].ptr, b.d["k"].ptr, b.d["v"].ptr, b.heads, b.d["inv_freq"].ptr, at(b.cache), 0, at(b.batch), b.d["context"].ptr, None)
    assert np.abs(b.context() - b.rotated()).max() <= 2.0 ** -20


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("fmt", FORMATS)
def test_append_by_depth(kt, fmt, page):
    rng = np.random.default_rng(3)
    counts = [1, 7, 64, 0, 33]
    b = Batch(kt, 3, [0, 250, 255, 9, 1000], counts, (4, 2, 64), fmt, page, parents=random_parents(rng, counts))
    b.rope()
    b.append()
    b.check_pool()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_steps(kt, fmt, shape):
    b = Batch(kt, 4, STEPS, [1] * len(STEPS), shape, fmt, 16)
    b.rope_attention()
    b.append()
    b.check_pool()
    b.check_context(b.context(), *b.attend(b.rotated()))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("fmt", FORMATS)
def test_pages(kt, fmt, page):
    b = Batch(kt, 5, [0, 255, 256, 257, 600, 15], [1] * 6, (8, 2, 64), fmt, page)
    b.rope_attention()
    b.append()
    b.check_pool()
    b.check_context(b.context(), *b.attend(b.rotated()))


@pytest.mark.parametrize("fmt,shape,length", [("float32", (8, 2, 64), 9000), ("float16", (8, 1, 128), 6001), ("bfloat16", (4, 4, 64), 12345), ("bfloat16", (4, 1, 256), 3100),
                                              ("float32", (40, 2, 128), 2500)])
def test_a_long_sequence_beside_short_ones(kt, fmt, shape, length):
    lengths = [3, length, 0, 70, length // 3]
    b = Batch(kt, 6, lengths, [1, 1, 1, 1, 2], shape, fmt, 64)
    b.rope_attention()
    b.append()
    b.check_context(b.context(), *b.attend(b.rotated()))
    first = b.context().tobytes()
    for _ in range(3):  # the same bits each time
        b.rope_attention()
        assert b.context().tobytes() == first


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_prompts_and_parts(kt, fmt, shape):
    b = Batch(kt, 7, [0, 3, 64, 100, 31, 0], [70, 1, 0, 33, 2, 5], shape, fmt, 32, extra=2, lead=1)
    b.append()
    b.upload()
    b.attention()
    b.check_context(b.context(), *b.attend(b.q))


@pytest.mark.parametrize("fmt,shape,length,count", [("float32", (8, 2, 64), 0, 300), ("float16", (8, 2, 64), 200, 257), ("bfloat16", (4, 2, 128), 333, 150), ("float32", (2, 1, 256), 40, 90),
                                                    ("bfloat16", (6, 6, 32), 0, 200), ("float16", (4, 1, 128), 1500, 65)])
def test_prompts_of_many_tiles(kt, fmt, shape, length, count):
    b = Batch(kt, 8, [length], [count], shape, fmt, 16)
    b.rope_attention()
    b.append()
    b.check_pool()
    b.check_context(b.context(), *b.attend(b.rotated()))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_trees(kt, fmt, shape):
    rng = np.random.default_rng(9)
    counts = [1, 7, 33, 0, 64, 2]
    b = Batch(kt, 9, [0, 40, 31, 5, 100, 63], counts, shape, fmt, 16, parents=random_parents(rng, counts), extra=1)
    b.rope_attention()
    b.append()
    b.check_pool()
    b.check_context(b.context(), *b.attend(b.rotated()))


@pytest.mark.parametrize("fmt,length,count", [("float32", 1000, 130), ("bfloat16", 4000, 20), ("float16", 65, 200)])
def test_large_trees(kt, fmt, length, count):
    rng = np.random.default_rng(10)
    b = Batch(kt, 10, [length, 3], [count, 4], (8, 2, 64), fmt, 64, parents=random_parents(rng, [count, 4]))
    b.rope_attention()
    b.append()
    b.check_context(b.context(), *b.attend(b.rotated()))


def test_masks_and_depths(kt):
    rng = np.random.default_rng(11)
    counts = [1, 31, 0, 32, 33, 300]
    parents = random_parents(rng, counts)
    parents[1][5:9] = [-1, 5, 99, -3]  # further roots; no parent comes at or after its row
    parents[5][200:] = np.arange(199, 299)  # a chain
    b = Batch(kt, 11, [0] * 6, counts, (2, 1, 32), "float32", 16, parents=parents, extra=4)
    for words in (b.words, b.words + 3):
        b.batch.mask_words = words
        guard = np.full(b.rows * words + 8, 0xABABABAB, np.uint32)
        d, m = kt.DeviceBuffer.from_numpy(np.full(b.rows, 77, np.int32)), kt.DeviceBuffer.from_numpy(guard)
        b.lib.call("kt_tree_masks", b.d["parents"].ptr, ctypes.byref(b.batch), d.ptr, m.ptr, None)
        depths, bits = d.download(np.int32), m.download(np.uint32)
        for s in range(6):
            want = paged_ref.masks(parents[s], words)
            r = b.sequence_rows(s)
            assert np.array_equal(depths[r], want[0]) and np.array_equal(bits[:b.rows * words].reshape(b.rows, words)[r], want[1])
        end = int(b.starts[-1])
        assert (depths[end:] == 77).all() and (bits[end * words:] == 0xABABABAB).all()


@pytest.mark.parametrize("seed", range(6))
def test_accept_and_keep(kt, seed):
    rng = np.random.default_rng(20 + seed)
    fmt, shape, page = FORMATS[seed % 3], SHAPES[seed % 5], [16, 32, 256][seed % 3]
    counts = [1, 0, 9, 64, 200, 5, 70]
    parents = random_parents(rng, counts)
    if seed == 0:  # a chain that is taken whole
        parents[3] = np.arange(-1, 63, dtype=np.int32)
    b = Batch(kt, 20 + seed, [0, 4, 15, 100, 16, 31, 1], counts, shape, fmt, page, layers=3, parents=parents)
    flat = np.concatenate(parents)
    tokens, chosen = rng.integers(0, 3, (2, b.rows)).astype(np.int32)
    if seed == 0:
        tokens[:] = chosen[:] = 1
    for layer in range(3):
        b.rope(layer, q=False)
        b.append(layer)
    stride = b.most + 2
    up = kt.DeviceBuffer.from_numpy
    d = {"tokens": up(tokens), "chosen": up(chosen), "kept": up(np.full((7, stride), 55, np.int32)), "counts": up(np.full(7, 55, np.int32)), "next": up(np.full(7, 55, np.int32))}
    b.lib.call("kt_tree_accept", d["tokens"].ptr, d["chosen"].ptr, b.d["parents"].ptr, ctypes.byref(b.batch), d["kept"].ptr, stride, d["counts"].ptr, d["next"].ptr, None)
    kept, counted, following = d["kept"].download(np.int32).reshape(7, stride), d["counts"].download(np.int32), d["next"].download(np.int32)
    want = []
    for s in range(7):
        r = b.sequence_rows(s)
        path = paged_ref.accept(parents[s], tokens[r], chosen[r])
        want.append(b.lengths[s] + len(path))
        assert counted[s] == len(path) and kept[s].tolist() == path + [-1] * (stride - len(path))
        assert following[s] == (chosen[r][path[-1]] if path else 55)
        b.pool.keep(b.tables[s], b.lengths[s], path)
    assert len(flat) == b.rows
    apart = up(np.zeros(7, np.int32))
    new = b.d["lengths"] if seed % 2 else apart
    b.lib.call("kt_paged_keep", ctypes.byref(b.cache), ctypes.byref(b.batch), d["kept"].ptr, stride, d["counts"].ptr, new.ptr, None)
    b.check_pool()
    assert new.download(np.int32)[:7].tolist() == want


def test_keep_stops_at_rows_that_do_not_ascend(kt):
    b = Batch(kt, 30, [3, 3, 3, 3], [6] * 4, (2, 1, 32), "float32", 16, parents=[np.full(6, -1, np.int32)] * 4)
    b.rope(q=False)
    b.append()
    lists = [[1, 3, 5], [2, 2, 3], [0, 4, 6], [-1, 2, 3]]
    kept, counts = kt.DeviceBuffer.from_numpy(np.array(lists, np.int32)), kt.DeviceBuffer.from_numpy(np.array([9, 3, 3, 3], np.int32))
    b.lib.call("kt_paged_keep", ctypes.byref(b.cache), ctypes.byref(b.batch), kept.ptr, 3, counts.ptr, b.d["lengths"].ptr, None)
    for s, fine in enumerate(([1, 3, 5], [2], [0, 4], [])):
        b.pool.keep(b.tables[s], 3, fine)
    b.check_pool()
    assert b.d["lengths"].download(np.int32)[:4].tolist() == [6, 4, 5, 3]


def test_advance(kt):
    b = Batch(kt, 31, [0, 5, 100], [1, 0, 7], (2, 1, 32))
    b.lib.call("kt_paged_advance", b.d["lengths"].ptr, ctypes.byref(b.batch), None)
    assert b.d["lengths"].download(np.int32)[:3].tolist() == [1, 5, 107]


@pytest.mark.parametrize("fmt", FORMATS)
def test_read(kt, fmt):
    b = Batch(kt, 32, [50, 7], [1, 1], (4, 2, 64), fmt, 16, layers=2)
    for s, first, count in ((0, 0, 50), (0, 17, 20), (1, 6, 1)):
        out = [kt.DeviceBuffer(4 * 2 * count * 64) for _ in range(2)]
        b.lib.call("kt_paged_read", ctypes.byref(b.cache), 1, b.d["tables"].ptr + 4 * s * b.stride, b.stride, first, count, out[0].ptr, out[1].ptr, None)
        for which, got in zip(("keys", "values"), out):
            want = b.pool.rows(which, 1, b.tables[s], range(first, first + count))
            assert got.download(np.float32).tobytes() == want.tobytes()
    out = kt.DeviceBuffer(4 * 2 * 3 * 64)  # a page outside the pool
    b.lib.call("kt_paged_read", ctypes.byref(b.cache), 0, b.d["tables"].ptr + 4 * b.stride, b.stride, 31, 3, None, out.ptr, None)
    assert np.isnan(out.download(np.float32)).all()


# ---- where it can go wrong -----------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tree", [False, True])
def test_pages_outside_the_pool_hold_nothing(kt, fmt, tree):
    counts = [20, 5, 1, 1]
    parents = random_parents(np.random.default_rng(40), counts) if tree else None
    b = Batch(kt, 40, [100, 30, 200, 40], counts, (8, 2, 64), fmt, 16, parents=parents)
    b.tables[0, 2], b.tables[0, 6], b.tables[1, 1], b.tables[2, :] = -1, b.pool.pages, 2 ** 31 - 1, -2 ** 31
    b.upload()
    b.rope_attention()
    b.append()
    b.check_pool()
    want, bound = b.attend(b.rotated())
    b.check_context(b.context(), want, bound)
    assert not want[b.sequence_rows(2)].any() and not b.context()[b.sequence_rows(2)].any()


@pytest.mark.parametrize("tree", [False, True])
def test_lengths_below_zero_and_past_the_table(kt, tree):
    counts = [4, 3, 2]
    parents = random_parents(np.random.default_rng(41), counts) if tree else None
    b = Batch(kt, 41, [-2, -40, 30], counts, (4, 2, 64), "float32", 16, parents=parents)
    b.upload()
    b.rope_attention()
    b.append()
    b.check_pool()
    b.check_context(b.context(), *b.attend(b.rotated()))
    for length in (2 ** 31 - 2, -2 ** 31):
        b.lengths = [length] * 3
        b.d["lengths"].upload(np.array(b.lengths, np.int32))
        b.rope(q=False)
        b.check_pool()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("tree", [False, True])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(kt, fmt, bad, tree):
    counts = [40, 6]
    parents = random_parents(np.random.default_rng(42), counts) if tree else None
    b = Batch(kt, 42, [35, 3], counts, (8, 2, 64), fmt, 16, parents=parents)
    b.v[0, 25, 1, 7] = bad
    b.k[0, 30] = np.nan
    b.upload()
    b.rope_attention()
    b.append()
    got, clean = b.context(), b.visible(0)
    b.v[0, 25, 1, 7] = 0.0
    b.k[0, 30] = 0.0
    b.append()
    want, bound = b.attend(b.rotated())
    for i in range(40):
        if clean[i, 35 + 30]:  # a key that is not a number
            assert np.isnan(got[i]).all()
            want[i] = got[i] = 0
        elif clean[i, 35 + 25]:
            assert not np.isfinite(got[i, 4:, 7]).any()
            want[i, 4:, 7] = got[i, 4:, 7] = 0
    b.check_context(got, want, bound)


def test_large_scores(kt):
    for loud in (20.0, 300.0):
        for fmt in FORMATS:
            b = Batch(kt, 43, [90, 700], [3, 40], (8, 2, 64), fmt, 32, loud=loud)
            b.rope_attention()
            b.append()
            b.check_context(b.context(), *b.attend(b.rotated()))


@pytest.mark.parametrize("fmt", FORMATS)
def test_quiet_and_loud_queries(kt, fmt):
    b = Batch(kt, 44, [90, 300], [3, 20], (8, 2, 64), fmt, 32)
    b.q *= np.exp2(np.random.default_rng(44).integers(-60, 3, b.q.shape[:2] + (1,))).astype(np.float32)
    b.q[1] = 0
    b.append()
    b.upload()
    b.attention()
    b.check_context(b.context(), *b.attend(b.q))


@pytest.mark.parametrize("tree", [False, True])
def test_key_bound(kt, tree):
    counts = [30, 1]
    parents = random_parents(np.random.default_rng(45), counts) if tree else None
    b = Batch(kt, 45, [100, 400], counts, (4, 2, 64), "bfloat16", 32, parents=parents, key_bound=117)
    b.append()
    b.upload()
    b.attention()
    b.check_context(b.context(), *b.attend(b.q))


def test_two_sequences_share_pages(kt):
    b = Batch(kt, 46, [64, 64], [1, 1], (4, 2, 64), "float32", 32)
    b.tables[1, :2] = b.tables[0, :2]
    b.upload()
    b.rope_attention()
    b.append()
    b.check_pool()
    b.check_context(b.context(), *b.attend(b.rotated()))


def test_many_sequences(kt):
    rng = np.random.default_rng(47)
    lengths, counts = rng.integers(0, 60, 300).tolist(), rng.integers(0, 3, 300).tolist()
    b = Batch(kt, 47, lengths, counts, (4, 2, 64), "float16", 16)
    b.rope_attention()
    b.append()
    b.check_pool()
    b.check_context(b.context(), *b.attend(b.rotated()))


@pytest.mark.parametrize("tree", [False, True])
def test_a_recorded_step_follows_its_arrays(kt, tree):
    stream = kt.Stream.create()
    counts = [3, 5, 2] if tree else [1, 1, 1]
    parents = random_parents(np.random.default_rng(48), counts) if tree else None
    b = Batch(kt, 48, [40, 1000, 0], counts, (8, 2, 64), "bfloat16", 16, parents=parents)
    b.rope_attention(stream=stream.handle)  # sizes the workspace
    stream.synchronize()
    graph = ctypes.c_void_p()
    b.lib.call("kt_graph_begin", stream.handle)
    if tree:
        b.masks(stream.handle)
    b.rope_attention(stream=stream.handle)
    b.lib.call("kt_graph_end", stream.handle, ctypes.byref(graph))
    rng = np.random.default_rng(49)
    for lengths in ([40, 1000, 0], [17, 3, 0], [0, 999, 0], [40, 64, 0]):
        b.lengths = lengths
        b.d["lengths"].upload(np.array(lengths, np.int32), stream)
        if tree:
            b.parents = random_parents(rng, counts)
            b.d["parents"].upload(np.concatenate(b.parents), stream)
        b.q = rng.standard_normal(b.q.shape).astype(np.float32)
        b.d["q"].upload(b.q, stream)
        b.append()
        b.lib.call("kt_graph_launch", graph, stream.handle)
        replayed = b.context(stream)
        b.check_context(replayed, *b.attend(b.rotated()))
        if tree:
            b.masks(stream.handle)
        b.rope_attention(stream=stream.handle)
        assert b.context(stream).tobytes() == replayed.tobytes()
    b.check_pool()
    b.lib.call("kt_graph_destroy", graph)
    stream.destroy()


def test_two_streams_at_once(kt):
    streams = [kt.Stream.create() for _ in range(2)]
    batches = [Batch(kt, 50 + i, [3000, 10], [1, 30], (8, 2, 64), "float32", 32) for i in range(2)]
    want = []
    for b in batches:
        b.rope_attention()
        want.append(b.context().tobytes())
    for b, s in zip(batches, streams):
        b.rope_attention(stream=s.handle)
        s.synchronize()
    for _ in range(5):
        for b in batches:
            b.d["context"].fill_zero()
        kt.synchronize()
        for b, s in zip(batches, streams):
            b.rope_attention(stream=s.handle)
        for b, s, w in zip(batches, streams, want):
            assert b.context(s).tobytes() == w
    for s in streams:
        s.destroy()


def test_offsets_past_32_bits(kt):
    """A pool whose last pages lie past 2^31 elements (and 2^32 bytes) of a layer."""
    from kotensor_amd import _lib
    banner("paged offsets past 32 bits")
    pages, kv, page, d = 9000, 8, 256, 128  # 2.36e9 elements, 4.7 GB in bf16
    c = _lib.PagedCache()
    c.format, c.layers, c.pages, c.kv_heads, c.page_tokens, c.head_dim = _lib.KT_PAGED_BF16, 1, pages, kv, page, d
    size = ctypes.c_int64()
    _lib.call("kt_paged_layout", ctypes.byref(c), ctypes.byref(size))
    assert size.value == 2 * pages * kv * page * d
    keys, values = kt.DeviceBuffer(size.value), kt.DeviceBuffer(size.value)
    c.keys, c.values = keys.ptr, values.ptr
    b = Batch(kt, 51, [0, 0], [40, 3], (8, 8, 128), "bfloat16", 256)
    b.pool.pages = pages
    b.tables[:, 0] = [pages - 1, pages - 2]
    b.d["tables"].upload(b.tables)
    b.cache = c
    b.rope_attention()
    got = b.context()
    small = Batch(kt, 51, [0, 0], [40, 3], (8, 8, 128), "bfloat16", 256)
    small.rope_attention()
    assert small.context().tobytes() == got.tobytes()
    for s in range(2):
        out = [kt.DeviceBuffer(4 * kv * 3 * d) for _ in range(4)]
        _lib.call("kt_paged_read", ctypes.byref(c), 0, b.d["tables"].ptr + 4 * s * b.stride, b.stride, 0, 3, out[0].ptr, out[1].ptr, None)
        _lib.call("kt_paged_read", ctypes.byref(small.cache), 0, small.d["tables"].ptr + 4 * s * b.stride, b.stride, 0, 3, out[2].ptr, out[3].ptr, None)
        assert out[0].download(np.float32).tobytes() == out[2].download(np.float32).tobytes()
        assert out[1].download(np.float32).tobytes() == out[3].download(np.float32).tobytes()


@pytest.mark.parametrize("tree", [False, True])
def test_rows_of_no_sequence_alone(kt, tree):
    """A padded batch whose sequences are all empty, eager and recorded: the pool and the context stay as they are."""
    counts = [0, 0, 0]
    b = Batch(kt, 52, [40, 0, 7], counts, (8, 2, 64), "float16", 16, parents=random_parents(np.random.default_rng(52), counts) if tree else None, extra=5, lead=2)
    stream, graph = kt.Stream.create(), ctypes.c_void_p()

    def calls():
        b.rope(stream=stream.handle)
        b.attention(stream=stream.handle)
        b.rope_attention(stream=stream.handle)
        b.lib.call("kt_paged_advance", b.d["lengths"].ptr, ctypes.byref(b.batch), stream.handle)

    calls()
    b.lib.call("kt_graph_begin", stream.handle)
    calls()
    b.lib.call("kt_graph_end", stream.handle, ctypes.byref(graph))
    for _ in range(3):
        b.lib.call("kt_graph_launch", graph, stream.handle)
        assert np.isnan(b.context(stream)).all()
        assert b.d["lengths"].download(np.int32)[:3].tolist() == [40, 0, 7]
        b.check_pool()
    b.lib.call("kt_graph_destroy", graph)
    stream.destroy()


@pytest.mark.parametrize("n", [4096, 4097])
def test_masks_of_large_trees(kt, n):
    """Trees whose parents fit LDS whole and one that does not: a chain, a star and a random one, beside a small tree."""
    rng = np.random.default_rng(53)
    chain = np.arange(-1, n - 1, dtype=np.int32)
    star = np.where(np.arange(n) == 0, -1, 0).astype(np.int32)
    for large in (chain, star, *random_parents(rng, [n])):
        parents = [np.array([-1, 0, 0], np.int32), large]
        b = Batch(kt, 53, [0, 0], [3, n], (2, 1, 32), "float16", 256, extra=1)
        d = {"parents": kt.DeviceBuffer.from_numpy(np.concatenate(parents + [np.array([-1], np.int32)])), "depths": kt.DeviceBuffer.from_numpy(np.full(b.rows, 77, np.int32)),
             "masks": kt.DeviceBuffer.from_numpy(np.full(b.rows * b.words, 0xABABABAB, np.uint32))}
        b.batch.depths, b.batch.masks = d["depths"].ptr, d["masks"].ptr
        b.lib.call("kt_tree_masks", d["parents"].ptr, ctypes.byref(b.batch), d["depths"].ptr, d["masks"].ptr, None)
        depths, bits = d["depths"].download(np.int32), d["masks"].download(np.uint32).reshape(b.rows, b.words)
        for s in range(2):  # each row's mask is its parent's and itself
            r = b.sequence_rows(s)
            want = np.zeros((len(parents[s]), b.words), np.uint32)
            deep = np.zeros(len(parents[s]), np.int32)
            for i, p in enumerate(parents[s]):
                if p >= 0:
                    want[i], deep[i] = want[p], deep[p] + 1
                want[i, i // 32] |= np.uint32(1 << (i % 32))
            assert np.array_equal(depths[r], deep) and np.array_equal(bits[r], want)
        assert depths[-1] == 77 and (bits[-1] == 0xABABABAB).all()


@pytest.mark.parametrize("n", [1024, 1025])
def test_accept_of_large_trees(kt, n):
    """Trees whose numbers fit LDS whole and one that does not: a chain that is kept whole, one that breaks at its last row, the last of many children, and a
    random tree, beside a small one."""
    rng = np.random.default_rng(54)
    chain, counting = np.arange(-1, n - 1, dtype=np.int32), np.arange(n, dtype=np.int32)
    star = np.where(np.arange(n) == 0, -1, 0).astype(np.int32)
    any_tree, few = random_parents(rng, [n])[0], rng.integers(0, 2, (2, n)).astype(np.int32)
    broken = counting.copy()
    broken[-1] = -5
    for large, tokens, chosen in ((chain, counting, counting + 1), (chain, broken, counting + 1), (star, counting, np.full(n, n - 1, np.int32)), (any_tree, few[0], few[1])):
        parents = [np.array([-1, 0, 0], np.int32), large]
        b = Batch(kt, 54, [0, 0], [3, n], (2, 1, 32), "float16", 256)
        tokens, chosen = [np.array([4, 5, 6], np.int32), tokens], [np.array([6, 0, 9], np.int32), chosen]
        up = lambda arrays: kt.DeviceBuffer.from_numpy(np.concatenate(arrays).astype(np.int32))
        d = {"parents": up(parents), "tokens": up(tokens), "chosen": up(chosen), "kept": up([np.full(2 * (n + 3), 55)]), "counts": up([np.full(2, 55)]), "next": up([np.full(2, 55)])}
        b.lib.call("kt_tree_accept", d["tokens"].ptr, d["chosen"].ptr, d["parents"].ptr, ctypes.byref(b.batch), d["kept"].ptr, n + 3, d["counts"].ptr, d["next"].ptr, None)
        kept, counts, following = d["kept"].download(np.int32).reshape(2, n + 3), d["counts"].download(np.int32), d["next"].download(np.int32)
        for s in range(2):
            path = paged_ref.accept(parents[s], tokens[s], chosen[s])
            assert counts[s] == len(path) and kept[s].tolist() == path + [-1] * (n + 3 - len(path)) and following[s] == chosen[s][path[-1]]
        if large is chain:
            assert counts[1] == (n if tokens[1][-1] != -5 else n - 1)
