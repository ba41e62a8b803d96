"""Attention over the cache in pages at the sizes that choose between its kernels (by rows of a kv head, key bound, head
dimension and format), and between its ways of cutting tiles into parts."""
import ctypes

import numpy as np
import pytest

from paged_helpers import Batch, random_parents

pytestmark = pytest.mark.gpu

FORMATS = ["float32", "float16", "bfloat16"]


def check(b):
    b.rope_attention()
    first = b.context()
    b.append()
    b.check_context(first, *b.attend(b.rotated()))
    b.rope_attention()
    assert b.context().tobytes() == first.tobytes()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("bound", [128, 129])
@pytest.mark.parametrize("tree", [False, True])
def test_few_keys(kt, fmt, dim, bound, tree):
    """Up to 128 keys a launch has tiles of 16 rows without parts; one more and it may have larger ones."""
    counts = [bound - 1, 1, 0, 40, 17]
    parents = random_parents(np.random.default_rng(dim), counts) if tree else None
    check(Batch(kt, 60, [1, 100, 5, 60, 0], counts, (4, 2, dim), fmt, 16, parents=parents, key_bound=bound, extra=1))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("rows", [16, 17, 64, 65, 128, 129])
def test_rows_of_a_tile(kt, fmt, dim, rows):
    """One query head a kv head: as many rows as tokens. Parts of a long text, beside a short one."""
    check(Batch(kt, 61 + rows, [1500, 200], [rows, 3], (2, 2, dim), fmt, 64))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [3, 5, 16, 17])
def test_rows_that_tiles_cut(kt, fmt, dim, group):
    """Tiles that end inside a token's query heads."""
    rng = np.random.default_rng(group)
    counts = [13, 6]
    check(Batch(kt, 62, [900, 31], counts, (group, 1, dim), fmt, 32, parents=random_parents(rng, counts)))


@pytest.mark.parametrize("fmt", ["float32", "bfloat16"])
def test_long_parts_of_few_tiles(kt, fmt):
    """More than LONG keys a workgroup: 64 or 128 tiles (fewer than 512) of 6500 tokens and more are cut finer."""
    check(Batch(kt, 63, [6900, 6500, 7100, 6000], [40, 33, 38, 40], (32, 8, 128), fmt, 64))


@pytest.mark.parametrize("fmt,shape,count", [("float16", (32, 8, 64), 1030), ("bfloat16", (32, 8, 64), 1024), ("float32", (32, 8, 64), 1024), ("bfloat16", (32, 8, 128), 1100)])
@pytest.mark.parametrize("given", [None, 50])
def test_one_sequence_that_fills_the_card(kt, fmt, shape, count, given):
    """A prompt whose tiles are not cut; also where the sequence has fewer rows than the call has room for."""
    n = count if given is None else given
    b = Batch(kt, 64, [7], [n], shape, fmt, 64, extra=count - n, spare=20)
    b.most, b.words, b.key_bound = count, -(-count // 32), count + 7
    b.tables = np.concatenate([b.tables, np.full((1, 20), -7, np.int32)], 1)
    b.stride += 20
    b.upload()
    check(b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_rows_at_any_float(kt, fmt, dim):
    """kt_rope_paged takes q, k, v and q_out that begin at any float."""
    b = Batch(kt, 65, [5, 40], [30, 3], (6, 3, dim), fmt, 16, extra=1)
    b.rope()
    want, pool = b.context().tobytes(), [p.tobytes() for p in b.pool_bits()]
    b.upload()
    at = {}
    for name in ("q", "k", "v", "context"):
        array = b.d["context"].download(np.float32) if name == "context" else getattr(b, name)
        buffer = at[name] = kt.DeviceBuffer(array.nbytes + 4)
        buffer.upload(array, offset=4)
    b.lib.call("kt_rope_paged", at["q"].ptr + 4, at["k"].ptr + 4, at["v"].ptr + 4, b.heads, b.d["inv_freq"].ptr, ctypes.byref(b.cache), 0,
               ctypes.byref(b.batch), at["context"].ptr + 4, None)
    assert at["context"].download(np.float32, offset=4).tobytes() == want
    assert [p.tobytes() for p in b.pool_bits()] == pool


@pytest.mark.parametrize("fmt,dim", [("float16", 64), ("bfloat16", 128), ("float32", 64), ("float32", 256)])
def test_many_sequences_of_many_rows(kt, fmt, dim):
    """More sequences than lanes, with tiles of many rows; a long one among the last is cut, one without rows is not there."""
    rng = np.random.default_rng(dim)
    lengths = rng.integers(0, 60, 150).tolist()
    counts = rng.integers(0, 50, 150).tolist()
    lengths[70], counts[70] = 2500, 0
    lengths[140], counts[140] = 4000, 45
    lengths[3], counts[3] = 1500, 33
    check(Batch(kt, 66, lengths, counts, (2, 1, dim), fmt, 64, extra=3))


def test_recorded_trees_of_many_rows(kt):
    """A recorded call whose tiles are cut and merged, with other lengths and trees from replay to replay, between eager calls."""
    counts, rng = [60, 0, 33], np.random.default_rng(67)
    stream = kt.Stream.create()
    b = Batch(kt, 67, [900, 1500, 40], counts, (8, 2, 64), "float16", 32, parents=random_parents(rng, counts))
    b.rope_attention(stream=stream.handle)
    graph = ctypes.c_void_p()
    b.lib.call("kt_graph_begin", stream.handle)
    b.masks(stream.handle)
    b.rope_attention(stream=stream.handle)
    b.lib.call("kt_graph_end", stream.handle, ctypes.byref(graph))
    for lengths in ([900, 1500, 40], [3, 1500, 0], [860, 0, 31], [900, 1500, 40]):
        b.lengths, b.parents = lengths, random_parents(rng, counts)
        b.d["lengths"].upload(np.array(lengths, np.int32), stream)
        b.d["parents"].upload(np.concatenate(b.parents), stream)
        b.append()
        b.lib.call("kt_graph_launch", graph, stream.handle)
        replayed = b.context(stream)
        b.check_context(replayed, *b.attend(b.rotated()))
        b.masks(stream.handle)
        b.rope_attention(stream=stream.handle)
        assert b.context(stream).tobytes() == replayed.tobytes()
    b.lib.call("kt_graph_destroy", graph)
    stream.destroy()
