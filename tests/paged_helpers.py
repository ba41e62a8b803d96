"""A batch of sequences over a cache in pages, on the device and in the oracle side by side."""
from __future__ import annotations

import ctypes

import numpy as np

from gpu_helpers import banner
from oracle import paged_ref

FORMATS = {"float32": 0, "float16": 1, "bfloat16": 2}


def random_parents(rng, counts):
    """A tree for each sequence: row 0 its root, each other row below an earlier one."""
    return [np.array([-1] + [int(rng.integers(0, i)) for i in range(1, n)], np.int32)[:n] for n in counts]


class Batch:
    """Sequences of `lengths` tokens with `counts` further rows each, in pages that lie in random order. Memory that no
    sequence holds is NaN. extra: rows behind the last sequence's; lead: rows before the first's."""

    def __init__(self, kt, seed, lengths, counts, shape, fmt="float32", page=16, layers=1, parents=None, extra=0, lead=0, spare=2, key_bound=None,
                 loud=1.0):
        from kotensor_amd import _lib
        banner("paged", seed, lengths, counts, shape, fmt, page, layers, "tree" if parents is not None else "text")
        self.kt, self.lib = kt, _lib
        self.rng = rng = np.random.default_rng(seed)
        self.heads, self.kv_heads, self.head_dim = shape
        self.lengths, self.counts, self.fmt, self.page, self.layers = list(lengths), list(counts), fmt, page, layers
        total = [max(length, 0) + n for length, n in zip(lengths, counts)]
        need = [-(-t // page) for t in total]
        self.stride = max(need + [1])
        pages = sum(need) + spare
        order = rng.permutation(pages).tolist()
        self.tables = np.full((len(lengths), self.stride), -7, np.int32)
        for s, n in enumerate(need):
            self.tables[s, :n] = [order.pop() for _ in range(n)]
        self.pool = paged_ref.Pool(layers, pages, self.kv_heads, page, self.head_dim, fmt, lambda shape: np.full(shape, np.nan, np.float32))
        for layer in range(layers):
            for s, length in enumerate(lengths):
                held = [loud * rng.standard_normal((max(length, 0), self.kv_heads, self.head_dim)).astype(np.float32) for _ in range(2)]
                self.pool.append(layer, self.tables[s], 0, *held)
        self.starts = np.concatenate([[lead], lead + np.cumsum(counts)]).astype(np.int32)
        self.rows = int(self.starts[-1]) + extra
        self.q = rng.standard_normal((self.rows, self.heads, self.head_dim)).astype(np.float32)
        self.k, self.v = (rng.standard_normal((layers, self.rows, self.kv_heads, self.head_dim)).astype(np.float32) for _ in range(2))
        self.parents = parents
        self.inv_freq = paged_ref.inv_freq(self.head_dim)
        self.most = max(list(counts) + [0])
        self.words = max(1, -(-self.most // 32))
        self.key_bound = max(max(total, default=0), self.most) if key_bound is None else key_bound
        self.upload()

    # -- the oracle's side ---------------------------------------------------------------
    def sequence_rows(self, s):
        return slice(int(self.starts[s]), int(self.starts[s + 1]))

    def positions(self, s):
        base = np.arange(self.counts[s]) if self.parents is None else paged_ref.masks(self.parents[s], self.words)[0]
        return self.lengths[s] + base

    def visible(self, s):
        """[rows x tokens] of sequence s."""
        length, n = self.lengths[s], self.counts[s]
        total = max(length + n, 0)
        token = np.arange(total)
        see = np.broadcast_to(token < length, (n, total)).copy()
        for i in range(n):
            rows = range(i + 1) if self.parents is None else paged_ref.above(self.parents[s])[i]
            for j in rows:
                if 0 <= length + j < total:
                    see[i, length + j] = True
        see &= np.array([self.pool.place(self.tables[s], t) is not None for t in token], bool)[None] if total else False
        return see & (token < self.key_bound)

    def append(self, layer=0):
        for s in range(len(self.counts)):
            r = self.sequence_rows(s)
            self.pool.append(layer, self.tables[s], self.lengths[s], paged_ref.rotate(self.k[layer, r], self.positions(s), self.inv_freq), self.v[layer, r])

    def rotated(self):
        out = self.q.copy()
        for s in range(len(self.counts)):
            r = self.sequence_rows(s)
            out[r] = paged_ref.rotate(self.q[r], self.positions(s), self.inv_freq)
        return out

    def attend(self, q, layer=0):
        """(context, bound) [rows x heads x d]; rows of no sequence are NaN."""
        out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
        for s in range(len(self.counts)):
            r, see = self.sequence_rows(s), self.visible(s)
            keys, values = (self.pool.rows(w, layer, self.tables[s], range(see.shape[1])) for w in ("keys", "values"))
            out[r], bound[r] = paged_ref.attend(q[r], keys, values, see)
        return out, bound

    # -- the device's side ---------------------------------------------------------------
    def upload(self):
        buf = self.kt.DeviceBuffer.from_numpy
        self.d = {n: buf(getattr(self, n)) for n in ("tables", "starts", "q", "k", "v", "inv_freq")}
        self.d["lengths"] = buf(np.array(self.lengths + [0], np.int32))
        self.d["keys"], self.d["values"] = buf(self.pool.keys), buf(self.pool.values)
        self.d["context"] = buf(np.full(self.q.shape, np.nan, np.float32))
        self.d["depths"], self.d["masks"] = self.kt.DeviceBuffer(4 * max(1, self.rows)), self.kt.DeviceBuffer(4 * max(1, self.rows) * self.words)
        flat = np.full(max(1, self.rows), -1, np.int32)
        for s, p in enumerate(self.parents or []):
            flat[self.sequence_rows(s)] = p
        self.d["parents"] = buf(flat)
        c, b = self.lib.PagedCache(), self.lib.PagedBatch()
        c.keys, c.values, c.format = self.d["keys"].ptr, self.d["values"].ptr, FORMATS[self.fmt]
        c.layers, c.pages, c.kv_heads, c.page_tokens, c.head_dim = self.layers, self.pool.pages, self.kv_heads, self.page, self.head_dim
        b.tables, b.lengths, b.starts = (self.d[n].ptr for n in ("tables", "lengths", "starts"))
        b.table_stride, b.sequences, b.rows, b.most_rows, b.key_bound, b.mask_words = self.stride, len(self.counts), self.rows, self.most, self.key_bound, self.words
        if self.parents is not None:
            b.depths, b.masks = self.d["depths"].ptr, self.d["masks"].ptr
        self.cache, self.batch = c, b
        if self.parents is not None and self.rows:
            self.masks()

    def masks(self, stream=None):
        self.lib.call("kt_tree_masks", self.d["parents"].ptr, ctypes.byref(self.batch), self.d["depths"].ptr, self.d["masks"].ptr, stream)

    def row_bytes(self, name):
        return getattr(self, name)[0].nbytes

    def rope(self, layer=0, q=True, stream=None):
        at = layer * self.row_bytes("k")
        self.lib.call("kt_rope_paged", self.d["q"].ptr if q else None, self.d["k"].ptr + at, self.d["v"].ptr + at, self.heads, self.d["inv_freq"].ptr,
                      ctypes.byref(self.cache), layer, ctypes.byref(self.batch), self.d["context"].ptr if q else None, stream)

    def attention(self, layer=0, stream=None):
        self.lib.call("kt_attention_paged", self.d["q"].ptr, self.heads, ctypes.byref(self.cache), layer, ctypes.byref(self.batch), self.d["context"].ptr, stream)

    def rope_attention(self, layer=0, stream=None):
        at = layer * self.row_bytes("k")
        self.lib.call("kt_rope_attention_paged", self.d["q"].ptr, self.d["k"].ptr + at, self.d["v"].ptr + at, self.d["inv_freq"].ptr, self.heads,
                      ctypes.byref(self.cache), layer, ctypes.byref(self.batch), self.d["context"].ptr, stream)

    def context(self, stream=None):
        return self.d["context"].download(np.float32, stream=stream).reshape(self.q.shape)

    def pool_bits(self):
        kind = self.pool.keys.dtype
        return tuple(self.d[n].download(kind).reshape(self.pool.keys.shape) for n in ("keys", "values"))

    # -- comparisons -----------------------------------------------------------------------
    def check_pool(self):
        for got, want, name in zip(self.pool_bits(), (self.pool.keys, self.pool.values), ("keys", "values")):
            kind = np.uint32 if got.dtype == np.float32 else np.uint16
            same = (got.view(kind) == want.view(kind)) | (np.isnan(paged_ref.from_bits(got, self.fmt)) & np.isnan(paged_ref.from_bits(want, self.fmt)))
            assert same.all(), (name, np.argwhere(~same)[:5].tolist())

    def check_context(self, got, want, bound):
        held = np.zeros(self.rows, bool)
        held[int(self.starts[0]):int(self.starts[-1])] = True
        assert np.isnan(got[~held]).all()
        off = np.abs(got[held] - want[held])
        worst = np.unravel_index(np.argmax(np.where(np.isnan(off), np.inf, off - bound[held])), off.shape) if off.size else None
        assert off.size == 0 or (off <= bound[held] + 2.0 ** -126).all(), (worst, got[held][worst], want[held][worst], bound[held][worst])
