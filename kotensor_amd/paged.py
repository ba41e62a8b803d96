"""``PagedKVCache``: a KV cache in pages that several sequences share (``kt_paged_cache``), its batches
(``PagedBatch``), and drafts of a text's next tokens from the text itself (``TextDraft``).

No counterpart in the reference, whose ``KVCache`` (KVCache.kt:3-59) holds one sequence; the names,
checks and messages are ``KVCache``'s.
"""
from __future__ import annotations

import contextlib
import ctypes

import numpy as np

from . import _lib
from .device import DeviceBuffer, Stream, default_stream

FORMATS = {"float32": _lib.KT_PAGED_F32, "float16": _lib.KT_PAGED_F16, "bfloat16": _lib.KT_PAGED_BF16}


class PagedKVCache:
    """Keys and values of up to ``sequences`` sequences in ``pages`` pages of ``page_tokens`` tokens, held as ``format``
    ("float32", "float16", "bfloat16"); by default as many pages as all sequences need at
    ``max_sequence_length`` tokens. Sequences take pages as they grow (``reserve``) and give them back (``release``). Lengths
    and page numbers are kept on the host and, for the kernels, on the device. All calls on a cache go to one stream."""

    def __init__(self, num_layers: int, num_heads: int, sequences: int, max_sequence_length: int, head_dim: int, format: str = "float32",
                 page_tokens: int = 64, pages: int | None = None, stream: Stream | None = None):
        for name, value in (("numLayers", num_layers), ("numHeads", num_heads), ("sequences", sequences),
                            ("maxSequenceLength", max_sequence_length), ("headDim", head_dim), ("pageTokens", page_tokens)):
            if value <= 0:
                raise _lib.IllegalArgumentException(f"{name} must be positive")
        if format not in FORMATS:
            raise _lib.IllegalArgumentException(f"cache format {format!r}: one of {', '.join(FORMATS)}")
        self.num_layers, self.num_heads, self.head_dim = int(num_layers), int(num_heads), int(head_dim)
        self.sequences, self.max_sequence_length = int(sequences), int(max_sequence_length)
        self.format, self.page_tokens = format, int(page_tokens)
        self.table_stride = -(-self.max_sequence_length // self.page_tokens)
        self.pages = self.sequences * self.table_stride if pages is None else int(pages)
        c = _lib.PagedCache()
        c.format, c.layers, c.pages, c.kv_heads = FORMATS[format], self.num_layers, self.pages, self.num_heads
        c.page_tokens, c.head_dim = self.page_tokens, self.head_dim
        size = ctypes.c_int64()
        _lib.call("kt_paged_layout", ctypes.byref(c), ctypes.byref(size))
        self.keys, self.values = DeviceBuffer(size.value), DeviceBuffer(size.value)
        c.keys, c.values = self.keys.ptr, self.values.ptr
        self.cache = c  # kt_paged_cache
        self.tables = DeviceBuffer.from_numpy(np.full((self.sequences, self.table_stride), -1, np.int32), stream)
        self.device_lengths = DeviceBuffer.from_numpy(np.zeros(self.sequences, np.int32), stream)
        self.lengths = [0] * self.sequences
        self._held: list[list[int]] = [[] for _ in range(self.sequences)]
        self._holders = [0] * self.pages  # sequences that hold a page
        self._free = list(range(self.pages - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def check_sequence(self, sequence: int) -> None:
        if not 0 <= sequence < self.sequences:
            raise _lib.IllegalArgumentException(f"sequence {sequence} out of bounds {self.sequences}")

    def reserve(self, counts: dict[int, int], stream: Stream | None = None) -> None:
        """Pages for ``counts[sequence]`` further tokens of each sequence, or an error and none."""
        need = {}
        for sequence, count in counts.items():
            self.check_sequence(sequence)
            if count < 0:
                raise _lib.IllegalArgumentException("count must not be negative")
            total = self.lengths[sequence] + count
            if total > self.max_sequence_length:
                raise _lib.IllegalArgumentException(
                    f"KV cache full: {self.lengths[sequence]} + {count} positions exceed maxSequenceLength {self.max_sequence_length}")
            need[sequence] = max(-(-total // self.page_tokens) - len(self._held[sequence]), 0)
        if sum(need.values()) > len(self._free):
            raise _lib.IllegalArgumentException(f"KV cache full: {sum(need.values())} pages needed, {len(self._free)} of {self.pages} free")
        for sequence, n in need.items():
            if n:
                taken = [self._free.pop() for _ in range(n)]
                for page in taken:
                    self._holders[page] = 1
                self._upload(sequence, taken, stream)

    def _upload(self, sequence: int, taken: list[int], stream) -> None:
        """Further pages of a sequence, on the host and on the device."""
        at = 4 * (sequence * self.table_stride + len(self._held[sequence]))
        self.tables.upload(np.array(taken, np.int32), stream, offset=at)
        self._held[sequence] += taken

    def set_length(self, sequence: int, length: int, stream: Stream | None = None) -> None:
        """Shortens a sequence to ``length`` tokens; it keeps its pages."""
        self.check_sequence(sequence)
        if not 0 <= length <= self.lengths[sequence]:
            raise _lib.IllegalArgumentException(f"Cannot keep {length} positions of a sequence holding {self.lengths[sequence]}")
        if any(self._holders[page] > 1 for page in self._held[sequence][length // self.page_tokens:]):
            raise _lib.IllegalArgumentException("pages that the sequence would write over are shared: release it instead")
        self.device_lengths.upload(np.array([length], np.int32), stream, offset=4 * sequence)
        self.lengths[sequence] = length

    def release(self, sequence: int, stream: Stream | None = None) -> None:
        """Empties a sequence; the pages that no other holds are free."""
        self.check_sequence(sequence)
        self.device_lengths.upload(np.zeros(1, np.int32), stream, offset=4 * sequence)
        self.lengths[sequence] = 0
        for page in reversed(self._held[sequence]):
            self._holders[page] -= 1
            if self._holders[page] == 0:
                self._free.append(page)
        self._held[sequence] = []

    def share(self, source: int, target: int, count: int, stream: Stream | None = None) -> int:
        """The first ``count`` tokens of ``source``, down to a whole number of pages, become the empty sequence ``target``'s as
        well, without a copy (several texts with one beginning). Returns how many tokens that are."""
        self.check_sequence(source)
        self.check_sequence(target)
        if not 0 <= count <= self.lengths[source]:
            raise _lib.IllegalArgumentException(f"Cannot share {count} positions of a sequence holding {self.lengths[source]}")
        if self._held[target]:
            raise _lib.IllegalArgumentException(f"sequence {target} is not empty")
        pages = self._held[source][:count // self.page_tokens]
        for page in pages:
            self._holders[page] += 1
        if pages:
            self._upload(target, list(pages), stream)
        shared = len(pages) * self.page_tokens
        self.device_lengths.upload(np.array([shared], np.int32), stream, offset=4 * target)
        self.lengths[target] = shared
        return shared

    @contextlib.contextmanager
    def unchanged_on_error(self, stream: Stream | None = None):
        """An error of what runs inside leaves the sequences as long as they were before, on the host and on the device (they keep
        the pages that they took)."""
        lengths = list(self.lengths)
        try:
            yield
        except BaseException:
            self.lengths = lengths
            self.device_lengths.upload(np.array(lengths, np.int32), stream)  # (after what is enqueued)
            raise

    @property
    def size_in_bytes(self) -> int:
        return self.keys.nbytes + self.values.nbytes

    def rows_numpy(self, layer: int, sequence: int, first: int = 0, count: int | None = None, stream: Stream | None = None):
        """(keys, values) of a sequence's tokens from ``first`` on as the cache holds them, fp32 ``[heads x count x head_dim]``."""
        self.check_sequence(sequence)
        count = self.lengths[sequence] - first if count is None else count
        shape = (self.num_heads, max(count, 0), self.head_dim)
        out = [DeviceBuffer(4 * int(np.prod(shape))) for _ in range(2)]
        _lib.call("kt_paged_read", ctypes.byref(self.cache), int(layer), ctypes.c_void_p(self.tables.ptr + 4 * sequence * self.table_stride),
                  self.table_stride, int(first), int(count), out[0].ptr, out[1].ptr, (stream or default_stream()).handle)
        return tuple(b.download(np.float32, stream=stream).reshape(shape) for b in out)


class PagedBatch:
    """The rows of a call on a ``PagedKVCache``: ``counts[s]`` further tokens of sequence s, which have pages (``reserve``), in the
    order of the sequences, as texts, or as trees when ``buffers`` holds their parents. key_bound: what the sequences' tokens stay below,
    where the call is recorded and they grow from replay to replay."""

    def __init__(self, cache: PagedKVCache, counts: list[int], starts: DeviceBuffer, key_bound: int | None = None,
                 buffers: "BatchBuffers | None" = None, stream: Stream | None = None):
        counts = [int(n) for n in counts]
        if len(counts) != cache.sequences:
            raise _lib.IllegalArgumentException(f"{len(counts)} counts for {cache.sequences} sequences")
        for sequence, n in enumerate(counts):
            if n < 0:
                raise _lib.IllegalArgumentException("counts must not be negative")
            if n and cache.lengths[sequence] + n > len(cache._held[sequence]) * cache.page_tokens:
                raise _lib.IllegalArgumentException(f"sequence {sequence} has no pages for {n} tokens after {cache.lengths[sequence]}: reserve them first")
        tokens = max((length + n for length, n in zip(cache.lengths, counts) if n), default=0)
        if key_bound is not None and key_bound < tokens:
            raise _lib.IllegalArgumentException(f"key bound {key_bound} for sequences of up to {tokens} tokens")
        if buffers is not None and sum(counts) > buffers.rows:
            raise _lib.IllegalArgumentException(f"{sum(counts)} tokens exceed the buffers' {buffers.rows} rows")
        first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        starts.upload(first, stream)
        b = _lib.PagedBatch()
        b.tables, b.lengths, b.starts = cache.tables.ptr, cache.device_lengths.ptr, starts.ptr
        b.table_stride, b.sequences = cache.table_stride, cache.sequences
        b.rows, b.most_rows = int(first[-1]), max(counts)
        b.key_bound = tokens if key_bound is None else key_bound
        if buffers is not None:
            b.depths, b.masks, b.mask_words = buffers.depths.ptr, buffers.masks.ptr, max(1, -(-b.most_rows // 32))
        self.cache, self.counts, self.starts = cache.cache, counts, first
        self.batch = b  # kt_paged_batch


class TextDraft:
    """Drafts of a text's next tokens from what followed its last tokens before: of the up to ``branches`` latest places where
    the longest matching run of its last ``match`` tokens or fewer occurs, the ``tokens`` tokens that follow, as one tree."""

    def __init__(self, tokens: int = 8, branches: int = 2, match: int = 3):
        if min(tokens, branches, match) <= 0:
            raise _lib.IllegalArgumentException("tokens, branches and match must be positive")
        self.tokens, self.branches, self.match = int(tokens), int(branches), int(match)

    @property
    def most_tokens(self) -> int:
        return self.tokens * self.branches

    def __call__(self, text: list[int]) -> tuple[list[int], list[int]]:
        """(tokens, parents) of the tree: parents[i] is the index of the token before tokens[i], -1 for the text's last."""
        places: list[int] = []
        for run in range(min(self.match, len(text) - 1), 0, -1):
            last = text[-run:]
            places = [end for end in range(len(text) - 1, run - 1, -1) if text[end - run:end] == last][:self.branches]
            if places:
                break
        tokens: list[int] = []
        parents: list[int] = []
        children: dict[tuple[int, int], int] = {}
        for end in places:
            at = -1
            for token in text[end:end + self.tokens]:
                if (at, token) not in children:
                    children[at, token] = len(tokens)
                    tokens.append(token)
                    parents.append(at)
                at = children[at, token]
        return tokens, parents
