"""``QuantizedKVCache``: the KV cache held in 8 bits, with a scale for each block of tokens and
head (``kt_kv8_cache``), in the place of ``KVCache`` in ``Transformer``'s calls.

A quarter of the fp32 cache's memory, and of what a decode step's attention reads of it. No
counterpart in the reference, whose ``KVCache`` (KVCache.kt:3-59) is fp32; the names, checks and
messages are ``KVCache``'s.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from .device import DeviceBuffer, Stream, default_stream

FORMATS = {"int8": _lib.KT_KV8_INT8, "e4m3": _lib.KT_KV8_E4M3}


class QuantizedKVCache:
    """Keys and values of ``[layers x heads x max_sequence_length x head_dim]`` as 8-bit codes
    (``format`` "int8" or "e4m3") in device memory, a scale for every ``block_tokens`` tokens of a
    head, the fp32 rows of the block that is not full, and the length, kept on the host and, for
    the kernels, as a device int32."""

    def __init__(self, num_layers: int, num_heads: int, max_sequence_length: int, head_dim: int, format: str = "int8",
                 block_tokens: int = 64, stream: Stream | None = None):
        if num_layers <= 0:
            raise _lib.IllegalArgumentException("numLayers must be positive")
        if num_heads <= 0:
            raise _lib.IllegalArgumentException("numHeads must be positive")
        if max_sequence_length <= 0:
            raise _lib.IllegalArgumentException("maxSequenceLength must be positive")
        if head_dim <= 0:
            raise _lib.IllegalArgumentException("headDim must be positive")
        if format not in FORMATS:
            raise _lib.IllegalArgumentException(f"cache format {format!r}: one of {', '.join(FORMATS)}")
        self.num_layers, self.num_heads = int(num_layers), int(num_heads)
        self.max_sequence_length, self.head_dim = int(max_sequence_length), int(head_dim)
        self.format, self.block_tokens = format, int(block_tokens)
        c = _lib.KV8Cache()
        c.format, c.layers, c.kv_heads = FORMATS[format], self.num_layers, self.num_heads
        c.max_seq, c.head_dim, c.block_tokens = self.max_sequence_length, self.head_dim, self.block_tokens
        sizes = (ctypes.c_int64 * 3)()
        _lib.call("kt_kv8_layout", ctypes.byref(c), sizes)
        self.keys, self.values = DeviceBuffer(sizes[0]), DeviceBuffer(sizes[0])
        self.key_scales, self.value_scales = DeviceBuffer(4 * sizes[1]), DeviceBuffer(4 * sizes[1])
        self.key_rows, self.value_rows = DeviceBuffer(4 * sizes[2]), DeviceBuffer(4 * sizes[2])
        self.position = DeviceBuffer(4)
        for name in ("keys", "values", "key_scales", "value_scales", "key_rows", "value_rows"):
            setattr(c, name, getattr(self, name).ptr)
            getattr(self, name).fill_zero(stream)
        self.position.fill_zero(stream)
        self.cache = c  # kt_kv8_cache
        self.length = 0

    @property
    def remaining(self) -> int:
        return self.max_sequence_length - self.length

    def check_room(self, count: int) -> None:
        if count < 0:
            raise _lib.IllegalArgumentException("count must not be negative")
        if self.length + count > self.max_sequence_length:
            raise _lib.IllegalArgumentException(
                f"KV cache full: {self.length} + {count} positions exceed maxSequenceLength {self.max_sequence_length}")

    def advance(self, count: int, stream: Stream | None = None) -> None:
        """The host length and the device length move together."""
        self.check_room(count)
        _lib.call("kt_position_add", self.position.ptr, int(count), (stream or default_stream()).handle)
        self.length += count

    def reset(self, stream: Stream | None = None) -> None:
        self.position.fill_zero(stream)
        self.length = 0

    def copy_from(self, source: "QuantizedKVCache", length: int, stream: Stream | None = None) -> None:
        """The first ``length`` positions of ``source`` (KVCache.copyFrom, KVCache.kt:41-55), which may
        be this cache: it is then shortened (drafted tokens that were not taken)."""
        shape = "a cache of {0.num_layers} layers × {0.num_heads} heads × {0.head_dim} dims, {0.format}, {0.block_tokens} tokens a block".format
        if shape(source) != shape(self):
            raise _lib.IllegalArgumentException(f"Cannot copy {shape(source)} into {shape(self)}")
        if not 0 <= length <= source.length:
            raise _lib.IllegalArgumentException(f"Cannot copy {length} positions from a cache holding {source.length}")
        if length > self.max_sequence_length:
            raise _lib.IllegalArgumentException(f"Cannot copy {length} positions into a cache of {self.max_sequence_length}")
        _lib.call("kt_kv8_copy", ctypes.byref(source.cache), source.length, ctypes.byref(self.cache), int(length),
                  (stream or default_stream()).handle)
        self.position.upload(np.array([length], np.int32), stream)
        self.length = length

    @property
    def size_in_bytes(self) -> int:
        return sum(getattr(self, n).nbytes for n in ("keys", "values", "key_scales", "value_scales", "key_rows", "value_rows"))

    def rows_numpy(self, layer: int, first: int = 0, count: int | None = None, stream: Stream | None = None):
        """(keys, values) of the tokens from ``first`` on as the cache holds them, fp32
        ``[heads x count x head_dim]``."""
        count = self.length - first if count is None else count
        shape = (self.num_heads, max(count, 0), self.head_dim)
        out = [DeviceBuffer(4 * int(np.prod(shape))) for _ in range(2)]
        _lib.call("kt_kv8_read", ctypes.byref(self.cache), int(layer), int(first), int(count), out[0].ptr, out[1].ptr,
                  (stream or default_stream()).handle)
        return tuple(b.download(np.float32, stream=stream).reshape(shape) for b in out)
