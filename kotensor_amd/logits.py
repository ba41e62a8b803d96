"""Control of the next token by the text so far: penalties for its tokens, biases, and a grammar's
mask on rows of logits (``kt_process_logits``). No counterpart in the reference, whose greedy
choice takes the logits as they are (Transformer.kt:253-266).
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from .device import DeviceBuffer, Stream, default_stream
from .matmul import DeviceTensor, _nbytes, _ptr

NO_CANDIDATE = -1e9  # kt_argmax takes logits above this only


class LogitsControls:
    """Penalties, biases and a mask, in this order on a logit x (oracle: the header's formulas):

    * ``repetition_penalty``: a token of the text has x / penalty (x > 0) or x * penalty;
    * ``frequency_penalty``, ``presence_penalty``: a token that occurs o > 0 times in the text's
      output has x - (o * frequency + presence);
    * ``bias``: {token: value} added to x;
    * ``allowed``: tokens that may follow, as a boolean array of the vocabulary (one for all rows,
      or one a row) or, packed, its 32-bit words; the others have minus infinity. A grammar replaces
      it between steps with ``set_allowed``, which keeps the device address.

    The argmax takes no logit at or below -1e9: a bias of that size bans its token, as minus infinity does, and so
    does such a penalty. Where the mask and the biases leave no token, ``greedy_decode``, ``decode_step`` and replays
    refuse; where penalties of 1e9 leave none, the argmax gives token 0.
    """

    def __init__(self, repetition_penalty: float = 1.0, frequency_penalty: float = 0.0, presence_penalty: float = 0.0,
                 bias: dict | None = None, allowed=None, stream: Stream | None = None):
        if not 0.0 < repetition_penalty < float("inf"):
            raise _lib.IllegalArgumentException("the repetition penalty must be positive and finite")
        for name, value in (("frequency", frequency_penalty), ("presence", presence_penalty)):
            if not abs(value) < float("inf"):
                raise _lib.IllegalArgumentException(f"the {name} penalty must be finite")
        self.repetition_penalty, self.frequency_penalty, self.presence_penalty = map(float, (repetition_penalty, frequency_penalty, presence_penalty))
        self.bias_count = len(bias or {})
        self._bias_ids = sorted(int(t) for t in bias or {})
        self._banned = [int(t) for t, v in (bias or {}).items() if not v > NO_CANDIDATE]
        if self.bias_count:
            self._bias_tokens = DeviceBuffer.from_numpy(np.array(list(bias.keys()), np.int32), stream)
            self._bias_values = DeviceBuffer.from_numpy(np.array(list(bias.values()), np.float32), stream)
        self._allowed, self._words = None, (0, 0)
        self._entries: int | None = None  # tokens of a boolean mask; packed words hold no length
        self._vocabulary: int | None = None  # of the calls that the mask was described for
        self._host_words: np.ndarray | None = None
        self._may_follow: int | None = None  # the vocabulary of which the present mask and biases leave a token
        if allowed is not None:
            self.set_allowed(allowed, stream)

    @property
    def penalized(self) -> bool:
        return (self.repetition_penalty, self.frequency_penalty, self.presence_penalty) != (1.0, 0.0, 0.0)

    @property
    def masked(self) -> bool:
        return self._allowed is not None

    def set_allowed(self, allowed, stream: Stream | None = None) -> None:
        """Sets the mask. Another one of the same shape replaces it in the same device memory, which a
        recorded step then reads at its next replay; one of another shape is refused. A boolean mask has
        one entry for each token of the vocabulary, packed words as many as hold them."""
        a = np.asarray(allowed)
        entries = a.shape[-1] if a.ndim and a.dtype == np.bool_ else None
        if a.ndim not in (1, 2) or a.size == 0:
            raise _lib.IllegalArgumentException(f"a mask is an array of the vocabulary, or one a row, got {list(a.shape)}")
        if a.dtype == np.bool_:
            pad = np.zeros(a.shape[:-1] + (-a.shape[-1] % 32,), np.bool_)
            a = np.packbits(np.concatenate([a, pad], -1), axis=-1, bitorder="little").view("<u4")
        elif a.dtype not in (np.dtype("u4"), np.dtype("i4")):
            raise _lib.IllegalArgumentException(f"a mask is boolean or packed in 32-bit words, got {a.dtype}")
        words = (a.shape[0] if a.ndim == 2 else 0, a.shape[-1])
        if self._vocabulary is not None and words == self._words:
            self._check_entries(entries, self._vocabulary)
        if self._allowed is None:
            self._allowed, self._words = DeviceBuffer(a.nbytes), words
        elif words != self._words:  # (a recorded step may address the memory)
            raise _lib.IllegalArgumentException(
                f"a mask of {words[0]} rows, {words[1]} words cannot replace one of {self._words[0]} rows, {self._words[1]} words")
        self._allowed.upload(a, stream)
        self._entries, self._host_words, self._may_follow = entries, a.view(np.uint32).copy(), None

    @staticmethod
    def _check_entries(entries: int | None, vocabulary: int) -> None:
        if entries not in (None, vocabulary):
            raise _lib.IllegalArgumentException(f"a mask of {entries} tokens for a vocabulary of {vocabulary}")

    def check(self, rows: int, vocabulary: int) -> None:
        """Refuses rows of logits that the biases or the mask do not fit."""
        if self._bias_ids and not 0 <= self._bias_ids[0] <= self._bias_ids[-1] < vocabulary:
            raise _lib.IllegalArgumentException(f"a biased token is out of vocab bounds {vocabulary}")
        if self._allowed is not None:
            if self._words[0] not in (0, rows):
                raise _lib.IllegalArgumentException(f"a mask of {self._words[0]} rows for {rows} rows of logits")
            if self._words[1] != (vocabulary + 31) // 32:
                raise _lib.IllegalArgumentException(f"a mask of {self._words[1]} words does not hold {vocabulary} tokens")
            self._check_entries(self._entries, vocabulary)
            self._vocabulary = vocabulary

    def check_choice(self, vocabulary: int) -> None:
        """Refuses a choice where the mask and the biases leave no token of the vocabulary, which the argmax would
        answer with token 0."""
        self.check(1, vocabulary)
        if self._may_follow == vocabulary:
            return
        words = np.full((vocabulary + 31) // 32, 0xFFFFFFFF, np.uint32) if self._host_words is None else self._host_words.reshape(-1).copy()
        if vocabulary % 32:
            words[vocabulary // 32] &= np.uint32((1 << vocabulary % 32) - 1)
        for t in self._banned:
            words[t // 32] &= np.uint32(~(1 << t % 32) & 0xFFFFFFFF)
        if not words[:(vocabulary + 31) // 32].any():
            raise _lib.IllegalArgumentException("no token may follow: the mask and the biases leave none of the vocabulary")
        self._may_follow = vocabulary

    def descriptor(self, rows: int, vocabulary: int, history=None, history_length=None, output_start=None, history_stride: int = 0,
                   history_capacity: int = 0, length_offset: int = 0) -> _lib.LogitsControls:
        """The kt_logits_controls of a call on ``rows`` rows (device buffers or addresses)."""
        self.check(rows, vocabulary)
        c = _lib.LogitsControls()
        c.history, c.history_length, c.output_start = _ptr(history), _ptr(history_length), _ptr(output_start)
        c.history_stride, c.history_capacity, c.length_offset = history_stride, history_capacity, length_offset
        c.repetition, c.frequency, c.presence = self.repetition_penalty, self.frequency_penalty, self.presence_penalty
        c.bias_count = self.bias_count
        if self.bias_count:
            c.bias_tokens, c.bias_values = self._bias_tokens.ptr, self._bias_values.ptr
        if self._allowed is not None:
            c.allowed, c.allowed_stride = self._allowed.ptr, self._words[1] if self._words[0] else 0
        return c


def process_logits(logits: DeviceTensor, controls: LogitsControls, history: DeviceBuffer | None = None, history_length: DeviceBuffer | None = None,
                   output_start: DeviceBuffer | None = None, out: DeviceTensor | None = None, stream: Stream | None = None) -> DeviceTensor:
    """The controls on logits ``[rows x vocabulary]``, into ``out`` (a new tensor when not given; it may
    be ``logits``). ``history`` holds int32 tokens ``[rows x capacity]``, ``history_length`` and
    ``output_start`` one int32 a row."""
    if len(logits.shape) != 2:
        raise _lib.IllegalArgumentException("not a matrix")
    rows, n = logits.shape
    if out is None:
        out = DeviceTensor(DeviceBuffer(rows * n * 4), (rows, n))
    if out.shape != logits.shape:
        raise _lib.IllegalArgumentException(f"out shape {list(out.shape)} != {list(logits.shape)}")
    capacity = 0
    if controls.penalized:
        if history is None or history_length is None:
            raise _lib.IllegalArgumentException("penalties need the history and its length")
        if rows and history.nbytes % (4 * rows):
            raise _lib.IllegalArgumentException(f"a history of {history.nbytes} bytes does not hold {rows} rows of tokens")
        capacity = history.nbytes // (4 * max(rows, 1))
        for name, b in (("history_length", history_length), ("output_start", output_start)):
            if b is not None and _nbytes(b) < 4 * rows:
                raise _lib.IllegalArgumentException(f"{name} has {_nbytes(b) // 4} elements, needs {rows}")
    c = controls.descriptor(rows, n, history, history_length, output_start, capacity, capacity)
    _lib.call("kt_process_logits", logits.ptr, rows, n, ctypes.c_int64(n), ctypes.byref(c), out.ptr, ctypes.c_int64(n),
              (stream or default_stream()).handle)
    return out
