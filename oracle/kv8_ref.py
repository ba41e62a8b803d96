"""The KV cache held in 8 bits and the controls on logits, restated in numpy: the format's
roundings in fp32 as it defines them, everything else in 64 bits.
"""
from __future__ import annotations

import numpy as np

import oracle
from oracle import decoder_ref

QMAX = {"int8": np.float32(127.0), "e4m3": np.float32(448.0)}
MIN_SCALE = np.float32(2.0 ** -120)


def _e4m3_values() -> np.ndarray:
    """The value of each e4m3 byte: 1 sign, 4 exponent (bias 7), 3 mantissa bits; 0x7F, 0xFF NaN."""
    out = np.empty(256)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[b] = np.nan if b & 0x7F == 0x7F else (-v if b & 0x80 else v)
    return out


E4M3 = _e4m3_values()


def code_values(stored: np.ndarray, fmt: str) -> np.ndarray:
    """What the stored bytes stand for, before the scale."""
    stored = np.asarray(stored, np.uint8)
    return stored.astype(np.float64) - 128.0 if fmt == "int8" else E4M3[stored]


def _nearest_e4m3(y: np.ndarray) -> np.ndarray:
    y = y.astype(np.float64)
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
    return np.clip(np.sign(y) * np.rint(np.abs(y) / step) * step, -448.0, 448.0)


def hold_block(rows: np.ndarray, fmt: str):
    """(codes as values, scale) of a block's fp32 rows."""
    rows = np.asarray(rows, np.float32)
    if not np.all(np.isfinite(rows)):
        return np.zeros(rows.shape), np.float32(np.nan)
    top = np.abs(rows).max() if rows.size else np.float32(0)
    s = max(np.float32(top / QMAX[fmt]), MIN_SCALE)
    with np.errstate(over="ignore"):
        y = rows * np.float32(np.float32(1.0) / s)
    if fmt == "int8":  # (+ 0: whole numbers have one zero)
        return np.clip(np.rint(y.astype(np.float64)), -127, 127) + 0.0, s
    return _nearest_e4m3(y), s


def hold(rows: np.ndarray, fmt: str, block: int) -> np.ndarray:
    """What a cache holds of the fp32 rows [kv_heads x n x d] (fp32: code * scale)."""
    out = np.empty(rows.shape, np.float32)
    for g in range(rows.shape[0]):
        for b in range(0, rows.shape[1], block):
            codes, s = hold_block(rows[g, b:b + block], fmt)
            out[g, b:b + block] = (codes * np.float64(s)).astype(np.float32)
    return out


def value_at(token: int) -> int:
    """The byte of a chunk's token among the 64 of a dim."""
    h, r = divmod(token, 32)
    p, u, i = 2 * (r // 16) + r % 8 // 4, r % 16 // 8, r % 4
    return 16 * p + 8 * h + 4 * u + i


VALUE_ORDER = np.array([value_at(t) for t in range(64)])


def pack_values(codes: np.ndarray) -> np.ndarray:
    """Bytes [kv x slots x d] in the order the cache holds values."""
    kv, slots, d = codes.shape
    out = np.empty((kv, slots // 64, d, 64), codes.dtype)
    out[..., VALUE_ORDER] = codes.reshape(kv, slots // 64, 64, d).transpose(0, 1, 3, 2)
    return out


def attend(q: np.ndarray, keys: np.ndarray, values: np.ndarray, start: int, heads: int) -> np.ndarray:
    """Causal attention in 64 bits of q [T x heads * d] over [kv x n x d]; rows without keys are zeros."""
    kv, n, d = keys.shape
    t = q.shape[0]
    out = np.zeros((t, heads * d))
    for h in range(heads):
        k, v = (x[h // (heads // kv)].astype(np.float64) for x in (keys, values))
        with np.errstate(invalid="ignore", over="ignore"):
            scores = q[:, h * d:(h + 1) * d].astype(np.float64) @ k.T / np.sqrt(d)
        for i in range(t):
            m = min(start + i + 1, n)
            if m <= 0:
                continue
            with np.errstate(invalid="ignore"):
                p = np.exp(scores[i, :m] - scores[i, :m].max())
                out[i, h * d:(h + 1) * d] = p @ v[:m] / p.sum()
    return out


def largest_score(q: np.ndarray, keys: np.ndarray, heads: int) -> float:
    """The largest magnitude of a score of attend()."""
    kv, _, d = keys.shape
    return max(float(np.abs(q[:, h * d:(h + 1) * d].astype(np.float64) @ keys[h // (heads // kv)].astype(np.float64).T).max()) for h in range(heads)) / np.sqrt(d)


def process_logits(logits, history=None, lengths=None, starts=None, repetition=1.0, frequency=0.0, presence=0.0, biases=(), allowed=None):
    """The controls in 64 bits. history [rows x capacity], biases (token, value) pairs, allowed a
    boolean array [rows x n] or [n]."""
    out = np.asarray(logits, np.float32).astype(np.float64)
    rows, n = out.shape
    biases = dict(biases)
    rep, freq, pres = (float(np.float32(x)) for x in (repetition, frequency, presence))
    for r in range(rows):
        text = [] if history is None else [int(t) for t in history[r][:max(0, min(lengths[r], len(history[r])))]]
        start = 0 if starts is None else int(starts[r])
        for t in set(x for x in text if 0 <= x < n):
            out[r, t] = out[r, t] / rep if out[r, t] > 0 else out[r, t] * rep
        counts: dict[int, int] = {}
        for i, t in enumerate(text):
            if i >= start and 0 <= t < n:
                counts[t] = counts.get(t, 0) + 1
        for t, o in counts.items():
            out[r, t] -= o * freq + pres
        for t, b in biases.items():
            if 0 <= t < n:
                out[r, t] += float(np.float32(b))
    if allowed is not None:
        out[~np.broadcast_to(allowed, out.shape)] = -np.inf
    return out


class HeldTransformer(decoder_ref.RefTransformer):
    """The oracle's decoder with its cache held in 8 bits: a call's tokens attend over the rows as the
    cache holds them after the call's append."""
    fmt = "int8"
    block = 64

    def _layer(self, x: np.ndarray, cache: decoder_ref.RefCache, layer: int) -> np.ndarray:
        c = self.config
        p, start, kv, d = f"block.{layer}.", cache.length, c.num_key_value_heads, c.head_dim
        n = start + x.shape[0]
        normed = oracle.rmsnorm(x, self.norms[p + "norm1"], c.norm_eps)
        q, k, v = (self._project(normed, p + "attention." + w) for w in ("wQ", "wK", "wV"))
        q, k = (oracle.rope_rows(y, d, self.inv_freq, start) for y in (q, k))
        held = []
        for rows, new in ((cache.keys, k), (cache.values, v)):
            rows = rows.reshape(c.num_layers, kv, -1, d)
            rows[layer, :, start:n] = new.reshape(-1, kv, d).transpose(1, 0, 2)
            held.append(hold(rows[layer, :, :n], self.fmt, self.block))
        context = attend(q, held[0], held[1], start, c.num_heads).astype(np.float32)
        x = (x + self._project(context, p + "attention.wOut")).astype(np.float32)
        normed = oracle.rmsnorm(x, self.norms[p + "norm2"], c.norm_eps)
        fused = oracle.silu_mul(self._project(normed, p + "ffn.wGate"), self._project(normed, p + "ffn.wUp"))
        return (x + self._project(fused, p + "ffn.wDown")).astype(np.float32)

    def prefill_chunks(self, prompt, cache: decoder_ref.RefCache, chunk: int) -> np.ndarray:
        for start in range(0, len(prompt), chunk):
            x = self.embed(prompt[start:start + chunk])
            for layer in range(self.config.num_layers):
                x = self._layer(x, cache, layer)
            cache.length += x.shape[0]
        return self._head(x[-1])
