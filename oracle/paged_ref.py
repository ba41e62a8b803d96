"""The cache in pages and the trees of drafted tokens, restated in numpy: the cache's roundings as its
formats define them, everything else in 64 bits, with bounds on what fp32 kernels may be off.
"""
from __future__ import annotations

import numpy as np

BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


def to_bits(x: np.ndarray, fmt: str) -> np.ndarray:
    """What the pool stores of fp32 numbers: to the nearest, ties to even."""
    x = np.ascontiguousarray(x, np.float32)
    if fmt == "float32":
        return x
    if fmt == "float16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    rounded = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), rounded)


def from_bits(bits: np.ndarray, fmt: str) -> np.ndarray:
    """The fp32 numbers that stored ones stand for."""
    if fmt == "bfloat16":
        return (bits.astype(np.uint32) << 16).view(np.float32)
    return bits.astype(np.float32)


def stored(x: np.ndarray, fmt: str) -> np.ndarray:
    return from_bits(to_bits(x, fmt), fmt)


def rotate(x: np.ndarray, positions, inv_freq: np.ndarray) -> np.ndarray:
    """Rotary positions on x [rows x heads x d], as the reference rounds them (fp32 steps)."""
    positions = np.asarray(positions)
    half = x.shape[-1] // 2
    angle = (positions.astype(np.float32)[:, None] * inv_freq.astype(np.float32)[None]).astype(np.float64)
    c, s = np.cos(angle).astype(np.float32)[:, None], np.sin(angle).astype(np.float32)[:, None]
    a, b = x[..., :half].astype(np.float32), x[..., half:].astype(np.float32)
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def above(parents) -> list[list[int]]:
    """The rows above each row of one tree, itself last; a parent that is not below its row is none."""
    out: list[list[int]] = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def masks(parents, words: int):
    """(depths, masks) of one tree."""
    paths = above(parents)
    bits = np.zeros((len(paths), words), np.uint32)
    for i, path in enumerate(paths):
        for j in path:
            bits[i, j // 32] |= np.uint32(1 << (j % 32))
    return np.array([len(p) - 1 for p in paths], np.int32), bits


def accept(parents, tokens, chosen) -> list[int]:
    """The rows that the greedy walk keeps."""
    path = [0] if len(parents) else []
    while path:
        follow = [i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and tokens[i] == chosen[path[-1]]]
        if not follow:
            break
        path.append(follow[0])
    return path


def attend(q, keys, values, visible):
    """(context, bound) of rows q [n x heads x d] over keys and values [kv x total x d], all as 64-bit numbers;
    visible [n x total]. bound: what fp32 products and sums may be off, elementwise. With u = 2^-24: a score is a sum
    of d products whose terms are off by 2^-22 of q's largest at most (the coarsest of the formats' parts), so
    by e = ((d + 8) sum|q k| + 4 max|q| sum|k|) u / sqrt(d) + 6 |score| u; a weight relative to its row's largest by 2 e
    and, in the parts, 2^-30; the sums over n keys by (n / 16 + 200) u."""
    n, heads, d = q.shape
    kv, total, _ = keys.shape
    u = 2.0 ** -24
    out, bound = np.zeros((n, heads, d)), np.zeros((n, heads, d))
    for h in range(heads):
        g = h // (heads // kv)
        for i in range(n):
            see = visible[i]
            if not see.any():
                continue
            k, v = keys[g][see].astype(np.float64), values[g][see].astype(np.float64)
            row = q[i, h].astype(np.float64)
            score = k @ row / np.sqrt(d)
            p = np.exp(score - score.max())
            weight = p / p.sum()
            out[i, h] = weight @ v
            e = ((d + 8) * (np.abs(k) @ np.abs(row)) + 4 * np.abs(row).max() * np.abs(k).sum(1)).max() * u / np.sqrt(d) + 6 * np.abs(score).max() * u
            count = int(see.sum())
            bound[i, h] = (4 * e + (count / 16 + 200) * u) * (weight @ np.abs(v)) + count * 2.0 ** -30 * np.abs(v).max(0)
    return out, bound


class Pool:
    """The pool's memory on the host, and the calls' effects on it."""

    def __init__(self, layers, pages, kv_heads, page, head_dim, fmt, fill):
        shape = (layers, pages, kv_heads, page, head_dim)
        self.fmt, self.page, self.kv_heads, self.head_dim, self.pages = fmt, page, kv_heads, head_dim, pages
        self.keys, self.values = to_bits(fill(shape), fmt), to_bits(fill(shape), fmt)

    def place(self, table, token):
        if token < 0 or token >= len(table) * self.page or not 0 <= table[token // self.page] < self.pages:
            return None
        return int(table[token // self.page]), token % self.page

    def rows(self, which, layer, table, tokens) -> np.ndarray:
        """fp32 rows [kv x tokens x d] of a sequence; NaN where a token has no place."""
        memory = getattr(self, which)[layer]
        out = np.full((self.kv_heads, len(tokens), self.head_dim), np.nan, np.float32)
        for i, token in enumerate(tokens):
            at = self.place(table, token)
            if at:
                out[:, i] = from_bits(memory[at[0], :, at[1]], self.fmt)
        return out

    def append(self, layer, table, first, keys, values) -> None:
        """Rows [n x kv x d] from token `first` on."""
        for i in range(keys.shape[0]):
            at = self.place(table, first + i)
            if at:
                self.keys[layer, at[0], :, at[1]] = to_bits(keys[i], self.fmt)
                self.values[layer, at[0], :, at[1]] = to_bits(values[i], self.fmt)

    def keep(self, table, length, kept) -> None:
        for m, r in enumerate(kept):
            source, target = self.place(table, length + r), self.place(table, length + m)
            if source and target:
                for memory in (self.keys, self.values):
                    memory[:, target[0], :, target[1]] = memory[:, source[0], :, source[1]]


def inv_freq(head_dim: int, base: float = 10000.0) -> np.ndarray:
    """RoPE.invFreq without scaling (RoPE.kt:42-46)."""
    return (1.0 / base ** (np.arange(0, head_dim, 2) / head_dim)).astype(np.float32)
