"""A row's output on an 8-bit cache is as precise as its own largest contribution allows, whatever the loudness of
blocks that it hardly attends to or does not see.

Tolerance: test_gpu_kv8 counts six fp32 roundings of a score of magnitude S, each at most 2^-24 S, which move its weight
by their sum; its bound for a whole case, 2^-24 (S + 24), is their root mean square, sqrt(6) * 0.41 * 2^-24 S, over many
rows. Here each row is looked at by itself, and one row's six may all be at their largest (a maximum of 159
powers of two, e^110, plus a shift is off by 2^-17, its weights by 5e-6 = 0.8 * 2^-24 * 110 from this one
rounding): 6 * 2^-24 S. The chain's 24 * 2^-24 stays: 2^-24 (6 S + 24)."""
import numpy as np
import pytest

from gpu_helpers import banner
from oracle import kv8_ref
from test_gpu_kv8 import _attend, _filled

pytestmark = pytest.mark.gpu


def _louden(cache, values, kv, blocks, block, factors):
    """Multiplies the value scales of `blocks` by powers of two; `values` are what the cache then holds."""
    scales = cache.value_scales.download(np.float32).reshape(kv, -1)
    for b, factor in zip(blocks, factors):
        scales[:, b] *= np.float32(factor)
        values[:, b * block:(b + 1) * block] *= factor
    cache.value_scales.upload(scales)


def _check_rows(got, want, q, keys, heads, start):
    kv, _, d = keys.shape
    for t in range(q.shape[0]):
        for h in range(heads):
            s = keys[h // (heads // kv), :start + t + 1] @ q[t, h * d:(h + 1) * d].astype(np.float64) / np.sqrt(d)
            a, b = got[t, h * d:(h + 1) * d].astype(np.float64), want[t, h * d:(h + 1) * d]
            off = np.linalg.norm(a - b) / np.linalg.norm(b)
            assert off <= 2.0 ** -24 * (6.0 * np.abs(s).max() + 24.0), (t, h, off)


@pytest.mark.parametrize("ratio", [12, 20, 28, 35, 60, 100])
@pytest.mark.parametrize("tokens,start,heads,kv,d,fmt,block", [
    (1, 300, 8, 2, 64, "int8", 32), (1, 3000, 8, 2, 64, "e4m3", 64), (1, 700, 4, 2, 128, "int8", 128), (1, 500, 4, 1, 256, "int8", 32),
    (7, 500, 4, 2, 32, "int8", 64), (5, 2000, 4, 2, 128, "e4m3", 32), (600, 100, 32, 8, 64, "int8", 64), (600, 90, 32, 8, 32, "e4m3", 32), (320, 60, 32, 8, 128, "int8", 32)])
def test_a_row_that_attends_to_a_quiet_block(kt, ratio, tokens, start, heads, kv, d, fmt, block):
    """Every other block is 2^ratio louder; each row's query points at one key of a quiet block, whose score is
    110 and the others' at most half of that: a loud block's values times their weight are below 2^ratio e^-55."""
    banner("kv8-loudness", ratio, tokens, start, heads, kv, d, fmt, block)
    rng = np.random.default_rng(tokens + d)
    n = start + tokens
    cache, keys, values = _filled(kt, rng, fmt, block, d, kv, n, n)
    blocks = np.arange((n + block - 1) // block)
    _louden(cache, values, kv, blocks, block, np.where(blocks % 2 == ratio // 4 % 2, 2.0 ** ratio, 1.0))
    q = np.empty((tokens, heads, d), np.float32)
    quiet = np.flatnonzero(np.arange(n) // block % 2 != ratio // 4 % 2)
    for t in range(tokens):
        mine = quiet[quiet <= start + t]
        for h in range(heads):
            k = keys[h // (heads // kv), rng.choice(mine)]
            q[t, h] = k * (110.0 * np.sqrt(d) / (k @ k))
    q = q.reshape(tokens, heads * d)
    some = slice(None) if tokens <= 8 else slice(tokens - 40, tokens)
    first = start if tokens <= 8 else n - 40
    want = kv8_ref.attend(q[some], keys, values, first, heads)
    _check_rows(_attend(kt, cache, 0, q, start, heads)[some], want, q[some], keys, heads, first)


@pytest.mark.parametrize("ratio", [20, 30, 100])
@pytest.mark.parametrize("tokens,start,heads,d,block", [(40, 10, 2, 64, 32), (40, 50, 2, 32, 64), (23, 120, 3, 128, 128), (300, 900, 8, 64, 32)])
def test_a_loud_block_that_a_row_does_not_see(kt, ratio, tokens, start, heads, d, block):
    """Rows before a block in a tile with rows that see it."""
    banner("kv8-unseen", ratio, tokens, start, heads, d, block)
    rng = np.random.default_rng(start)
    n = start + tokens
    cache, keys, values = _filled(kt, rng, "int8", block, d, heads, n, n)
    later = [b for b in range((n + block - 1) // block) if b * block > start]
    _louden(cache, values, heads, later, block, [2.0 ** (ratio * (i + 1) / len(later)) for i in range(len(later))])
    q = rng.standard_normal((tokens, heads * d)).astype(np.float32)
    want = kv8_ref.attend(q, keys, values, start, heads)
    _check_rows(_attend(kt, cache, 0, q, start, heads), want, q, keys, heads, start)


@pytest.mark.parametrize("tokens,start,heads,kv,d", [(1, 900, 4, 2, 64), (1, 5000, 4, 2, 64), (6, 2000, 4, 2, 128), (400, 300, 32, 8, 64)])
def test_blocks_ever_louder_or_quieter(kt, tokens, start, heads, kv, d):
    """Value scales that grow, and that fall, by 2^1.5 a block over 2^100: flat scores, so the loudest block seen
    makes a row; and scores that grow against the loudness, so that several blocks do."""
    rng = np.random.default_rng(d + tokens)
    block, n = 32, start + tokens
    for sign in (1, -1):
        for slope in (0.0, 1.0):
            banner("kv8-slope", tokens, start, sign, slope)
            cache, keys, values = _filled(kt, rng, "int8", block, d, kv, n, n)
            blocks = np.arange((n + block - 1) // block)
            _louden(cache, values, kv, blocks, block, np.exp2(np.clip(np.rint(sign * 1.5 * (blocks - len(blocks) / 2)), -50, 50)))
            q = 0.3 * rng.standard_normal((tokens, heads, d))
            if slope:  # a direction in which the keys' product falls as the loudness grows
                for h in range(heads):
                    k = keys[h // (heads // kv)]
                    along = np.linalg.lstsq(k, -sign * np.arange(n) / block, rcond=None)[0]
                    q[:, h] += slope * along * np.sqrt(d)
            q = q.reshape(tokens, heads * d).astype(np.float32)
            some, first = (slice(None), start) if tokens <= 8 else (slice(tokens - 24, tokens), n - 24)
            want = kv8_ref.attend(q[some], keys, values, first, heads)
            _check_rows(_attend(kt, cache, 0, q, start, heads)[some], want, q[some], keys, heads, first)
