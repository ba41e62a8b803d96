"""Attention over the cache in pages at scores from small to far above 2^16 powers of two, where a weight's exponent is the difference of rounded
products: queries and keys of small whole numbers, whose scores every format holds exactly, so that only what is said below may be off."""
import numpy as np
import pytest

from oracle import paged_ref
from paged_helpers import Batch
from test_gpu_paged_infinities import CASES

pytestmark = pytest.mark.gpu

FORMATS = ["float32", "float16", "bfloat16"]


def batch(kt, seed, case, fmt, page, keys):
    """A batch whose rotation does nothing, with keys(s, tokens) [tokens x kv heads x dims] for each sequence."""
    lengths, counts, shape = CASES[case]
    b = Batch(kt, seed, lengths, counts, shape, fmt, page)
    b.inv_freq = np.zeros_like(b.inv_freq)
    for s, (length, n) in enumerate(zip(lengths, counts)):
        k = keys(s, length + n).astype(np.float32)
        assert np.array_equal(paged_ref.stored(k, fmt), k)
        for token in range(length):
            page_of, row = b.pool.place(b.tables[s], token)
            b.pool.keys[0, page_of, :, row] = paged_ref.to_bits(k[token], fmt)
        b.k[0, b.sequence_rows(s)] = k[length:]
    return b


def average_of_magnitudes(b):
    """The same attention over the values' magnitudes."""
    out, q = np.zeros(b.q.shape), b.rotated()
    for s in range(len(b.counts)):
        r, see = b.sequence_rows(s), b.visible(s)
        keys, values = (b.pool.rows(w, 0, b.tables[s], range(see.shape[1])) for w in ("keys", "values"))
        out[r] = paged_ref.attend(q[r], keys, np.abs(values), see)[0]
    return out


def largest_value(b):
    values = paged_ref.from_bits(b.pool.values, b.fmt)
    return np.abs(values[np.isfinite(values)]).max()


def run(b):
    b.upload()
    b.rope_attention()
    b.append()
    b.check_pool()
    return b.context()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("order,power", [("any", 10), ("up", 11), ("down", 20), ("any", 40), ("up", 100), ("any", None), ("down", None)])
@pytest.mark.parametrize("case", list(CASES))
def test_one_token_or_equal_ones_have_all_the_weight(kt, fmt, order, power, case):
    """Keys of 1 .. 255 in one dim, a query of +-2^power there (None: another for each row and head): scores are equal or e^64 apart
    and more. What is seen of the largest ones is averaged, whichever chunk, wave and part they lie in. Off by an exponential's 2^-23 in a wave and one in
    each of two merges, a weight's parts, 2^-22, a value's, 2^-24, and quotients, 2^-22, which is below 2^-20 of the largest value; by a sum of n equal
    weights' values, n 2^-24."""
    rng = np.random.default_rng(80)
    shape, ties = CASES[case][2], []

    def keys(s, total):
        level = {"any": rng.integers(1, 256, (total, shape[1])), "up": np.linspace(1, 255, total)[:, None].round() + np.zeros((1, shape[1])),
                 "down": np.linspace(255, 1, total)[:, None].round() + np.zeros((1, shape[1]))}[order]
        ties.append(max(np.unique(level[:, g], return_counts=True)[1].max() for g in range(shape[1])))
        k = np.zeros((total, shape[1], shape[2]))
        k[..., 5] = level
        k[..., 6:] = rng.integers(-9, 10, k[..., 6:].shape)  # (dims that the queries do not have)
        return k

    b = batch(kt, 80, case, fmt, 32, keys)
    b.q[:] = 0
    powers = rng.choice([10, 11, 12, 20, 40, 100], b.q.shape[:2]) if power is None else np.full(b.q.shape[:2], power)
    b.q[..., 5] = np.ldexp(rng.choice([-1.0, 1.0], b.q.shape[:2]), powers)
    assert np.ldexp(1.0, powers.min()) / np.sqrt(shape[2]) >= 64
    got = run(b)
    want, _ = b.attend(b.rotated())
    most = largest_value(b)
    assert np.isfinite(got).all() and np.abs(got - want).max() <= (2.0 ** -20 + max(ties) * 2.0 ** -24) * most


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("base", [0, 1400, 1460, 3000, -1460])
@pytest.mark.parametrize("case", list(CASES))
def test_scores_close_to_each_other(kt, fmt, base, case):
    """Scores base * 250 apart from zero that differ by some powers of two among each other, rising and falling from chunk to chunk: sums of products below
    2^24, so exact ones. A score is rounded once, as it is scaled (2^-24 of itself), and the scale is (three roundings, of the distance of at most 25): a weight is
    off by (|score| + 128) 2^-24 ln 2 and its parts' 2^-22, an average by twice that of the weighted values' magnitudes; sums and quotients add 2^-19. Of 3001 tokens,
    each weight is off by 2^-30 of the largest besides."""
    rng = np.random.default_rng(81)
    shape = CASES[case][2]

    def keys(s, total):
        k = np.zeros((total, shape[1], shape[2]))
        k[..., 3] = 250
        k[..., 4] = (3 * np.sin(np.arange(total) / 40)).round()[:, None] + rng.integers(-3, 4, (total, shape[1]))
        return k

    b = batch(kt, 81, case, fmt, 64, keys)
    b.q[:] = 0
    b.q[..., 3] = base
    b.q[..., 4] = rng.integers(-8, 9, b.q.shape[:2])
    got = run(b)
    scores = abs(base) * 250 + 48
    assert scores < 2 ** 24
    u, bits = 2.0 ** -24, 1.4426950408889634 / np.sqrt(shape[2])
    want, _ = b.attend(b.rotated())
    weighted = average_of_magnitudes(b)
    most = largest_value(b)
    tolerance = (2 * (scores * bits + 128) * u * np.log(2) + 2.0 ** -21 + 2.0 ** -19) * weighted + 3001 * 2.0 ** -30 * most
    off = np.abs(got - want)
    assert (off <= tolerance).all(), (float((off - tolerance).max()), float(off.max()))
