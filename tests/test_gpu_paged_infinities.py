"""Values that are not finite in the cache in pages: the weight of a token that a row sees is above zero, so one infinity makes the row's
context of that dim infinite wherever it lies in the text, infinities of both signs and NaNs make it NaN, and nothing else changes."""
import numpy as np
import pytest

from oracle import paged_ref
from paged_helpers import Batch, random_parents

pytestmark = pytest.mark.gpu

FORMATS = ["float32", "float16", "bfloat16"]
INF = np.inf
# lengths, rows, heads: the forms that the rule on rows, keys and dims takes, with texts that are cut into parts and such that are not
CASES = {
    "steps": ([0, 31, 32, 95, 700, 3000], [1] * 6, (8, 2, 64)),
    "steps 32": ([5, 64, 900], [1] * 3, (6, 6, 32)),
    "steps 128": ([40, 1500], [1] * 2, (4, 2, 128)),
    "steps 256": ([33, 1200], [1] * 2, (4, 1, 256)),
    "few rows": ([100, 1500], [4, 3], (8, 2, 64)),
    "few rows 256": ([100, 700], [2, 4], (4, 1, 256)),
    "few keys": ([30, 60, 0], [50, 68, 33], (8, 2, 64)),
    "some rows": ([900, 64], [15, 9], (8, 2, 64)),
    "some rows 128": ([1300, 64], [15, 9], (4, 1, 128)),
    "many rows": ([0, 300], [150, 33], (8, 2, 64)),
    "many rows 32": ([200, 70], [60, 70], (6, 2, 32)),
    "many rows 128": ([350, 30], [100, 200], (4, 2, 128)),
    "many rows 256": ([200, 10], [60, 90], (2, 1, 256)),
}


def plant(b, bad):
    """bad: (sequence, token, kv head, dim, value); in the pool or among the rows of the call."""
    for s, token, g, d, value in bad:
        if token < b.lengths[s]:
            page, row = b.pool.place(b.tables[s], token)
            b.pool.values[0, page, g, row, d] = paged_ref.to_bits(np.float32([value]), b.fmt)[0]
        else:
            b.v[0, int(b.starts[s]) + token - b.lengths[s], g, d] = value


def check(b, bad):
    plant(b, bad)
    b.upload()
    b.rope_attention()
    got = b.context()
    first = got.tobytes()
    b.append()
    b.check_pool()
    b.rope_attention()
    assert b.context().tobytes() == first
    group = b.heads // b.kv_heads
    special = np.zeros(got.shape)
    hit = np.zeros(got.shape, bool)
    for s, token, g, d, value in bad:
        value = float(paged_ref.stored(np.float32([value]), b.fmt)[0])
        assert not np.isfinite(value)
        rows = int(b.starts[s]) + np.flatnonzero(b.visible(s)[:, token])
        with np.errstate(invalid="ignore"):
            special[rows, g * group:(g + 1) * group, d] += value
        hit[rows, g * group:(g + 1) * group, d] = True
    assert hit.any()
    wrong = np.argwhere(hit & ~((got == special) | (np.isnan(got) & np.isnan(special))))
    assert not wrong.size, [(at.tolist(), got[tuple(at)], special[tuple(at)]) for at in wrong[:5]]
    for s, token, g, d, _ in bad:
        page, row = b.pool.place(b.tables[s], token)
        b.pool.values[0, page, g, row, d] = 0
    want, bound = b.attend(b.rotated())
    want[hit] = got[hit] = 0
    b.check_context(got, want, bound)


def some(b, rng):
    """Infinities and NaNs all over the sequences: first tokens, last ones, the call's own; two of them often in one dim."""
    bad = []
    for s, (length, n) in enumerate(zip(b.lengths, b.counts)):
        total = length + n
        for token in {0, length // 2, length - 1, length, total - 1} | set(rng.integers(0, total, 3).tolist()):
            if token >= 0:
                bad.append((s, int(token), int(rng.integers(0, b.kv_heads)), int(rng.choice([0, 1, 7, b.head_dim // 2, b.head_dim - 1])), float(rng.choice([INF, -INF, np.nan, INF]))))
    return list({at[:4]: at for at in bad}.values())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("case", list(CASES))
def test_forms(kt, fmt, page, tree, case):
    lengths, counts, shape = CASES[case]
    rng = np.random.default_rng(70)
    b = Batch(kt, 70, lengths, counts, shape, fmt, page, parents=random_parents(rng, counts) if tree else None, extra=1, lead=1)
    check(b, some(b, rng))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", ["steps", "steps 256", "few rows", "some rows", "many rows", "many rows 128", "few keys"])
def test_weights_that_fp32_does_not_hold(kt, fmt, case):
    """Keys so loud that most weights are below fp32's smallest number, infinities among their tokens."""
    lengths, counts, shape = CASES[case]
    b = Batch(kt, 71, lengths, counts, shape, fmt, 64, loud=300.0)
    check(b, some(b, np.random.default_rng(71)))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("case", ["steps", "steps 128", "few rows", "some rows", "many rows", "many rows 256"])
@pytest.mark.parametrize("token", [0, 20, -1])
@pytest.mark.parametrize("value", [INF, -INF, np.nan])
def test_one_value(kt, fmt, case, token, value):
    """One value of one token, in a chunk that all rows see and in the last one: the same result."""
    lengths, counts, shape = CASES[case]
    b = Batch(kt, 72, lengths, counts, shape, fmt, 32)
    at = [(s, token % (length + n) if token < 0 else min(token, length + n - 1), 0, 9, value) for s, (length, n) in enumerate(zip(lengths, counts))]
    check(b, at)


@pytest.mark.parametrize("sign", [1, -1])
def test_numbers_that_fp16_does_not_hold(kt, sign):
    """A value of 70000 appended to fp16 pages is an infinity."""
    b = Batch(kt, 73, [50, 0], [40, 30], (8, 2, 64), "float16", 16)
    check(b, [(0, 55, 1, 3, sign * 70000.0), (1, 2, 0, 63, sign * 65520.0)])


@pytest.mark.parametrize("fmt", FORMATS)
def test_bad_pages_hold_nothing_here_too(kt, fmt):
    """Memory that rows do not see is NaN in these tests; a page outside the pool among pages with infinities."""
    b = Batch(kt, 74, [200, 100], [20, 1], (8, 2, 64), fmt, 16)
    bad = [(0, 5, 0, 4, INF), (0, 190, 1, 4, -INF), (1, 99, 0, 4, INF)]
    plant(b, bad)
    b.tables[0, 4], b.tables[1, 0] = -1, b.pool.pages
    check(b, bad)
