"""Draws whose top-p ends exactly between two ids, and the same row drawn alone and among others."""
import numpy as np
import pytest

from tests.test_gpu_sample_rows import SETTINGS, check, draw, logits, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("below", [-np.inf, -70.0])
@pytest.mark.parametrize("vocab", [1000, 16385, 32003, 262144, 300001, (1 << 20) + 3])
@pytest.mark.parametrize("best", [2, 4, 8, 1000, 15000])
def test_borders_among_equals(gpu, best, vocab, below):
    """`best` equal logits, the others masked or without any weight: a quarter, half or three quarters of the row's weight are
    a whole number of ids, or one more where they are not, whatever the logit's size; in one place of the row and
    spread over it, few rows and many."""
    ms = gpu
    say(f"sample_rows: borders among {best} equals of {vocab} ids, the others {below}")
    if best > vocab:
        best = vocab
    rng = np.random.default_rng(best * vocab)
    for rows in (6, 70) if vocab < 1 << 20 else (3,):
        x = np.full((rows, vocab), -np.inf, np.float32)
        at, top_p = [], []
        for r in range(rows):
            top = np.float32(1.0 if r == 0 else 6 * rng.standard_normal())
            x[r] = top + np.float32(below)
            wide = max(100, best)
            near = rng.integers(0, vocab - wide + 1) + np.arange(wide)
            at.append(np.sort(rng.choice(near if r % 2 else vocab, best, replace=False)))
            x[r, at[r]] = top
            top_p.append((0.25, 0.5, 0.75)[r // 2 % 3])
        n = [int(np.ceil(p * best)) for p in top_p]
        j = [int(rng.integers(0, k)) for k in n]
        u = np.array([(i + 0.5) / k for i, k in zip(j, n)], np.float32)
        ids, kept, prob = draw(ms, x, [ms.SampleRow(top_p=p) for p in top_p], u)
        bad = [r for r in range(rows) if (kept[r], ids[r]) != (n[r], at[r][j[r]])]
        assert not bad, (len(bad), bad[0], top_p[bad[0]], kept[bad[0]], n[bad[0]])
        assert np.all(np.abs(prob * n - 1) <= 2.0 ** -23)


@pytest.mark.parametrize("vocab", [5003, 100003, 262144])
def test_alone_and_among_others(gpu, vocab):
    """A row's draw is the same bit for bit whatever rows are beside it: their number decides how rows are cut."""
    ms = gpu
    say(f"sample_rows: rows of {vocab} ids alone and among others")
    rng = np.random.default_rng(vocab)
    R = 66
    x = logits(R, vocab, vocab + 2)
    settings = [SETTINGS[r % len(SETTINGS)] for r in range(R)]
    for r in range(0, R, 3):  # equal logits, more or fewer than a slice's list holds
        some = rng.choice(vocab, (vocab // 8, vocab // 30, 6)[r // 3 % 3], replace=False)
        x[r] = -np.inf
        x[r, some] = np.float32(2 * rng.standard_normal())
        settings[r] = dict(top_p=(0.5, 0.25, 0.9)[r // 9 % 3], min_p=(0.0, 0.3)[r // 27 % 2])
    u = rng.random(R).astype(np.float32)
    rows = [ms.SampleRow(**s) for s in settings]
    many = draw(ms, x, rows, u)
    for r in range(0, R, 1 if vocab < 10000 else 4):
        one = draw(ms, x[r:r + 1], rows[r:r + 1], u[r:r + 1])
        assert all(np.array_equal(a.view(np.int32)[:1], b.view(np.int32)[r:r + 1]) for a, b in zip(one, many)), (r, settings[r])


@pytest.mark.parametrize("size", [90850.0, -90850.0, 1453635.0 / 16, -1453635.0 / 16, 2e5, -2e5])
def test_logits_far_from_zero(gpu, size):
    """Rows some of whose slices lie past 2^17 octaves from 0 and some do not: these weigh as much."""
    say(f"sample_rows: logits about {size}")
    rng = np.random.default_rng(1)
    V = 40000
    settings = [dict(top_p=0.5), dict(top_p=0.9, min_p=0.01), dict(), dict(top_p=0.97), dict(top_k=300, top_p=0.6)] * 3
    x = np.full((len(settings), V), -np.inf, np.float32)
    for r in range(len(settings)):
        x[r, rng.choice(np.arange(20000, 36000), 1000, replace=False)] = size - 3 - rng.integers(0, 3, 1000) * (r % 3)
        x[r, rng.integers(0, 8000)] = size
        if size == 2e5:
            x[r, 38000:38100] = size - 0.5
    check(gpu, x, settings, rng.random(len(settings)).astype(np.float32))
