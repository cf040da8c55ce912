"""Token ids drawn for rows of logits on the GPU (temperature, top-k, top-p, min-p), against the definition in
64-bit numbers and whole weights."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"\n[case] {msg}", flush=True)


def weights(x, temperature, n):
    """Whole weights of logits x (64 bits, the largest first)."""
    s = min(49, 63 - (n - 1).bit_length())
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == x[0], 1.0, np.exp((x - x[0]) / np.float64(np.float32(temperature))))
    return w, [int(v) for v in np.rint(np.ldexp(w, s))]


def pick(row, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.5):
    """(id, how many are left, probability, whether a border is nearer than 64 bits of exp can say)."""
    x = row.astype(np.float64)
    order = np.lexsort((np.arange(len(x)), -np.where(np.isnan(x), -np.inf, x)))
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, 0, 0.0, False
    order = order[:1 if temperature == 0 else top_k or len(order)]
    w, whole = weights(x[order], temperature or 1.0, len(x))
    n, close = len(order), False
    upto = np.cumsum(np.array(whole, object))
    if temperature and top_p < 1:
        want = max(1, math.ceil(np.float64(np.float32(top_p)) * np.float64(upto[-1])))
        n = 1 + int(np.searchsorted(upto, want))
        close |= bool(min(abs(float(upto[n - 1]) - want), abs(float(upto[max(n - 2, 0)]) - want)) < 2e-14 * float(upto[-1]))
    low = w >= np.float64(np.float32(min_p))
    low[0] = True
    close |= bool(np.any((np.abs(w - np.float32(min_p)) < 1e-13 * w) & (w < 1))) and min_p > 0
    n = min(n, int(np.count_nonzero(low)))
    left = np.sort(order[:n])
    at = {i: v for i, v in zip(order[:n], whole[:n])}
    upto = np.cumsum(np.array([at[i] for i in left], object))
    u = np.float64(np.float32(u))
    total = upto[-1]
    target = 0 if not u > 0 else total - 1 if u >= 1 else min(int(u * np.float64(total)), total - 1)
    j = int(np.searchsorted(upto, target, side="right"))
    if 0 < u < 1:
        close |= bool(min(abs(float(upto[j]) - u * float(total)), abs(float(upto[max(j - 1, 0)]) - u * float(total))) < 2e-14 * float(total))
    # (weights of 1 are whole numbers without any rounding: every border is exact)
    return int(left[j]), n, at[left[j]] / total, close and not np.all(w == 1)


def draw(ms, x, rows, u, pad=0, prob=True, kept=True):
    R, V = x.shape
    buf = np.full((R, V + pad), 1e30, np.float32)  # (what lies between the rows would win)
    buf[:, :V] = x
    d, du = ms.DeviceBuffer.from_array(buf), ms.DeviceBuffer.from_array(np.asarray(u, np.float32))
    mark = np.full(R + 2, -777, np.int32)
    ids, k, p = (ms.DeviceBuffer.from_array(mark) for _ in range(3))
    ms.sample_rows(d, V + pad, V, rows, du, ids, p if prob else None, k if kept else None)
    ms.synchronize()
    got = [b.download(t, (R + 2,)) for b, t in ((ids, np.int32), (k, np.int32), (p, np.float32))]
    for b, on in zip((ids, k, p), (True, kept, prob)):
        raw = b.download(np.int32, (R + 2,))
        assert np.all(raw[R:] == -777) and (on or np.all(raw == -777))
    assert np.array_equal(d.download(np.float32, buf.shape), buf, equal_nan=True)
    return [g[:R] for g in got]


def check(ms, x, settings, u, pad=0):
    """All rows; ids and counts are those of the definition, probabilities to fp32's rounding and what the weights'
    (2^-44 of the largest, at 2^18 ids) and exp's own leave."""
    rows = [ms.SampleRow(**s) for s in settings]
    ids, kept, prob = draw(ms, x, rows, u, pad)
    far = 0
    for r in range(len(x)):
        i, n, p, close = pick(x[r], **settings[r], u=u[r])
        if close:
            continue
        far += 1
        assert (ids[r], kept[r]) == (i, n), (r, settings[r], u[r], ids[r], kept[r], i, n)
        assert abs(prob[r] - p) <= 2.0 ** -23 * p + 1e-12, (r, prob[r], p)
    assert far >= 0.9 * len(x)
    return ids, kept, prob


SETTINGS = [dict(), dict(temperature=0.7, top_p=0.95), dict(top_k=50), dict(temperature=0.8, top_k=40, top_p=0.9, min_p=0.05),
            dict(temperature=1.2, min_p=0.02), dict(temperature=0.0), dict(temperature=1.5, top_k=1000, top_p=0.6),
            dict(top_p=0.5), dict(temperature=0.05, top_k=64), dict(temperature=30.0, top_p=0.99), dict(top_k=1),
            dict(top_p=0.0), dict(min_p=1.0), dict(top_k=2, min_p=0.5), dict(temperature=1e-30), dict(temperature=1e30, top_k=7),
            dict(top_k=20000, top_p=0.8), dict(top_p=0.9999)]


def logits(R, V, seed, std=2.5):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((R, V)) * std).astype(np.float32)
    few = rng.integers(0, V, (R, min(V, 20)))
    np.put_along_axis(x, few, (6 + 2 * rng.standard_normal(few.shape)).astype(np.float32), 1)
    return x


@pytest.mark.parametrize("vocab,pad", [(1, 0), (2, 1), (63, 0), (64, 0), (65, 3), (1000, 0), (4097, 1), (32003, 2), (262144, 0)])
def test_settings(gpu, vocab, pad):
    say(f"sample_rows: {vocab} ids, every setting")
    R = len(SETTINGS)
    check(gpu, logits(R, vocab, vocab), SETTINGS, np.random.default_rng(vocab + 1).random(R).astype(np.float32), pad)


@pytest.mark.parametrize("vocab,pad", [(262144, 4), (262145, 0), (300001, 2), (1 << 20, 0), ((1 << 20) + 1, 3)])
def test_large_vocabularies(gpu, vocab, pad):
    """Few rows of many ids: small and large slices, rows gone over as a whole, rows at any alignment."""
    say(f"sample_rows: few rows of {vocab} ids")
    settings = [SETTINGS[i] for i in (0, 1, 3, 6, 16)]
    x = logits(len(settings), vocab, vocab)
    x[2, : vocab // 2] = -np.inf  # (slices without any id)
    check(gpu, x, settings, np.random.default_rng(vocab).random(len(settings)).astype(np.float32), pad)


@pytest.mark.parametrize("vocab,shift", [(1250, 0.0), (1700, 0.0), (2300, 0.0), (6000, -1.0), (3000, -30.0), (9000, 0.0), (100003, 0.0)])
def test_top_k_across_zero(gpu, vocab, shift):
    """Cuts far below the largest logit in size, at zero and beyond, by top-k alone and with the others; few ids that can be drawn."""
    say(f"sample_rows: top-k down to logits about zero, {vocab} ids")
    settings = [dict(top_k=k, temperature=t, top_p=p, min_p=m)
                for k in (300, 1000, 1800, 2048) for t, p, m in ((1.5, 0.6, 0.0), (1.0, 1.0, 0.0), (30.0, 0.97, 0.0), (5.0, 1.0, 0.01))]
    rng = np.random.default_rng(vocab)
    x = logits(len(settings), vocab, vocab + 1) + np.float32(shift)
    if shift:
        x[:, 17] = -1e-3  # (the largest logit is the smallest in size)
        x = np.minimum(x, np.float32(-1e-3))
    x[::3][rng.random(x[::3].shape) < 0.3] = -np.inf
    if vocab > 50000:
        x[rng.random(x.shape) < 0.97] = -np.inf
    check(gpu, x, settings, rng.random(len(settings)).astype(np.float32))


def test_flat_large_slices(gpu):
    """More candidates in a slice than it may list."""
    say("sample_rows: flat rows of 300000 ids")
    settings = [dict(), dict(top_p=0.3), dict(top_k=3000), dict(top_k=40, top_p=0.5), dict(temperature=0.0)]
    rng = np.random.default_rng(31)
    x = (1e-6 * rng.integers(0, 3, (len(settings), 300000))).astype(np.float32)
    x[3] = 0.0
    check(gpu, x, settings, rng.random(len(settings)).astype(np.float32))


@pytest.mark.parametrize("std", [0.0, 1e-3, 0.5, 30.0, 1e4])
def test_flat_and_steep(gpu, std):
    """Rows from all alike (only the ids order them) to one far ahead."""
    say(f"sample_rows: logits of spread {std}")
    R, V = len(SETTINGS), 40000
    x = (np.random.default_rng(3).standard_normal((R, V)) * std).astype(np.float32)
    check(gpu, x, SETTINGS, np.random.default_rng(4).random(R).astype(np.float32))


def test_ties(gpu):
    """Few different logits: borders lie among equals, of which the lowest ids stay."""
    say("sample_rows: ties")
    R, V = len(SETTINGS), 30000
    rng = np.random.default_rng(5)
    x = rng.choice(np.array([-3.0, -0.0, 0.0, 1.5, 2.0], np.float32), (R, V))
    check(gpu, x, SETTINGS, rng.random(R).astype(np.float32))
    x = np.where(rng.random((R, V)) < 0.01, np.float32(4), np.float32(4 - 1e-6))
    check(gpu, x, SETTINGS, rng.random(R).astype(np.float32))


@pytest.mark.parametrize("what", ["-inf", "lowest", "nan", "inf", "none", "one"])
def test_masked(gpu, what):
    """Masks of -infinity and of the type's lowest value, NaN, infinities, rows without any id or with one."""
    say(f"sample_rows: {what}")
    R, V = len(SETTINGS), 5003
    rng = np.random.default_rng(6)
    x = logits(R, V, 7)
    off = rng.random((R, V)) < 0.9
    if what == "-inf":
        x[off] = -np.inf
    elif what == "lowest":
        x[off] = np.finfo(np.float32).min
    elif what == "nan":
        x[off] = np.nan
    elif what == "inf":
        x[rng.random((R, V)) < 0.01] = np.inf
        x[off & (x != np.inf)] = -np.inf
    else:
        x[:] = np.where(rng.random((R, V)) < 0.5, -np.inf, np.nan)
        if what == "one":
            x[np.arange(R), rng.integers(0, V, R)] = rng.standard_normal(R) * 100
    ids, kept, prob = check(gpu, x, SETTINGS, rng.random(R).astype(np.float32))
    if what == "none":
        assert np.all(ids == -1) and np.all(kept == 0) and np.all(prob == 0)


def test_random_numbers(gpu):
    """u at its ends and outside them."""
    say("sample_rows: random numbers")
    u = np.array([0, -1, np.nan, -np.inf, 2.0 ** -149, 1 - 2.0 ** -24, 1, 7, np.inf, 0.5], np.float32)
    x = np.repeat(logits(1, 2000, 8), len(u), 0)
    for s in (dict(), dict(top_k=30), dict(top_p=0.7)):
        ids, kept, _ = check(gpu, x, [s] * len(u), u)
        assert len(set(ids[:5])) == 1 and len(set(ids[6:9])) == 1


def test_many_rows(gpu):
    """More rows than a launch takes, and the same twice: bit for bit; without the optional results."""
    ms = gpu
    say("sample_rows: 300 rows")
    R, V = 300, 777
    x, u = logits(R, V, 9), np.random.default_rng(10).random(R).astype(np.float32)
    settings = [SETTINGS[r % len(SETTINGS)] for r in range(R)]
    a = check(ms, x, settings, u, pad=5)
    rows = [ms.SampleRow(**s) for s in settings]
    b = draw(ms, x, rows, u)
    assert all(np.array_equal(p.view(np.int32), q.view(np.int32)) for p, q in zip(a, b))
    for prob in (False, True):
        assert np.array_equal(draw(ms, x, rows, u, prob=prob, kept=not prob)[0], a[0])
    assert np.array_equal(draw(ms, x[:0], [], u[:0])[0], np.zeros(0, np.int32))


def test_frequencies(gpu):
    """Over evenly spread u each id comes as often as its probability says, to one draw."""
    ms = gpu
    say("sample_rows: frequencies")
    n = 4000
    row = np.array([1.0, 0.5, -2.0, 3.0, 2.9, -np.inf, 0.0], np.float32)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    ids, _, _ = draw(ms, np.repeat(row[None], n, 0), [ms.SampleRow(0.9, 4, 1.0, 0.0)] * n, u)
    w = np.exp((row.astype(np.float64) - 3) / np.float64(np.float32(0.9)))
    w[np.argsort(-row, kind="stable")[4:]] = 0
    want = n * w / w.sum()
    assert np.all(np.abs(np.bincount(ids, minlength=7) - want) <= 1.01)


def test_buffers_side_by_side(gpu):
    """Refused on the host: results over the logits or each other are the caller's; what must be refused is."""
    ms = gpu
    say("sample_rows: refused")
    d = ms.DeviceBuffer(4096)
    lib, p, one = ms.lib(), d.ptr, (ms.SampleRow * 1)(ms.SampleRow())
    good = dict(x=p, ld=100, n=1, v=100, r=one, u=p + 1024, ids=p + 2048)
    for change in (dict(x=None), dict(r=None), dict(u=None), dict(ids=None), dict(ld=99), dict(n=-1), dict(v=0)):
        a = {**good, **change}
        assert lib.ms_sample_rows(a["x"], a["ld"], a["n"], a["v"], a["r"], a["u"], a["ids"], None, None) == -1, change
