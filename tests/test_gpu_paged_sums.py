"""Attention's sums over the pages where one key outweighs the others: in the probabilities, or in its values' scale."""
import numpy as np
import pytest

from tests.paged_ext_ref import VALUE, SetupExt
from tests.paged_ref import encode

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"\n[case] {msg}", flush=True)


def put(st, k, v):
    """Sequence 0's keys and values."""
    g = st.slots(0, 0, st.len[0])
    for n, x in (("k", k), ("v", v)):
        if st.eight:
            y = st.pool[n].copy()
            y[g] = x
            st.fill(n, y)
        else:
            st.pool[n][g] = encode(x.astype(np.float32), st.dtype)
    st.upload()


@pytest.mark.parametrize("dtype", ["e4m3", "i8", "f32", "bf16", "f16"])
def test_one_key_before_many(gpu, dtype):
    """The first key weighs about as much as the 50,000 to 65,000 behind it, which are all alike, and it alone has a
    value: a row is the first key's share, 1 / (1 + pos e^-c(S)).

    A lane adds up 2048 tiles: sixteen of them, then those sums, each of 16 + 128 additions off by 2^-24 of the sum at
    most; the lanes' and the division, 4.  (All 2048 one after the other lose up to half of the sum's last place
    each, always the same way: 3e-5 of it in the mean, 8e-5 at most.)  The other keys' probability: its distance to
    the first, at most 18.1 in log2, has nine roundings (q times the scale and its factor, three sums, the cap's
    three, the distance), 9 * 18.1 * ln 2 = 113, the exponential 4."""
    say(f"one key before many: {dtype}")
    kv, G, hd, new, n = 2, 2, 64, 16384, 65536
    st = SetupExt(gpu, [(new, n)], kv * G, kv, hd, dtype, 128, cap=1000.0, max_rows=new)
    k, v = np.zeros((n, kv, hd)), np.zeros((n, kv, hd))
    k[0, :, 0], v[0] = 8.0, 1.0
    put(st, k, v)
    q = np.zeros((new, kv * G, hd), np.float32)
    q[:, :, 0] = np.random.default_rng(1).uniform(9.5, 12.5, (new, kv * G))
    got = st.run_attention(q.reshape(new, -1)).reshape(q.shape)
    s = 1000 * np.tanh(q[:, :, 0].astype(np.float64) / 1000)
    others = np.arange(n - new, n)[:, None] * np.exp(-s)
    want = 1 / (1 + others)
    tol = (16 + 128 + 4 + (113 + 4) * others * want) * 2.0 ** -24
    off = np.abs(got / want[..., None] - 1).max(-1)
    assert np.all(off <= tol), (off.max(), (off > tol).mean())


@pytest.mark.parametrize("cap", [0.0, 40.0])
@pytest.mark.parametrize("dtype", ["e4m3", "i8"])
@pytest.mark.parametrize("new,hd,heads,kv", [(1, 64, 4, 4), (1, 128, 8, 2), (3, 128, 8, 1), (1, 512, 8, 2), (6, 256, 4, 1),
                                             (60, 64, 2, 1), (60, 128, 8, 2), (60, 256, 2, 1), (60, 512, 2, 1)])
def test_large_scale_of_no_weight(gpu, new, hd, heads, kv, dtype, cap):
    """A key of no weight whose values' scale is 2^8 to 2^40 times the others': what they weigh keeps its bits,
    wherever the key lies and however the running maximum rises.

    Probabilities times scales come in two fp16 parts: off by 2^-22 of themselves or by half of fp16's smallest step,
    2^-25, in units of 2^-7 of at most twice the largest such product: 2^-31 of that for each key, times its code.
    The other roundings as for any pool (Setup.attend; a score's scale and q's 22 bits are five more)."""
    say(f"a large scale of no weight: {dtype} new={new} hd={hd} cap={cap}")
    n = 300
    st = SetupExt(gpu, [(new, n)], heads, kv, hd, dtype, 16, cap=cap, seed=hd + new)
    rng = np.random.default_rng(7 * hd + new)
    for at, ratio, best in ((1, 40, 0), (0, 16, 200), (37, 28, 5), (n - 61, 20, 100), (130, 12, 130 - 32), (210, 8, 0), (2, 30, 1)):
        k, v = 0.25 * rng.standard_normal((n, kv, hd)), rng.standard_normal((n, kv, hd))
        k[best], k[at] = 1.0, -1.0
        k[20] = 0.4  # (the running maximum rises more than once)
        v[at] *= 2.0 ** ratio
        put(st, k, v)
        q = (1 + 0.1 * rng.standard_normal((new, heads, hd))).astype(np.float32) * np.float32(45 / np.sqrt(hd))
        got = st.run_attention(q.reshape(new, -1)).reshape(q.shape)
        K, V = (st.pool[m][st.slots(0, 0, n)] for m in "kv")
        code, scale = np.abs(VALUE[dtype][st.raw["v"][st.slots(0, 0, n)]]), st.scales["v"].transpose(0, 2, 1)[st.slots(0, 0, n)].astype(np.float64)
        for r in range(new):
            p = n - new + r + 1
            for h in range(heads):
                g = h * kv // heads
                x = K[:p, g] @ q[r, h].astype(np.float64) / np.sqrt(hd)
                d = (hd + 8) * 2.0 ** -24 * (np.abs(K[:p, g]) @ np.abs(q[r, h]).astype(np.float64)).max() / np.sqrt(hd) + 2.0 ** -22
                if cap:
                    x = cap * np.tanh(x / cap)
                    d += 2.0 ** -20 * np.abs(x).max()
                w = np.exp(x - x.max())
                w /= w.sum()
                assert w[at] * 2.0 ** ratio < 2.0 ** -30
                want = w @ V[:p, g]
                tol = 2 * (d + (p + 9) * 2.0 ** -24) * (w @ np.abs(V[:p, g])) + 2.0 ** -31 * (w * scale[:p, g]).max() * code[:p, g].sum(0) + 1e-30
                off = np.abs(got[r, h] - want)
                assert np.all(off <= tol), (at, ratio, r, h, (off / tol).max())


@pytest.mark.parametrize("dtype", ["e4m3", "i8", "f32", "bf16", "f16"])
@pytest.mark.parametrize("seqs,heads,kv,hd", [([(1, 40000), (1, 3)], 3, 1, 64), ([(2, 12000)], 6, 2, 128), ([(1, 9000)], 16, 1, 256),
                                              ([(3, 5000), (1, 1)], 4, 1, 512), ([(1, 131065)], 4, 1, 128), ([(1, 20000)] * 3, 10, 2, 128)])
def test_every_part_counts(gpu, seqs, heads, kv, hd, dtype):
    """Few rows over many keys that all score 0, their values whole numbers of 0 to 16 that turn slowly along the keys: every
    sum is a whole number below 2^24, and exact; a mean is off by its division, 2^-22 of it with room for one more rounding.
    Were 32 keys or more side by side left out, some dim would be off by more."""
    say(f"every part counts: {dtype} {seqs} hd={hd}")
    st = SetupExt(gpu, seqs, heads, kv, hd, dtype, 32, cap=25.0, seed=22)
    n = max(st.len)
    v = ((np.arange(n)[:, None] // max(1, n // 16) + np.arange(hd)) % 17).astype(np.float64)
    for s, length in enumerate(st.len):
        g = st.slots(s, 0, length)
        for name, x in (("k", np.zeros((length, kv, hd))), ("v", np.repeat(v[:length, None], kv, 1))):
            if st.eight:
                code = np.argsort(VALUE[dtype][:128], kind="stable")[np.searchsorted(np.sort(VALUE[dtype][:128]), x)]
                st.raw[name][g] = code.astype(np.uint8)
                st.scales[name].transpose(0, 2, 1)[g] = 1.0
            else:
                st.pool[name][g] = encode(x.astype(np.float32), dtype)
    st.upload()
    q = np.random.default_rng(1).standard_normal((st.rows, heads * hd)).astype(np.float32)
    got = st.run_attention(q).reshape(st.rows, heads, hd)
    upto = np.concatenate([np.zeros((1, hd)), np.cumsum(v, 0)])
    for r, (s, p) in enumerate(st.row_of()):
        want = upto[p + 1] / (p + 1)
        assert np.all(np.abs(got[r] - want) <= 2.0 ** -22 * want)
        at = np.arange(32, p - 63, 32)
        less = (upto[p + 1] - upto[at + 32] + upto[at]) / (p + 1 - 32)
        assert np.all(np.any(np.abs(less - want) > 2.0 ** -20 * want, axis=1))
