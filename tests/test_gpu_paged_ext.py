"""8-bit paged pools, normed heads, both rotations and capped scores on the GPU: append, read and attention
against 64 bits, at the sizes, masks and contents where they can go wrong."""
import ctypes as C

import numpy as np
import pytest

from tests.paged_ext_ref import E4M3, HALF, MAX32, VALUE, SetupExt, append_in_64, decode, nearest, scale_of
from tests.paged_ref import encode

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"\n[case] {msg}", flush=True)


def f32(*shape, seed=0, scale=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * scale).astype(np.float32)


class At:
    def __init__(self, b, off):
        self.ptr = b.ptr + 4 * off


# ---- append ------------------------------------------------------------------------
APPENDS = [
    # seqs (new, length), heads, kv, hd, rot, page, page_rows, norm, gamma, pairs
    ([(1, 1)], 8, 2, 64, 64, 16, 0, 7, True, False),
    ([(1, 301), (0, 17), (1, 16), (1, 17), (0, 0)], 40, 8, 128, 128, 16, 0, 3, True, False),
    ([(33, 33), (1, 5), (70, 135)], 8, 2, 512, 128, 24, 60, 3, True, True),
    ([(5, 9)], 5, 1, 256, 0, 1, 1, 4, False, False),
    ([(7, 7), (2, 64)], 6, 3, 64, 2, 7, 9, 2, False, True),
    ([(9, 40)], 4, 4, 128, 126, 32, 32, 1, True, False),
    ([(300, 1000)], 2, 2, 256, 256, 128, 0, 0, False, True),
    ([(3, 20)], 3, 1, 512, 254, 16, 0, 7, True, True),
    ([(6, 6)], 2, 2, 256, 6, 8, 0, 7, True, False),
]


@pytest.mark.parametrize("dtype", ["e4m3", "i8", "f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(gpu, case, dtype):
    """q and the pools' values within what fp32 may be off; 8-bit codes and scales those of 64 bits; every other
    slot keeps its bits.  q, k and v side by side, apart, or no q, by case."""
    ms = gpu
    seqs, heads, kv, hd, rot, page, pr, norm, gamma, pairs = APPENDS[case]
    how = ("fused", "apart", "kv")[case % 3]
    say(f"append {dtype} {APPENDS[case]} {how}")
    st = SetupExt(ms, seqs, heads, kv, hd, dtype, page, pr, rot=rot, norm=norm, gamma=gamma, pairs=pairs, seed=case)
    nq, nkv, n_pos = heads * hd, kv * hd, max(st.len)
    c, s = ms.rope_table(rot, 1e4, n_pos, wide=True) if rot else (None, None)
    ms.synchronize()
    hc, hs = (t.download(np.float32, (n_pos, rot // 2)) if rot else None for t in (c, s))
    x = f32(st.rows + 2, nq + 2 * nkv + 4, seed=case + 50) * np.exp2(3 * f32(st.rows + 2, 1, seed=case))
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:nq + 2 * nkv]
    ld = x.shape[1]
    d = ms.DeviceBuffer.from_array(x)
    out = ms.DeviceBuffer.from_array(np.full((st.rows + 2, nq + 8), -777, np.float32))
    before = st.download8() if st.eight else st.download()
    if how == "fused":
        ms.paged_append(st.layer, st.batch, At(d, nq), At(d, nq + nkv), ld, d, ld, d, ld, c, s, n_pos)
        got_q = d.download(np.float32, x.shape)
        assert np.array_equal(got_q[st.rows:], x[st.rows:]) and np.array_equal(got_q[:, nq:], x[:, nq:])
    elif how == "apart":
        ms.paged_append(st.layer, st.batch, At(d, nq), At(d, nq + nkv), ld, d, ld, out, nq + 8, c, s, n_pos)
        got_q = out.download(np.float32, (st.rows + 2, nq + 8))
        assert np.all(got_q[st.rows:] == -777) and np.all(got_q[:, nq:] == -777)
    else:
        ms.paged_append(st.layer, st.batch, At(d, nq), At(d, nq + nkv), ld, cos=c, sin=s, n_pos=n_pos)
    ms.synchronize()
    (wq, wk, wv), (tq, tk, tv) = append_in_64(st, q[:st.rows], k[:st.rows], v[:st.rows], hc, hs)
    if how != "kv":
        assert np.all(np.abs(got_q[:st.rows, :nq].reshape(wq.shape) - wq) <= tq + 1e-37)
    for n, w, t in (("k", wk, tk), ("v", wv, tv)):
        if st.eight:
            codes, scales = st.download8()
            for r, (sq, p) in enumerate(st.row_of()):
                pg, sl = st.pages[sq, p // page], p % page
                want_s = scale_of(w[r], dtype)
                # (64-bit sums in another order: the last bit of a scale may be another)
                assert np.all(np.abs(scales[n][pg, :, sl] / want_s - 1) <= 2.0 ** -23)
                if not (norm >> (1 if n == "k" else 2) & 1) and not (n == "k" and rot):
                    assert np.array_equal(scales[n][pg, :, sl], want_s)
                want_c, near = nearest(w[r] / scales[n][pg, :, sl, None].astype(np.float64), dtype)
                got_c = codes[n][pg, sl]
                same = VALUE[dtype][got_c] == VALUE[dtype][want_c]
                assert np.all(same | near) and near.mean() < 0.01
                before[0][n][pg, sl], before[1][n][pg, :, sl] = got_c, scales[n][pg, :, sl]
            assert np.array_equal(codes[n], before[0][n])
            assert np.array_equal(scales[n].view(np.uint32), before[1][n].view(np.uint32))
        else:
            got = st.download()[n]
            half = HALF[dtype] if dtype != "f32" else 0.0
            tiny = {"f32": 1e-37, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}[dtype]
            for r, (sq, p) in enumerate(st.row_of()):
                at = (st.pages[sq, p // page], p % page)
                g = decode(got[at], dtype)
                assert np.all(np.abs(g - w[r]) <= (1 + half) * t[r] + half * np.abs(w[r]) + tiny)
                before[n][at] = got[at]
            assert np.array_equal(got.view(np.uint8), before[n].view(np.uint8))


@pytest.mark.parametrize("dtype", ["e4m3", "i8"])
def test_append_roundings(gpu, dtype):
    """Every code, every middle between two and its neighbours, with a scale of 1 and of 3: the nearest
    code, even where two are as near."""
    ms = gpu
    say(f"append: roundings of {dtype}")
    v = np.sort(np.unique(VALUE[dtype][np.isfinite(VALUE[dtype]) & (np.abs(VALUE[dtype]) <= (448 if dtype == "e4m3" else 127))]))
    mid = (v[1:] + v[:-1]) / 2
    x = np.concatenate([v, mid, np.nextafter(mid.astype(np.float32), np.float32(1e9)),
                        np.nextafter(mid.astype(np.float32), np.float32(-1e9))]).astype(np.float32)
    top = np.float32(448 if dtype == "e4m3" else 127)
    hd = 64
    rows = -(-len(x) // (hd - 1))
    x = np.concatenate([x, np.zeros(rows * (hd - 1) - len(x), np.float32)]).reshape(rows, hd - 1)
    x = np.concatenate([x, np.full((rows, 1), top)], 1)
    for scale in (1.0, 3.0, 2.0 ** -100):
        st = SetupExt(ms, [(rows, rows)], 1, 1, hd, dtype, 16)
        y = (x * np.float32(scale)).astype(np.float32)
        d = ms.DeviceBuffer.from_array(y)
        ms.paged_append(st.layer, st.batch, d, d, hd)
        ms.synchronize()
        codes, scales = st.download8()
        g = st.slots(0, 0, rows)
        for n in "kv":
            assert np.all(scales[n][g[0], 0, g[1]] == np.float32(scale))
            want, _ = nearest(y.astype(np.float64) / scale, dtype)
            got = codes[n][g][:, 0]
            assert np.array_equal(VALUE[dtype][got], VALUE[dtype][want])
    assert np.array_equal(E4M3[:127], np.sort(E4M3[:127]))


@pytest.mark.parametrize("dtype", ["e4m3", "i8"])
def test_append_special_values(gpu, dtype):
    """A head with a value that is not finite gets NaN as its scale and reads back as NaN, alone; zeros stay zeros;
    the smallest and largest magnitudes keep their signs and sizes."""
    ms = gpu
    say(f"append: special values, {dtype}")
    st = SetupExt(ms, [(6, 6)], 2, 2, 64, dtype, 4)
    x = f32(6, 2, 64, seed=1)
    x[0, 0, 3], x[0, 1, 5], x[1, 0, 63] = np.nan, np.inf, -np.inf
    x[2] = 0
    x[3, 0] = np.sign(x[3, 0]) * 2.0 ** -149
    x[3, 1] *= 1e-40
    x[4] = np.sign(x[4]) * np.float32(MAX32)
    d = ms.DeviceBuffer.from_array(x)
    ms.paged_append(st.layer, st.batch, d, d, 128)
    out = ms.DeviceBuffer(2 * 6 * 128 * 4)
    ms.paged_read(st.layer, st.batch, 0, 0, 6, out, At(out, 6 * 128), 128)
    ms.synchronize()
    for got in out.download(np.float32, (2, 6, 2, 64)):
        bad = ~np.isfinite(x).all(-1)
        assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
        assert np.all(got[2] == 0)
        s = scale_of(x[~bad].astype(np.float64), dtype)[:, None].astype(np.float64)
        # half a step: an eighth of the value by two (at least 2^-10), or half a whole number
        half = np.maximum(np.abs(x[~bad]) * 2.0 ** -4, s * 2.0 ** -10) if dtype == "e4m3" else 0.5 * s
        assert np.all(np.abs(got[~bad] - x[~bad].astype(np.float64)) <= half * (1 + 1e-6))


@pytest.mark.parametrize("dtype", ["e4m3", "i8"])
@pytest.mark.parametrize("pairs", [False, True])
def test_append_past_the_range(gpu, dtype, pairs):
    """Rotations and gammas that lead past fp32's largest number, or to it."""
    ms = gpu
    say(f"append: past the range, {dtype} pairs={pairs}")
    st = SetupExt(ms, [(4, 4)], 2, 2, 64, dtype, 4, rot=64, pairs=pairs)
    x = f32(4, 2, 64, seed=3)
    x[0] = MAX32                            # sqrt 2 of it
    x[1] *= np.float32(0.7 * MAX32) / np.abs(x[1]).max()
    x[2] = np.float32(0.72 * MAX32)
    x[2, 0, ::2], x[2, 0, 1::2] = 0, 0      # (zeros beside a head that is past it)
    x[3] = -np.float32(0.707 * MAX32)
    cs = np.full((4, 32), np.float32(np.sqrt(0.5)))
    d, c = ms.DeviceBuffer.from_array(x), ms.DeviceBuffer.from_array(cs)
    ms.paged_append(st.layer, st.batch, d, d, 128, cos=c, sin=c, n_pos=4)
    ms.synchronize()
    codes, scales = st.download8()
    (_, wk, wv), _ = append_in_64(st, np.zeros((4, 2, 64)), x, x, cs, cs)
    seen = []
    for n, w in (("k", wk), ("v", wv)):
        for r, (sq, p) in enumerate(st.row_of()):
            pg, sl = st.pages[sq, p // 4], p % 4
            s, want = scales[n][pg, :, sl], scale_of(w[r], dtype)
            assert np.array_equal(np.isnan(s), np.isnan(want)) and np.all(np.isnan(s) | (np.abs(s / want - 1) <= 2.0 ** -23))
            c_, near = nearest(w[r] / np.where(np.isnan(s), 1e300, s.astype(np.float64))[:, None], dtype)
            ok = (VALUE[dtype][codes[n][pg, sl]] == VALUE[dtype][c_]) | near | np.isnan(s)[:, None]
            assert ok.all()
            seen += np.isnan(s).tolist()
    assert 0 < sum(seen) < len(seen)


def test_append_tiny_norms(gpu):
    """Heads of the smallest numbers under a norm without eps: their inverse is past fp32's range, the result is not."""
    ms = gpu
    say("append: norms of tiny heads")
    for dtype in ("f32", "bf16", "e4m3"):
        st = SetupExt(ms, [(3, 3)], 2, 2, 128, dtype, 4, norm=7, eps=0.0)
        x = (f32(3, 2, 128, seed=4).astype(np.float64) * np.array([1e-40, 1e-30, 1e37])[:, None, None]).astype(np.float32)
        d, o = ms.DeviceBuffer.from_array(x), ms.DeviceBuffer(3 * 256 * 4)
        ms.paged_append(st.layer, st.batch, d, d, 256, d, 256, o, 256)
        ms.synchronize()
        (wq, wk, wv), (tq, _, _) = append_in_64(st, x, x, x, None, None)
        assert np.all(np.abs(o.download(np.float32, x.shape) - wq) <= tq) and np.all(np.isfinite(wq))
        got = st.download8() if st.eight else st.download()
        for r, (sq, p) in enumerate(st.row_of()):
            pg, sl = st.pages[sq, p // 4], p % 4
            for n, w in (("k", wk), ("v", wv)):
                g = VALUE[dtype][got[0][n][pg, sl]] * got[1][n][pg, :, sl, None].astype(np.float64) if st.eight else decode(got[n][pg, sl], dtype)
                step = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "e4m3": 2.0 ** -4}[dtype]
                least = np.abs(w[r]).max() / 448 * 2.0 ** -10 if st.eight else 0.0
                assert np.all(np.abs(g - w[r]) <= (step + 4 * 2.0 ** -24) * np.abs(w[r]) + least * 1.001)


def test_append_norm_sizes(gpu):
    """Norms of very small and very large rows, and of zeros: the squares neither vanish nor overflow."""
    ms = gpu
    say("append: sizes of normed rows")
    for eps in (1e-6, 0.0):
        st = SetupExt(ms, [(5, 5)], 2, 1, 128, "f32", 16, norm=7, eps=eps)
        x = f32(5, 4 * 128, seed=3) + 0.5
        x[1] *= 1e30
        x[2] *= 1e-30
        x[3] = 0
        x[4, 5] = np.nan
        d = ms.DeviceBuffer.from_array(x)
        ms.paged_append(st.layer, st.batch, At(d, 256), At(d, 384), 512, d, 512, d, 512)
        ms.synchronize()
        (wq, wk, wv), (tq, tk, tv) = append_in_64(st, x[:, :256], x[:, 256:384], x[:, 384:], None, None)
        got = d.download(np.float32, x.shape)[:, :256].reshape(wq.shape)
        pool = st.download()
        g = st.slots(0, 0, 5)
        for a, w, t in ((got, wq, tq), (pool["k"][g], wk, tk), (pool["v"][g], wv, tv)):
            assert np.array_equal(np.isnan(a), np.isnan(w))
            ok = np.isfinite(w)
            assert np.all(np.abs(a[ok] - w[ok]) <= t[ok] + 1e-37)
            assert np.isnan(w[3]).all() == (eps == 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_plain_is_append(gpu, dtype):
    """Without norms, pairs or 8 bits the call is ms_paged_append, bit for bit."""
    ms = gpu
    say(f"append_ext as append, {dtype}")
    a, b = (SetupExt(ms, [(9, 20), (1, 4)], 4, 2, 64, dtype, 16, rot=32, seed=4) for _ in range(2))
    c, s = ms.rope_table(32, 1e4, 20)
    x = f32(10, 8 * 64, seed=5)
    got = []
    for st, layer in ((a, a.layer), (b, b.layer.base)):
        d = ms.DeviceBuffer.from_array(x)
        ms.paged_append(layer, st.batch, At(d, 256), At(d, 384), 512, d, 512, d, 512, c, s, 20)
        ms.synchronize()
        got.append([d.download(np.uint8, (x.nbytes,))] + [p.view(np.uint8) for p in st.download().values()])
    assert all(np.array_equal(p, q) for p, q in zip(*got))


# ---- read ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["e4m3", "i8", "f32", "bf16", "f16"])
@pytest.mark.parametrize("kv,hd,page,pr", [(1, 64, 16, 0), (3, 128, 7, 9), (2, 512, 1, 1), (8, 256, 128, 130)])
def test_read(gpu, dtype, kv, hd, page, pr):
    """A code's value times its scale, rounded once; rows behind and columns between keep what they held."""
    ms = gpu
    say(f"read {dtype} kv={kv} hd={hd} page={page}")
    st = SetupExt(ms, [(1, 33), (0, 300), (2, 2)], kv, kv, hd, dtype, page, pr, seed=6, spread=4.0)
    for seq, p0, n, pad, which in ((0, 0, 33, 0, "kv"), (1, 5, 290, 4, "kv"), (1, 299, 1, 0, "k"), (2, 0, 2, 8, "v"),
                                   (1, 300, 0, 0, "kv"), (1, 17, 3, 0, "kv")):
        ld = kv * hd + pad
        buf = {x: ms.DeviceBuffer.from_array(np.full((n + 2, ld), -777, np.float32)) for x in "kv"}
        ms.paged_read(st.layer, st.batch, seq, p0, n, buf["k"] if "k" in which else None,
                      buf["v"] if "v" in which else None, ld)
        ms.synchronize()
        for x in "kv":
            got = buf[x].download(np.float32, (n + 2, ld))
            assert np.all(got[n:] == -777) and np.all(got[:, kv * hd:] == -777)
            if x in which:
                want = decode(st.pool[x][st.slots(seq, p0, p0 + n)], st.dtype).reshape(n, kv * hd)
                assert np.array_equal(got[:n, :kv * hd], want.astype(np.float32))
            else:
                assert np.all(got == -777)


@pytest.mark.parametrize("dtype", ["i8", "bf16"])
def test_read_many(gpu, dtype):
    """More rows than the caches hold, and half of them."""
    ms = gpu
    say(f"read of 138 MB, {dtype}")
    kv, hd, n = 8, 512, 4200
    st = SetupExt(ms, [(0, n)], kv, kv, hd, dtype, 128, seed=8, max_rows=1)
    buf = {x: ms.DeviceBuffer.from_array(np.full((n + 1, kv * hd), -777, np.float32)) for x in "kv"}
    for which in ("k", "kv"):
        ms.paged_read(st.layer, st.batch, 0, 0, n, buf["k"], buf["v"] if "v" in which else None, kv * hd)
        ms.synchronize()
        for x in "kv":
            got = buf[x].download(np.float32, (n + 1, kv * hd))
            assert np.all(got[n:] == -777)
            want = decode(st.pool[x][st.slots(0, 0, n)], st.dtype).reshape(n, -1).astype(np.float32)
            assert np.array_equal(got[:n], want) if x in which else np.all(got == -777)


# ---- attention -------------------------------------------------------------------------
ATTENDS = [
    # seqs, heads, kv, hd, page, page_rows, window
    ([(1, 1)], 8, 2, 512, 16, 0, 0),                                     # one key
    ([(1, 700)], 8, 2, 512, 16, 0, 0),                                   # split over the keys
    ([(1, 33), (1, 1), (0, 9), (1, 2048), (1, 31), (1, 32), (0, 0), (1, 65)], 40, 8, 128, 16, 0, 0),
    ([(1, 5000)], 8, 2, 256, 32, 0, 512),                                # sliding
    ([(1, 300), (1, 100)], 5, 5, 64, 24, 30, 40),
    ([(17, 17)], 8, 2, 256, 16, 0, 0),                                   # a prompt
    ([(100, 260)], 40, 8, 128, 64, 0, 0),                                # a chunk
    ([(70, 200), (1, 90), (3, 3), (0, 50), (33, 500)], 8, 2, 512, 32, 0, 0),
    ([(130, 700), (40, 40)], 8, 2, 256, 7, 11, 64),                      # sliding chunks, odd pages
    ([(37, 41)], 16, 1, 64, 1, 0, 5),                                    # pages of one slot
    ([(2, 640)], 20, 1, 128, 128, 0, 1),                                 # a window of one: v itself
    ([(4, 1500)], 4, 1, 128, 16, 0, 0),                                  # exactly 16 (row, head) pairs
    ([(9, 1111)], 8, 1, 64, 16, 0, 0),
    ([(250, 250)], 3, 3, 64, 32, 0, 100),
    ([(5, 300), (8, 8), (1, 40)], 8, 2, 256, 16, 0, 0),                  # 17 to 32 pairs
    ([(5, 300), (8, 8)], 8, 2, 128, 16, 0, 33),
    ([(7, 500), (1, 77)], 4, 1, 64, 32, 0, 0),
    ([(4, 90)], 16, 2, 512, 16, 0, 0),
    ([(1, 9000)], 4, 1, 128, 64, 0, 0),                                  # many parts of one result
    ([(40, 3001)], 8, 1, 512, 16, 0, 0),                                 # chunks over split keys
    ([(200, 4100)], 4, 1, 128, 16, 0, 0),
    ([(90, 400), (33, 33)], 4, 2, 128, 16, 0, 70),
    ([(129, 129)], 1, 1, 256, 16, 0, 0),                                 # one pair past a block's
]


@pytest.mark.parametrize("dtype", ["e4m3", "i8"])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention(gpu, case, dtype):
    seqs, heads, kv, hd, page, pr, window = ATTENDS[case]
    cap = 3.0 if (case + (dtype == "i8")) % 2 else 0.0
    say(f"attention {dtype} cap={cap} {ATTENDS[case]}")
    st = SetupExt(gpu, seqs, heads, kv, hd, dtype, page, pr, window, cap=cap, seed=case)
    st.check(pad=4 * (case % 3))


@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention_capped(gpu, case):
    """Capped scores over the other pools, near the cap and far below it."""
    seqs, heads, kv, hd, page, pr, window = ATTENDS[case]
    dtype, cap = ("f32", "bf16", "f16")[case % 3], (2.0, 50.0)[case // 3 % 2]
    say(f"attention {dtype} cap={cap} {ATTENDS[case]}")
    st = SetupExt(gpu, seqs, heads, kv, hd, dtype, page, pr, window, cap=cap, seed=case)
    st.check(pad=4 * (case % 3), scale=3.0)


@pytest.mark.parametrize("dtype", ["e4m3", "i8", "bf16", "f16"])
@pytest.mark.parametrize("new,hd", [(1, 64), (3, 128), (40, 128), (30, 512)])
def test_attention_cap_far_from_scores(gpu, new, hd, dtype):
    """Scores far past any cap, or far below it, among scores of 0."""
    say(f"attention, cap and scores far apart: {dtype} new={new} hd={hd}")
    st = SetupExt(gpu, [(new, 150)], 4, 2, hd, dtype, 16, cap=1.0, seed=24)
    g = [i[::2] for i in st.slots(0, 0, 150)]
    (st.raw if st.eight else st.pool)["k"][tuple(g)] = 0
    st.upload()
    for cap in (2.0 ** -60, 1.0, 2.0 ** 60):
        st.cap = st.layer.score_cap = cap
        for scale in (2.0 ** 90, 2.0 ** -90):
            q, got = st.check(scale=scale)
            assert np.all(np.isfinite(got))
            if scale < 1 or cap < 1:  # (scores of 0 to fp32: the values' mean; tanh of +-infinity times the least cap, too)
                v = decode(st.pool["v"][st.slots(0, 0, 150)], dtype)
                want = (np.cumsum(v, 0) / np.arange(1, 151)[:, None, None])[150 - new:]
                want = np.repeat(want, 2, 1).reshape(new, -1)
                # (a probability off by 2^-22, 160 rounded sums, the division)
                assert np.all(np.abs(got - want) <= 2 * (2.0 ** -22 + 160 * 2.0 ** -24) * np.abs(v).max())


@pytest.mark.parametrize("dtype", ["e4m3", "i8", "f32", "bf16", "f16"])
def test_attention_cap_of_later_keys(gpu, dtype):
    """Rows of small scores keep their bits where keys behind them are past the cap."""
    say(f"attention, later keys past the cap: {dtype}")
    heads, n = 16, 40
    st = SetupExt(gpu, [(n, n)], heads, 1, 64, dtype, 16, cap=50.0, seed=25)
    g = st.slots(0, 0, n)
    k, v = np.zeros((n, 1, 64)), np.zeros((n, 1, 64))
    k[:, 0, 0] = 448.0
    k[0, 0, 0], k[1, 0, 0] = 1.0, -1.0
    v[:, 0, 0] = 1.0
    v[1, 0, 0] = -1.0
    for name, x in (("k", k), ("v", v)):
        if st.eight:
            y = st.pool[name].copy()
            y[g] = x
            st.fill(name, y)
        else:
            st.pool[name][g] = encode(x.astype(np.float32), dtype)
    st.upload()
    q = np.zeros((n, heads, 64), np.float32)
    q[:, :, 0] = 1.7 + 0.137 * np.arange(heads)  # scores 0.2 to 0.5 in size, of later keys 95 to 210
    got = st.run_attention(q.reshape(n, -1)).reshape(n, heads, 64)[1, :, 0]
    s = q[1, :, 0].astype(np.float64) / 8
    want = np.tanh(50 * np.tanh(s / 50))
    # scores of half a unit in log2, four roundings; their distance to the maximum, one; two powers of 2^-22; the sums
    # and the division, four: below 2^-24 (4 + 2 + 8 + 4)
    assert np.all(np.abs(got - want) <= 18 * 2.0 ** -24), np.abs(got - want).max()


@pytest.mark.parametrize("dtype,hd,kv,G,rows,cap", [
    ("e4m3", 512, 32, 2, 320, 0.0), ("i8", 128, 64, 1, 1280, 20.0), ("bf16", 512, 32, 2, 290, 20.0), ("e4m3", 64, 64, 2, 641, 5.0)])
def test_attention_last_turn(gpu, dtype, hd, kv, G, rows, cap):
    """Chunks whose blocks are all busy more than once, the last time few of them: some rows' keys are cut, others not."""
    say(f"attention, a short last turn: {dtype} hd={hd} {rows} rows")
    st = SetupExt(gpu, [(rows, rows + 1200)], kv * G, kv, hd, dtype, 64, cap=cap, seed=21)
    st.check(only=(0, 1, 17, 31, 63, 64, 100, 127, 128, rows // 2, rows - 33, rows - 1))


@pytest.mark.parametrize("dtype", ["e4m3", "i8", "f32", "bf16", "f16"])
@pytest.mark.parametrize("seqs,heads,kv,hd", [([(1, 40000), (1, 3)], 3, 1, 64), ([(2, 12000)], 6, 2, 128), ([(1, 9000)], 16, 1, 256),
                                              ([(3, 5000), (1, 1)], 4, 1, 512)])
def test_attention_many_parts(gpu, seqs, heads, kv, hd, dtype):
    """Few rows over many keys, whose parts are merged by several blocks."""
    say(f"attention, many parts: {dtype} {seqs} hd={hd}")
    st = SetupExt(gpu, seqs, heads, kv, hd, dtype, 32, cap=25.0, seed=22)
    st.check()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("dtype", ["e4m3", "i8", "f32", "bf16", "f16"])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_attention_every_kernel(gpu, new, dtype, hd):
    """Few pairs, some, many; capped, at caps from the smallest to the largest."""
    say(f"attention {dtype} hd={hd} new={new}")
    st = SetupExt(gpu, [(new, 150), (1, 70)], 16, 2, hd, dtype, 16, cap=7.0, seed=3)
    for cap in (7.0, 2.0 ** -60, 0.3, 2.0 ** 60):
        st.cap = st.layer.score_cap = cap
        st.check()


@pytest.mark.parametrize("dtype", ["e4m3", "i8"])
@pytest.mark.parametrize("new,hd", [(1, 128), (7, 64), (50, 128), (20, 256), (40, 512)])
def test_attention_spread_scales(gpu, dtype, new, hd):
    """Scales of very different size beside each other (2^-40 to 2^40 and more in the values)."""
    ms = gpu
    say(f"attention, spread scales: {dtype} new={new} hd={hd}")
    st = SetupExt(ms, [(new, 150)], 4, 2, hd, dtype, 16, seed=13)
    g = st.slots(0, 0, 150)
    x = st.pool["v"].copy()
    x[g] *= 2.0 ** (20 * np.random.default_rng(5).standard_normal((150, 2, 1)))
    x[st.slots(0, 3, 4)] = 0
    st.fill("v", x)
    y = st.pool["k"].copy()
    y[g] *= 2.0 ** np.random.default_rng(6).uniform(-8, 1, (150, 2, 1))
    st.fill("k", y)
    st.upload()
    st.check()
    q = f32(new, 4, hd, seed=14)
    q[:, 0] *= 1e-30
    q[:, 1] *= 1e-4
    q[:, 2, ::2] *= 1e-6
    q[:, 3] = 0
    want, tol = st.attend(q.reshape(new, -1))
    got = st.run_attention(q.reshape(new, -1))
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("dtype", ["e4m3", "i8", "bf16"])
@pytest.mark.parametrize("new,length,window", [(1, 400, 0), (40, 170, 0), (40, 170, 50), (3, 1200, 0)])
def test_attention_not_finite(gpu, dtype, new, length, window, cap):
    """Values that are not finite reach only the rows that attend to them, as the formula says (an 8-bit head is
    NaN as a whole; infinite keys score the cap, or minus the cap)."""
    ms = gpu
    if dtype == "bf16" and not cap:
        pytest.skip("ms_paged_attention's own test")
    say(f"attention, not finite: {dtype} new={new} length={length} window={window} cap={cap}")
    st = SetupExt(ms, [(new, length), (2, 30)], 4, 2, 128, dtype, 16, window=window, cap=cap, seed=9)
    q = np.abs(f32(st.rows, 4 * 128, seed=4)) + 0.1
    late = length - 1 - min(new - 1, 1)  # a position that the first rows of a chunk do not see
    for kind in ("k nan", "v nan") + (() if st.eight else ("v inf", "k -inf", "k inf")):
        n, what = kind.split()
        keep = (st.raw[n].copy(), st.scales[n].copy()) if st.eight else st.pool[n].copy()
        for pos, head in ((late, 0), (length - min(length, 30), 1)):
            g = st.slots(0, pos, pos + 1)
            if st.eight:
                st.scales[n][g[0], head, g[1]] = np.nan
            else:
                x = decode(st.pool[n][g], dtype).astype(np.float32)
                x[0, head, 5] = {"nan": np.nan, "inf": np.inf, "-inf": -np.inf}[what]
                st.pool[n][g] = encode(x, dtype)
        st.upload()
        want, tol = st.attend(q)
        got = st.run_attention(q)
        for kind_of in (np.isnan, np.isposinf, np.isneginf):
            assert np.array_equal(kind_of(got), kind_of(want)), kind
        fine = np.isfinite(want)
        assert fine.any() and np.all(np.abs(got[fine] - want[fine]) <= tol[fine]), kind
        if st.eight:
            st.raw[n], st.scales[n] = keep
        else:
            st.pool[n] = keep


@pytest.mark.parametrize("dtype", ["e4m3", "i8", "f32"])
@pytest.mark.parametrize("new,hd", [(1, 128), (8, 64), (50, 128), (50, 512)])
def test_attention_rows_not_finite(gpu, dtype, new, hd):
    """A query that is not finite spoils its own row alone."""
    ms = gpu
    say(f"attention, rows not finite: {dtype} new={new} hd={hd}")
    st = SetupExt(ms, [(new, 90), (1, 40)], 4, 2, hd, dtype, 16, seed=23, cap=4.0 if dtype == "f32" else 0.0)
    q = f32(st.rows, 4, hd, seed=24)
    q[0, 1, 3] = np.nan
    want, tol = st.attend(q.reshape(st.rows, -1))
    got = st.run_attention(q.reshape(st.rows, -1))
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want).any()
    fine = np.isfinite(want)
    assert np.all(np.abs(got[fine] - want[fine]) <= tol[fine])


@pytest.mark.parametrize("size", [1e9, 1e30])
@pytest.mark.parametrize("dtype", ["e4m3", "i8"])
@pytest.mark.parametrize("seqs,hd", [([(1, 20)] * 50, 128), ([(1, 9)] * 30, 64), ([(1, 30)] * 30, 256),
                                     ([(1, 3000)] * 3, 128), ([(40, 40), (1, 20)], 128), ([(40, 60), (1, 20)], 512)])
def test_attention_large_scores(gpu, seqs, hd, dtype, size):
    """Finite scores of any size: the best key, where it is far ahead, takes all.  A score may be off by (hd + 8)
    2^-24 of the sum of its products' magnitudes; a key that is behind by twice that and 150 weighs nothing in fp32."""
    say(f"attention, large scores: {len(seqs)} x {seqs[0]} hd={hd} {dtype} q x {size}")
    st = SetupExt(gpu, seqs, 2, 2, hd, dtype, 32, seed=31)
    q = f32(st.rows, 2 * hd, seed=32) * np.float32(size)
    got = st.run_attention(q).reshape(st.rows, 2, hd)
    sure = 0
    for r, (s, p) in enumerate(st.row_of()):
        k, v = (st.pool[n][st.slots(s, 0, p + 1)] for n in "kv")
        for h in range(2):
            y = q[r, h * hd:(h + 1) * hd].astype(np.float64) / np.sqrt(hd)
            x = k[:, h] @ y
            off = (hd + 8) * 2.0 ** -24 * (np.abs(k[:, h]) @ np.abs(y)).max()
            best = np.argmax(x)
            if len(x) == 1 or x[best] - np.delete(x, best).max() > 2 * off + 150:
                # (what is left: the probability times the scale, three parts added up on the matrix cores, by 2^-23
                # each, the division as two roundings: 7 times 2^-24)
                assert np.all(np.abs(got[r, h] - v[best, h]) <= 2.0 ** -21 * np.abs(v[best, h]))
                sure += 1
    assert sure > 0.9 * 2 * st.rows


def test_attention_scale_and_freed_pages(gpu):
    ms = gpu
    say("attention: a scale of its own, freed pages, a shared prefix")
    st = SetupExt(ms, [(3, 200), (1, 40), (5, 90)], 4, 2, 64, "i8", 16, window=50, seed=5, scale=-0.3)
    q, want = st.check()
    st.pages[0, :(200 - 3 - 50 + 1) // 16] = -1
    st.batch.set(st.new, st.len, st.pages)
    assert np.array_equal(st.run_attention(q), want)
    st.layer.base.window = 0
    with pytest.raises(ms.MSError, match="page is -1"):
        st.run_attention(q)
    d = ms.DeviceBuffer(200 * 128 * 4)
    with pytest.raises(ms.MSError, match="page is -1"):
        ms.paged_read(st.layer, st.batch, 0, 100, 10, d, None, 128)
    ms.paged_read(st.layer, st.batch, 0, 150, 50, d, None, 128)
    ms.synchronize()


def test_far_pages(gpu):
    """Pools past 2^32 bytes: the far pages' bytes and scales, and no others."""
    ms = gpu
    say("paged_ext: offsets past 32 bits")
    kv, hd, page, n_pages = 4, 512, 16, 150000  # 32 KiB a page, 4.9 GB a pool
    assert n_pages * page * kv * hd > 2 ** 32
    pools = [ms.DeviceBuffer(n_pages * page * kv * hd) for _ in range(2)]
    scales = [ms.DeviceBuffer(n_pages * page * kv * 4) for _ in range(2)]
    base = ms.PagedLayer(n_heads=8, n_kv_heads=kv, head_dim=hd, dtype=ms.MS_KV_I8, k=pools[0].ptr, v=pools[1].ptr)
    layer = ms.PagedLayerExt(base=base, k_scale=scales[0].ptr, v_scale=scales[1].ptr)
    n = 55
    st = SetupExt(ms, [(n, n)], 8, kv, hd, "i8", page, seed=8)
    pages = np.array([[149999, 3, 140000, 131073]], np.int32)
    b = ms.PagedBatch(page, n_pages, 1, n, 4)
    b.set([n], [n], pages)
    x = {m: st.pool[m][st.slots(0, 0, n)].reshape(n, -1).astype(np.float32) for m in "kv"}
    dk, dv = (ms.DeviceBuffer.from_array(x[m]) for m in "kv")
    ms.paged_append(layer, b, dk, dv, kv * hd)
    out = ms.DeviceBuffer(n * kv * hd * 4)
    for m in range(2):
        ms.paged_read(layer, b, 0, 0, n, out if m == 0 else None, out if m else None, kv * hd)
        ms.synchronize()
        got = out.download(np.float32, x["kv"[m]].shape)
        # (values that were codes times a scale: their own scale again, to its last bit)
        assert np.all(np.abs(got - x["kv"[m]]) <= 2.0 ** -22 * np.abs(x["kv"[m]]))
        st.pool["kv"[m]][st.slots(0, 0, n)] = got.reshape(n, kv, hd)
    st.batch, st.layer, old = b, layer, (st.batch, st.layer)
    st.check()
    b.set([1], [n], pages)  # a single token takes another way
    st.new, st.rows = [1], 1
    st.check()
    del old


def test_refusals_with_a_batch(gpu):
    """Row arguments, refused once a batch is set."""
    ms = gpu
    say("paged_ext: refused rows")
    st = SetupExt(ms, [(2, 9), (1, 4)], 4, 2, 64, "e4m3", 16, rot=64, seed=1)
    d = ms.DeviceBuffer(1 << 16)
    L, h, p = C.byref(st.layer), st.batch.h, d.ptr
    far = p + (1 << 15)
    at = ms.lib().ms_paged_attention_ext
    for args in ((None, 256, far, 256), (p, 256, None, 256), (p + 4, 256, far, 256), (p, 256, far + 8, 256),
                 (p, 255, far, 256), (p, 252, far, 256), (p, 256, p, 256), (p, 512, p + 1008, 512)):
        assert at(L, h, *args) == -1, args
    ap = ms.lib().ms_paged_append_ext
    good = dict(k=p, v=p, kvs=128, q=p + 4096, qs=256, o=far, os=256, c=p, s=p, n=9)
    for change in (dict(k=None), dict(v=None), dict(k=p + 4), dict(kvs=126), dict(kvs=124), dict(o=None),
                   dict(q=p + 4100), dict(o=far + 4), dict(qs=252), dict(os=258), dict(n=8), dict(c=None),
                   dict(o=p + 4096 + 1024), dict(o=p), dict(v=far, o=far)):
        a = {**good, **change}
        assert ap(L, h, a["k"], a["v"], a["kvs"], a["q"], a["qs"], a["o"], a["os"], a["c"], a["s"], a["n"]) == -1, change
    rd = ms.lib().ms_paged_read
    for args in ((-1, 0, 1, p, far, 128), (2, 0, 1, p, far, 128), (0, -1, 1, p, far, 128), (0, 9, 1, p, far, 128),
                 (0, 0, 10, p, far, 128), (0, 0, -1, p, far, 128), (0, 0, 2, p + 4, far, 128), (0, 0, 2, p, far, 124),
                 (0, 0, 2, p, far, 126), (0, 0, 2, p, p + 512, 128)):
        assert rd(L, h, *args) == -1, args


# ---- a step of all of them -----------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["e4m3", "i8"])
def test_steps(gpu, dtype):
    """A prompt's chunk and then single tokens of a batch: append, attention, read, and a token drawn from logits, one
    handle for all; each step against 64 bits over what the pages then hold."""
    ms = gpu
    say(f"steps, {dtype}")
    heads, kv, hd, rot, page, vocab = 4, 2, 128, 64, 16, 1000
    st = SetupExt(ms, [(0, 60), (0, 41)], heads, kv, hd, dtype, page, rot=rot, norm=3, gamma=True, cap=30.0, max_rows=96,
                  seed=2)
    c, s = ms.rope_table(rot, 1e6, 64)
    ms.synchronize()
    hc, hs = (t.download(np.float32, (64, rot // 2)) for t in (c, s))
    nq, nkv = heads * hd, kv * hd
    ld = nq + 2 * nkv
    w_out = f32(nq, vocab, seed=3, scale=0.2)
    for step, (new, length) in enumerate((((50, 33), (50, 33)), ((1, 1), (51, 34)), ((1, 0), (52, 34)), ((1, 2), (53, 36)))):
        st.new, st.len, st.rows = list(new), list(length), sum(new)
        st.batch.set(st.new, st.len, st.pages)
        x = f32(st.rows, ld, seed=10 + step)
        d, o = ms.DeviceBuffer.from_array(x), ms.DeviceBuffer(st.rows * nq * 4)
        ms.paged_append(st.layer, st.batch, At(d, nq), At(d, nq + nkv), ld, d, ld, d, ld, c, s, 64)
        ms.paged_attention(st.layer, st.batch, d, ld, o, nq)
        back = ms.DeviceBuffer(st.len[0] * nkv * 4)
        ms.paged_read(st.layer, st.batch, 0, 0, st.len[0], None, back, nkv)
        ms.synchronize()
        codes, scales = st.download8()
        st.raw, st.scales = codes, scales
        for n in "kv":
            st.pool[n] = st.values(n)
        q = d.download(np.float32, x.shape)[:, :nq]
        (wq, _, _), (tq, _, _) = append_in_64(st, x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:], hc, hs)
        assert np.all(np.abs(q.reshape(wq.shape) - wq) <= tq)
        want, tol = st.attend(np.ascontiguousarray(q))
        att = o.download(np.float32, want.shape)
        assert np.all(np.abs(att - want) <= tol)
        assert np.array_equal(back.download(np.float32, (st.len[0], nkv)),
                              st.pool["v"][st.slots(0, 0, st.len[0])].reshape(-1, nkv).astype(np.float32))
        logits = (att.astype(np.float64) @ w_out).astype(np.float32)
        dl, du = ms.DeviceBuffer.from_array(logits), ms.DeviceBuffer.from_array(np.full(st.rows, 0.4, np.float32))
        ids = ms.DeviceBuffer(st.rows * 4)
        ms.logits_process(dl, vocab, dl, vocab, vocab, [ms.LogitsRow()] * st.rows)
        ms.sample_rows(dl, vocab, vocab, [ms.SampleRow(0.7, 20, 0.9)] * st.rows, du, ids)
        ms.synchronize()
        for r, got in enumerate(ids.download(np.int32, (st.rows,))):
            order = np.argsort(-logits[r], kind="stable")[:20]
            w = np.exp((logits[r][order].astype(np.float64) - logits[r].max()) / np.float64(np.float32(0.7)))
            order = order[:1 + np.searchsorted(np.cumsum(w), np.float64(np.float32(0.9)) * w.sum())]
            order = np.sort(order)
            w = np.exp((logits[r][order].astype(np.float64) - logits[r].max()) / np.float64(np.float32(0.7)))
            assert got == order[np.searchsorted(np.cumsum(w), np.float64(np.float32(0.4)) * w.sum(), side="right")]
