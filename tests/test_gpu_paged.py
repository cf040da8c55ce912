"""The paged cache on the GPU: append and attention against 64 bits, at the sizes, masks and
contents where they can go wrong."""
import numpy as np
import pytest

from tests.paged_ref import HALF, Setup, decode, encode, raw_type

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"\n[case] {msg}", flush=True)


def f32(*shape, seed=0, scale=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * scale).astype(np.float32)


def tables(ms, rot, n_pos, wide=True, pos0=0, theta=1e4):
    c, s = ms.rope_table(rot, theta, n_pos, pos0, wide)
    ms.synchronize()
    return c, s, c.download(np.float32, (n_pos, rot // 2)), s.download(np.float32, (n_pos, rot // 2))


# ---- rotary tables --------------------------------------------------------------
@pytest.mark.parametrize("rot,pos0,n", [(2, 0, 5), (64, 0, 300), (128, 131000, 73), (254, 7, 1)])
def test_rope_table_wide(gpu, rot, pos0, n):
    """64-bit angles, one rounding: 2^-24 of the value, and what 64 bits lose of angles up to
    1.4e5 (1.4e5 * 2^-50)."""
    say(f"rope table rot={rot} pos0={pos0} n={n}")
    _, _, c, s = tables(gpu, rot, n, True, pos0)
    ang = (pos0 + np.arange(n))[:, None] * 1e4 ** (-2.0 * np.arange(rot // 2) / rot)
    for got, want in ((c, np.cos(ang)), (s, np.sin(ang))):
        assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 2e-10)


def test_rope_table_is_ms_rope(gpu):
    """wide = 0: the angles of ms_rope, bit for bit (unit vectors turned by it)."""
    ms, rot, n, pos0 = gpu, 128, 40, 4000
    say("rope table against ms_rope")
    _, _, c, s = tables(ms, rot, n, False, pos0, 1e6)
    x = np.zeros((n, rot), np.float32)
    x[:, :rot // 2] = 1
    d = ms.DeviceBuffer.from_array(x)
    ms.check(ms.lib().ms_rope(d.ptr, n, rot, 1, rot, rot, 1e6, pos0))
    got = d.download(np.float32, x.shape)
    assert np.array_equal(got[:, :rot // 2], c) and np.array_equal(got[:, rot // 2:], s)


# ---- append ------------------------------------------------------------------------
def rotate(x, c, s, rot):
    """64-bit rotation of x [rows][heads][hd] and what fp32 may be off: three roundings."""
    x = x.astype(np.float64)
    h = rot // 2
    y, tol = x.copy(), np.zeros_like(x)
    a, b = x[..., :h], x[..., h:rot]
    c, s = c[:, None].astype(np.float64), s[:, None].astype(np.float64)
    y[..., :h], y[..., h:rot] = a * c - b * s, a * s + b * c
    tol[..., :h] = 2.0 ** -23 * (np.abs(a * c) + np.abs(b * s))
    tol[..., h:rot] = 2.0 ** -23 * (np.abs(a * s) + np.abs(b * c))
    return y, tol


APPENDS = [
    # seqs (new, length), heads, kv, hd, rot, page, page_rows, dtype
    ([(1, 1)], 8, 2, 64, 64, 16, 0, "f32"),
    ([(1, 301), (0, 17), (1, 16), (1, 17), (0, 0)], 40, 8, 128, 128, 16, 0, "bf16"),
    ([(33, 33), (1, 5), (70, 135)], 8, 2, 512, 128, 24, 60, "f16"),
    ([(5, 9)], 5, 1, 256, 0, 1, 1, "bf16"),
    ([(7, 7), (2, 64)], 6, 3, 64, 2, 7, 9, "f32"),
    ([(9, 40)], 4, 4, 128, 126, 32, 32, "f16"),
    ([(300, 1000)], 2, 2, 256, 256, 128, 0, "f32"),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
@pytest.mark.parametrize("how", ["apart", "fused", "kv"])
def test_append(gpu, case, how):
    """Pool values: fp32 rotation, one rounding to the pool's type; every other slot keeps
    its bits.  q: apart, in place in fused q | k | v rows, or not at all."""
    ms = gpu
    seqs, heads, kv, hd, rot, page, pr, dtype = APPENDS[case]
    say(f"append {APPENDS[case]} {how}")
    st = Setup(ms, seqs, heads, kv, hd, dtype, page, pr, rot=rot, seed=case)
    nq, nkv = heads * hd, kv * hd
    n_pos = max(st.len)
    c, s, hc, hs = tables(ms, rot, n_pos, case % 2 == 0) if rot else (None, None, None, None)
    x = f32(st.rows + 2, nq + 2 * nkv + 4, seed=case + 50)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:nq + 2 * nkv]
    ld = x.shape[1]

    class At:
        def __init__(self, b, off):
            self.ptr = b.ptr + 4 * off

    if how == "fused":
        d = ms.DeviceBuffer.from_array(x)
        ms.paged_append(st.layer, st.batch, At(d, nq), At(d, nq + nkv), ld, d, ld, d, ld, c, s, n_pos)
        got_q = d.download(np.float32, x.shape)
        assert np.array_equal(got_q[st.rows:], x[st.rows:]) and np.array_equal(got_q[:, nq:], x[:, nq:])
        got_q = got_q[:st.rows, :nq]
    else:
        dk, dv, dq = (ms.DeviceBuffer.from_array(np.ascontiguousarray(t)) for t in (k, v, q))
        do = ms.DeviceBuffer.from_array(np.full((st.rows + 2, nq + 8), -777, np.float32))
        if how == "apart":
            ms.paged_append(st.layer, st.batch, dk, dv, nkv, dq, nq, do, nq + 8, c, s, n_pos)
        else:
            ms.paged_append(st.layer, st.batch, dk, dv, nkv, cos=c, sin=s, n_pos=n_pos)
        out = do.download(np.float32, (st.rows + 2, nq + 8))
        assert np.all(out[st.rows:] == -777) and np.all(out[:, nq:] == -777)
        got_q = out[:st.rows, :nq]
    ms.synchronize()
    pos = np.array([p for _, p in st.row_of()])
    q, k, v = q[:st.rows], k[:st.rows], v[:st.rows]
    turn = (lambda y, n: rotate(y.reshape(-1, n, hd), hc[pos], hs[pos], rot)) if rot else \
        (lambda y, n: (y.reshape(-1, n, hd).astype(np.float64), np.zeros((len(y), n, hd))))
    if how != "kv":
        want, tol = turn(q, heads)
        assert np.all(np.abs(got_q.reshape(want.shape) - want) <= tol)
    else:
        assert np.all(got_q == -777)
    wk, tk = turn(k, kv)
    got = st.download()
    for r, (sq, p) in enumerate(st.row_of()):
        at = (st.pages[sq, p // page], p % page)
        half = HALF[dtype] if dtype != "f32" else 0.0
        # (a value of fp16's or bf16's smallest steps: half of one)
        tiny = {"f32": 0.0, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}[dtype]
        g = decode(got["k"][at], dtype)
        assert np.all(np.abs(g - wk[r]) <= (1 + half) * tk[r] + half * np.abs(wk[r]) + tiny)
        assert np.array_equal(got["v"][at], encode(v[r].reshape(kv, hd), dtype))
        st.pool["k"][at], st.pool["v"][at] = got["k"][at], got["v"][at]
    for n in "kv":
        assert np.array_equal(got[n].view(np.uint8), st.pool[n].view(np.uint8))


def test_append_special_values(gpu):
    """Infinities and NaN arrive as they are; what fp16 cannot hold becomes infinity."""
    ms = gpu
    say("append: special values")
    st = Setup(ms, [(2, 5)], 2, 2, 64, "f16", 4, seed=3)
    v = f32(2, 128, seed=1)
    v[0, :6] = [np.inf, -np.inf, np.nan, 65519.0, 65520.0, -1e9]
    d = ms.DeviceBuffer.from_array(v)
    ms.paged_append(st.layer, st.batch, d, d, 128)
    ms.synchronize()
    got = st.download()
    for r, (s, p) in enumerate(st.row_of()):
        for n in "kv":
            assert np.array_equal(got[n][st.pages[s, p // 4], p % 4].ravel(), encode(v[r], "f16"), equal_nan=True)
    assert encode(v, "f16")[0, 3] == np.float16(65504) and np.isinf(encode(v, "f16")[0, 4])


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
    ([(40, 3000)], 8, 1, 512, 16, 0, 0),                                 # chunks over split keys
    ([(200, 4100)], 4, 1, 128, 16, 0, 0),
    ([(90, 400), (33, 33)], 4, 2, 128, 16, 0, 70),
    ([(129, 129)], 1, 1, 256, 16, 0, 0),                                 # one pair past a block's
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention(gpu, case, dtype):
    seqs, heads, kv, hd, page, pr, window = ATTENDS[case]
    say(f"attention {dtype} {ATTENDS[case]}")
    st = Setup(gpu, seqs, heads, kv, hd, dtype, page, pr, window, seed=case)
    st.check_attention(pad=4 * (case % 3))


def test_attention_scale(gpu):
    say("attention: a scale of its own, and scores far apart")
    st = Setup(gpu, [(5, 77)], 4, 2, 128, "f32", scale=0.3, seed=2)
    st.check_attention()
    st.layer.scale = st.scale = -0.02
    st.check_attention()
    # one key far above the others, and values of very different size
    st.layer.scale = st.scale = 0.0
    s, o = st.slots(0, 0, 77)
    st.pool["k"][s[40], o[40]] *= 40
    st.pool["v"][s[::3], o[::3]] *= 1e6
    st.pool["v"][s[1::3], o[1::3]] *= 1e-6
    st.upload()
    st.check_attention()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new,hd", [(1, 128), (7, 64), (50, 128), (20, 256)])
def test_attention_sizes_of_q(gpu, dtype, new, hd):
    """Queries of very different size: between rows, and between the dims of one."""
    ms = gpu
    say(f"attention, sizes of q: {dtype} new={new} hd={hd}")
    st = Setup(ms, [(new, 150)], 4, 2, hd, dtype, 16, seed=13)
    q = f32(new, 4, hd, seed=14)
    q[:, 0] *= 1e-30
    q[:, 1] *= 1e-4
    q[:, 2, ::2] *= 1e-6
    q[:, 3] = 0
    q = q.reshape(new, -1)
    want, tol = st.attend(q)
    got = st.run_attention(q)
    assert np.all(np.abs(got - want) <= tol)
    # far beyond fp16, the best key takes all: a finite result, that key's values
    g = st.slots(0, 0, 150)
    k, v = decode(st.pool["k"][g], dtype), decode(st.pool["v"][g], dtype)
    q = f32(new, 4, hd, seed=15)
    big = (q * np.float32(1e30)).reshape(new, -1)
    got = st.run_attention(big).reshape(new, 4, hd)
    for r in range(new):
        for h in range(4):
            best = np.argmax(k[:150 - new + r + 1, h // 2] @ q[r, h].astype(np.float64))
            assert np.array_equal(got[r, h], v[best, h // 2].astype(np.float32))


@pytest.mark.parametrize("new,hd", [(1, 128), (6, 128), (1, 512), (60, 64), (60, 512)])
@pytest.mark.parametrize("dtype,tiny", [("f16", 2.0 ** -19), ("bf16", 2.0 ** -100), ("f32", 2.0 ** -90)])
def test_attention_tiny_values(gpu, dtype, tiny, new, hd):
    """Values far below 1 (fp16: below its smallest normal number) keep what their type holds."""
    say(f"attention, tiny values: {dtype} {tiny} new={new} hd={hd}")
    st = Setup(gpu, [(new, 100)], 4, 2, hd, dtype, 16, seed=21)
    for n in "kv":
        x = decode(st.pool[n], dtype) * tiny
        st.pool[n] = encode(x.astype(np.float32), dtype)
    st.upload()
    st.layer.scale = st.scale = 1.0
    st.check_attention(scale=0.1 / tiny)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new,length,window", [(1, 400, 0), (40, 170, 0), (40, 170, 50), (3, 1200, 0)])
def test_attention_not_finite(gpu, dtype, new, length, window):
    """Values that are not finite reach only the rows that attend to them, as the formula
    says: NaN in a key or value, infinity in a value (infinity where its weight is not
    zero), minus infinity as a score (no weight)."""
    ms = gpu
    say(f"attention, not finite: {dtype} new={new} length={length} window={window}")
    st = Setup(ms, [(new, length), (2, 30)], 4, 2, 128, dtype, 16, window=window, seed=9)
    q = np.abs(f32(st.rows, 4 * 128, seed=4)) + 0.1
    late = length - 1 - min(new - 1, 1)  # a position that the first rows of a chunk do not see
    for kind in ("k nan", "v nan", "v inf", "k -inf", "k inf"):
        st2 = {n: p.copy() for n, p in st.pool.items()}
        for pos, head in ((late, 0), (length - min(length, 30), 1)):
            g = st.slots(0, pos, pos + 1)
            x = decode(st.pool[kind[0]][g], dtype).astype(np.float32)
            x[0, head, 5] = {"nan": np.nan, "inf": np.inf, "-inf": -np.inf}[kind.split()[1]]
            st.pool[kind[0]][g] = encode(x, dtype)
        st.upload()
        want, tol = st.attend(q)
        got = st.run_attention(q)
        for kind_of in (np.isnan, np.isposinf, np.isneginf):
            assert np.array_equal(kind_of(got), kind_of(want)), kind
        fine = np.isfinite(want)
        assert fine.any()
        assert np.all(np.abs(got[fine] - want[fine]) <= tol[fine]), kind
        st.pool = st2


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new,hd", [(1, 128), (8, 64), (50, 128), (50, 512)])
def test_attention_rows_not_finite(gpu, dtype, new, hd):
    """A query that is not finite spoils its own row alone; a row all of whose keys score minus
    infinity has no result (NaN, as the formula)."""
    ms = gpu
    say(f"attention, rows not finite: {dtype} new={new} hd={hd}")
    st = Setup(ms, [(new, 90), (1, 40)], 4, 2, hd, dtype, 16, seed=23)
    q = f32(st.rows, 4, hd, seed=24)
    q[0, 1, 3], q[new // 2, 2, 7] = np.nan, np.inf
    want, tol = st.attend(q.reshape(st.rows, -1))
    got = st.run_attention(q.reshape(st.rows, -1))
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want).any()
    fine = np.isfinite(want)
    assert np.all(np.abs(got[fine] - want[fine]) <= tol[fine])
    # every key of kv head 1
    g = st.slots(0, 0, 90)
    x = decode(st.pool["k"][g], dtype).astype(np.float32)
    x[:, 1, 0] = -np.inf
    st.pool["k"][g] = encode(x, dtype)
    st.upload()
    q = np.abs(f32(st.rows, 4, hd, seed=25)) + 0.1
    got = st.run_attention(q.reshape(st.rows, -1)).reshape(st.rows, 4, hd)
    assert np.isnan(got[:new, 2:]).all() and np.isfinite(got[:new, :2]).all() and np.isfinite(got[new]).all()


def one_key_takes_all(st, q):
    """Rows and heads whose best key takes all, and those keys' values, in 64 bits.  A score may be off
    by (hd + 8) 2^-24 of the sum of its products' magnitudes; a key that is behind by twice
    that and 150 has a weight below fp32's smallest number (e^-150 < 2^-149 2^-67)."""
    G = st.heads // st.kv
    want, sure = np.zeros((st.rows, st.heads, st.hd), np.float32), np.zeros((st.rows, st.heads), bool)
    q, sc = q.reshape(st.rows, st.heads, st.hd).astype(np.float64), st.scale or 1 / np.sqrt(st.hd)
    for r, (s, p) in enumerate(st.row_of()):
        k, v = (decode(st.pool[n][st.slots(s, 0, p + 1)], st.dtype) for n in "kv")
        for h in range(st.heads):
            x = k[:, h // G] @ q[r, h] * sc
            off = (st.hd + 8) * 2.0 ** -24 * (np.abs(k[:, h // G]) @ np.abs(q[r, h])).max() * abs(sc)
            best = np.argmax(x)
            want[r, h] = v[best, h // G]
            sure[r, h] = len(x) == 1 or x[best] - np.delete(x, best).max() > 2 * off + 150
    return want, sure


@pytest.mark.parametrize("size", [3e8, 1e9, 1e10, 1e30])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("seqs,hd", [([(1, 20)] * 150, 128), ([(1, 9)] * 60, 64), ([(1, 30)] * 60, 256),
                                     ([(1, 30)] * 60, 512), ([(1, 3000)] * 3, 128), ([(40, 40), (1, 20)], 128),
                                     ([(40, 60), (1, 20)], 512)])
def test_attention_large_scores(gpu, seqs, hd, dtype, size):
    """Finite scores of any size: where one key is far above the others the result is its value,
    also for a row that has an item to itself (1 pair a kv head)."""
    say(f"attention, large scores: {len(seqs)} x {seqs[0]} hd={hd} {dtype} q x {size}")
    st = Setup(gpu, seqs, 2, 2, hd, dtype, 32, seed=31)
    q = f32(st.rows, 2 * hd, seed=32) * np.float32(size)
    want, sure = one_key_takes_all(st, q)
    assert sure.mean() > 0.9
    got = st.run_attention(q).reshape(want.shape)
    assert np.array_equal(got[sure], want[sure])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new,hd", [(2, 128), (50, 64)])
def test_attention_large_scale_beside_nan(gpu, dtype, new, hd):
    """A row beside one whose key is NaN, with a scale whose product with q alone
    passes fp32 (1e30 * 1e10), while the scores do not."""
    say(f"attention, large scale beside NaN: {dtype} new={new} hd={hd}")
    st = Setup(gpu, [(new, 90)], 2, 2, hd, dtype, 16, seed=33, scale=1e30)
    st.pool["k"] = encode((decode(st.pool["k"], dtype) * 1e-20).astype(np.float32), dtype)
    g = st.slots(0, 89, 90)
    st.pool["k"][g] = encode(np.full((1, 2, hd), np.nan, np.float32), dtype)
    st.upload()
    q = f32(new, 2 * hd, seed=34) * np.float32(1e10)
    got = st.run_attention(q).reshape(new, 2, hd)
    st.new, st.len, st.rows = [new - 1], [89], new - 1
    want, sure = one_key_takes_all(st, q[:-1])
    assert sure.mean() > 0.9 and np.isnan(got[-1]).all()
    assert np.array_equal(got[:-1][sure], want[sure])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_window_far_along(gpu, dtype):
    """A sliding window's work is that of its keys: a token at position 599 and one at 128599,
    with the same keys in the window, are computed alike, to the bit."""
    ms = gpu
    say(f"attention: a window far along, {dtype}")
    near = Setup(ms, [(1, 600)], 8, 2, 256, dtype, 16, window=512, seed=35)
    q, want = near.check_attention()
    ahead = 128000  # whole pages and whole tiles of keys
    pages = np.full((1, (ahead + 600 + 15) // 16), -1, np.int32)
    pages[0, ahead // 16:] = near.pages[0]
    pages[0, :(ahead + 599 - 511) // 16] = -1
    near.batch = ms.PagedBatch(16, near.n_pages, 1, 1, pages.shape[1])
    near.batch.set([1], [ahead + 600], pages)
    assert np.array_equal(near.run_attention(q), want)


def test_attention_freed_pages(gpu):
    """Pages behind a window may be given back: -1 in the table; full attention is refused."""
    ms = gpu
    say("attention: freed pages")
    st = Setup(ms, [(3, 200), (1, 40)], 4, 2, 64, "bf16", 16, window=50, seed=5)
    q, want = st.check_attention()
    st.pages[0, :(200 - 3 - 50 + 1) // 16] = -1
    st.batch.set(st.new, st.len, st.pages)
    assert np.array_equal(st.run_attention(q), want)
    st.layer.window = 51 + 16
    with pytest.raises(ms.MSError, match="page is -1"):
        st.run_attention(q)
    st.layer.window = 0
    with pytest.raises(ms.MSError, match="page is -1"):
        st.run_attention(q)


def test_batch_used_again(gpu):
    """One handle through several steps and layers of different shape: every call sees the
    step that was set last, and a refused one changes nothing."""
    ms = gpu
    say("batch: several steps, several layers")
    st = Setup(ms, [(40, 60), (1, 33), (0, 20)], 8, 2, 128, "bf16", 16, seed=6, max_rows=64)
    other = Setup(ms, [(40, 60), (1, 33), (0, 20)], 4, 4, 256, "f32", 16, window=17, seed=6)
    assert np.array_equal(st.pages, other.pages)
    other.batch = st.batch
    for new in ([40, 1, 0], [1, 1, 1], [0, 33, 1], [60, 0, 0], [1, 0, 0], [0, 0, 0]):
        st.new = other.new = new
        st.rows = other.rows = sum(new)
        st.batch.set(st.new, st.len, st.pages)
        with pytest.raises(ms.MSError):
            st.batch.set([1, 1, 21], st.len, st.pages)
        for x in (st, other, st):
            if x.rows:
                x.check_attention(seed=sum(new))
            else:
                x.run_attention(np.zeros((0, x.heads * x.hd), np.float32))
    st.batch.set([], [], np.zeros((0, 1), np.int32))
    st.rows = 0
    st.run_attention(np.zeros((0, 8 * 128), np.float32))


def test_shared_prefix(gpu):
    say("attention: two sequences with the same first pages")
    ms = gpu
    st = Setup(ms, [(1, 80), (5, 90)], 4, 2, 128, "f16", 16, seed=7)
    st.pages[1, :3] = st.pages[0, :3]
    st.batch.set(st.new, st.len, st.pages)
    st.check_attention()


def test_far_pages(gpu):
    """Pools past 2^32 bytes: the far pages' bytes, and no others."""
    ms = gpu
    say("paged: offsets past 32 bits")
    kv, hd, page, n_pages = 2, 512, 16, 70000  # 64 KiB a page, 4.6 GB a pool
    assert n_pages * page * kv * hd * 4 > 2 ** 32
    pools = [ms.DeviceBuffer(n_pages * page * kv * hd * 4) for _ in range(2)]
    layer = ms.PagedLayer(n_heads=8, n_kv_heads=kv, head_dim=hd, dtype=0, k=pools[0].ptr, v=pools[1].ptr)
    pages = np.array([[69999, 3, 66000, 65537]], np.int32)
    n = 55
    st = Setup(ms, [(n, n)], 8, kv, hd, "f32", page, seed=8)
    g = st.slots(0, 0, n)
    k, v = (st.pool[x][g].reshape(n, -1) for x in "kv")
    dk, dv = ms.DeviceBuffer.from_array(k), ms.DeviceBuffer.from_array(v)
    b = ms.PagedBatch(page, n_pages, 1, n, 4)
    b.set([n], [n], pages)
    ms.paged_append(layer, b, dk, dv, kv * hd)
    st.batch, st.layer, old = b, layer, (st.batch, st.layer)
    st.check_attention()
    b.set([1], [n], pages)  # a single token takes another way
    st.new, st.rows = [1], 1
    st.check_attention()
    out = np.empty((page, kv * hd), np.float32)
    ms.synchronize()
    ms.check(ms.lib().ms_memcpy_d2h(out.ctypes.data, pools[0].ptr + 69999 * page * kv * hd * 4, out.nbytes))
    assert np.array_equal(out, k[:page])
    del old


def test_refusals_with_a_batch(gpu):
    """Row arguments, refused once a batch is set."""
    import ctypes as C
    ms = gpu
    say("paged: refused rows")
    st = Setup(ms, [(2, 9), (1, 4)], 4, 2, 64, "f32", 16, rot=64, seed=1)
    d = ms.DeviceBuffer(1 << 16)
    L, h, p = C.byref(st.layer), st.batch.h, d.ptr
    far = p + (1 << 15)
    at = ms.lib().ms_paged_attention
    for args in ((None, 256, far, 256), (p, 256, None, 256), (p + 4, 256, far, 256), (p, 256, far + 8, 256),
                 (p, 255, far, 256), (p, 252, far, 256), (p, 256, far, 254), (p, 256, p, 256),
                 (p, 256, p + 1024, 256), (p, 512, p + 1008, 512)):
        assert at(L, h, *args) == -1, args
    ap = ms.lib().ms_paged_append
    good = dict(k=p, v=p, kvs=128, q=p + 4096, qs=256, o=far, os=256, c=p, s=p, n=9)
    for change in (dict(k=None), dict(v=None), dict(k=p + 4), dict(kvs=126), dict(kvs=124), dict(o=None),
                   dict(q=p + 4100), dict(o=far + 4), dict(qs=252), dict(os=258), dict(n=8), dict(c=None),
                   dict(o=p + 4096 + 1024), dict(o=p + 4096, os=260), dict(o=p), dict(v=far, o=far)):
        a = {**good, **change}
        assert ap(L, h, a["k"], a["v"], a["kvs"], a["q"], a["qs"], a["o"], a["os"], a["c"], a["s"], a["n"]) == -1, change


def test_call_after_a_failed_allocation(gpu):
    """An allocation that fails leaves no error behind for the calls that follow it."""
    ms = gpu
    say("paged: calls after a failed allocation")
    st = Setup(ms, [(3, 20)], 4, 2, 64, "f32", 16, seed=36)
    q = f32(3, 4 * 64, seed=37)
    d = ms.DeviceBuffer.from_array(q)
    for _ in range(2):
        with pytest.raises(ms.MSError, match="memory"):
            ms.DeviceBuffer(1 << 50)
        ms.paged_append(st.layer, st.batch, d, d, 128)
        with pytest.raises(ms.MSError, match="memory"):
            ms.DeviceBuffer(1 << 50)
        st.run_attention(q)
    c, s = ms.rope_table(64, 1e4, 3, wide=True)
    ms.synchronize()


def test_plan_of_the_longest_batch(gpu):
    """A batch whose even share of work passes 32 bits is planned, and refused for its number of
    blocks before anything is launched (the pools' and rows' addresses are not memory)."""
    ms = gpu
    say("paged: a plan past 32 bits")
    rows, page, n_pages = (1 << 20) - 1, 1 << 20, 1 << 10
    batch = ms.PagedBatch(page, n_pages, 1, rows, n_pages)
    batch.set([rows], [page * n_pages], np.arange(n_pages)[None])

    class At:
        def __init__(self, ptr):
            self.ptr = ptr

    layer = ms.PagedLayer(n_heads=1024, n_kv_heads=1024, head_dim=512, dtype=1, k=4096, v=8192)
    with pytest.raises(ms.MSError, match="too many rows for one call"):
        ms.paged_attention(layer, batch, At(4096), 1024 * 512, At(1 << 43), 1024 * 512)
