"""ms_logits_process against 64 bits, and a serving step from append to the drawn token."""
import numpy as np
import pytest

from tests.paged_ref import Setup

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"\n[case] {msg}", flush=True)


def reference(x, rows, hist, ids, bias, masks):
    """64-bit result, and what fp32 may be off: at most six roundings of the largest
    intermediate magnitude (a bias sum rounds once an entry)."""
    x = x.astype(np.float64)
    V = x.shape[1]
    tol = np.zeros_like(x)
    for r, w in enumerate(rows):
        h = hist[w.history:w.history + w.n_prompt + w.n_generated]
        rep, freq, pres = (np.float64(np.float32(v)) for v in (w.repetition, w.frequency, w.presence))
        ok = (h >= 0) & (h < V)
        seen = np.unique(h[ok])
        made = np.bincount(h[w.n_prompt:][ok[w.n_prompt:]], minlength=V)
        with np.errstate(invalid="ignore"):
            x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
            mag = np.abs(x[r]) + np.abs(freq) * made + np.abs(pres) * (made > 0)
            x[r] -= np.where(made > 0, freq * made + pres, 0.0)
            b = ids[w.bias:w.bias + w.n_bias]
            val = bias[w.bias:w.bias + w.n_bias].astype(np.float64)
            on = (b >= 0) & (b < V)
            np.add.at(x[r], b[on], val[on])
            np.add.at(mag, b[on], np.abs(val[on]))
            n = np.bincount(b[on], minlength=V) if len(b) else np.zeros(V)
            tol[r] = np.where(np.isfinite(mag), mag, 0) * (6 + n) * 2.0 ** -24 + 1e-44
        if w.mask >= 0:
            bits = np.unpackbits(masks[w.mask].view(np.uint8), bitorder="little")[:V]
            x[r, bits == 0] = -np.inf
    return x, tol


def inputs(ms, rng, R, V, n_hist, n_bias, n_masks=2, density=0.4):
    rows, hist, ids, bias = [], [], [], []
    nh = nb = 0
    for r in range(R):
        h = int(rng.integers(0, n_hist + 1)) if r else n_hist
        b = int(rng.integers(0, n_bias + 1)) if r else n_bias
        few = rng.integers(-2, V + 2, max(1, h // 4))
        hist.append(few[rng.integers(0, len(few), h)])
        i = rng.integers(-1, V + 1, b)
        i[b // 2:] = i[:b - b // 2][::-1]  # the same ids again
        ids.append(i)
        bias.append(rng.uniform(-9, 9, b))
        p = int(rng.integers(0, h + 1))
        rows.append(ms.LogitsRow(repetition=float(rng.choice([1.0, 1.3, 0.8])), frequency=float(rng.choice([0, 0.3, -0.2])),
                                 presence=float(rng.choice([0, 0.7])), n_prompt=p, n_generated=h - p, history=nh,
                                 bias=nb, n_bias=b, mask=int(rng.integers(-1, n_masks))))
        nh += h
        nb += b
    masks = (rng.random((n_masks, (V + 31) // 32 * 32)) < density)
    masks = np.packbits(masks, axis=1, bitorder="little").view(np.uint32)
    return rows, np.concatenate(hist).astype(np.int32), np.concatenate(ids).astype(np.int32), \
        np.concatenate(bias).astype(np.float32), masks


def process(ms, x, V, rows, hist, ids, bias, masks, ld_out=None):
    """x [rows][stride]; ld_out None: in place."""
    buf = [ms.DeviceBuffer.from_array(a if a.size else np.zeros(1, a.dtype)) for a in (x, hist, ids, bias, masks)]
    R, ld = x.shape
    out = buf[0] if ld_out is None else ms.DeviceBuffer.from_array(np.full((R, ld_out), -777, np.float32))
    ms.logits_process(buf[0], ld, out, ld_out or ld, V, rows, buf[1], hist.size, buf[2], buf[3], ids.size, buf[4], len(masks))
    ms.synchronize()
    got = out.download(np.float32, (R, ld_out or ld))
    rest = x[:, V:] if ld_out is None else np.full((R, ld_out - V), -777, np.float32)
    assert np.array_equal(got[:, V:], rest)
    if ld_out is not None:
        assert np.array_equal(buf[0].download(np.float32, x.shape), x, equal_nan=True)
    return got[:, :V]


def check(got, want, tol):
    for kind in (np.isnan, np.isposinf, np.isneginf):
        assert np.array_equal(kind(got), kind(want))
    fine = np.isfinite(want)
    bad = np.abs(got[fine] - want[fine]) > tol[fine]
    assert not bad.any(), np.abs(got[fine] - want[fine]).max()


@pytest.mark.parametrize("R,V,pad,ld_out,n_hist,n_bias", [
    (1, 1, 0, None, 3, 2), (1, 31, 0, 31, 0, 0), (2, 33, 1, 40, 50, 5), (3, 4095, 0, 4096, 300, 40),
    (3, 4096, 0, None, 300, 0), (2, 4097, 3, None, 0, 300), (5, 32003, 2, 32003, 150, 5), (1, 262144, 0, 262144, 8192, 300),
    (2, 262143, 1, None, 70000, 1000), (70, 1000, 0, 1000, 64, 8), (64, 129, 3, 133, 10, 2)])
def test_logits(gpu, R, V, pad, ld_out, n_hist, n_bias):
    say(f"logits R={R} V={V} pad={pad} out={ld_out} history={n_hist} bias={n_bias}")
    rng = np.random.default_rng(V + R)
    args = inputs(gpu, rng, R, V, n_hist, n_bias)
    x = (rng.standard_normal((R, V + pad)) * 4).astype(np.float32)
    got = process(gpu, x, V, *args, ld_out=ld_out)
    check(got, *reference(x[:, :V], *args))


def test_logits_one_id(gpu):
    """One id many times: counted, and its biases added in their order (values whose sum in
    another order rounds differently)."""
    say("logits: one id many times")
    V, n = 500, 700
    bias = np.resize(np.array([1.0, 2.0 ** 24, 1.0, -2.0 ** 24, 2.0 ** -20], np.float32), n)
    ids = np.full(n, 77, np.int32)
    hist = np.full(9000, 77, np.int32)
    rows = [gpu.LogitsRow(frequency=0.25, presence=0.5, n_prompt=1000, n_generated=8000, n_bias=n)]
    x = np.zeros((1, V), np.float32)
    got = process(gpu, x, V, rows, hist, ids, bias, np.zeros((1, 16), np.uint32))
    acc = np.float32(0)
    for b in bias:
        acc = np.float32(acc + b)
    assert got[0, 77] == np.float32(np.float32(-0.25 * 8000 - 0.5) + acc)
    assert np.all(np.delete(got[0], 77) == 0)


def test_logits_values(gpu):
    """Infinities and NaN in and behind the mask; a mask that allows nothing; biases of
    minus infinity."""
    say("logits: odd values")
    V = 5000
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, V)).astype(np.float32)
    x[:, 10:40] = np.inf
    x[:, 40:70] = -np.inf
    x[:, 70:100] = np.nan
    hist = np.arange(0, 200, 3, dtype=np.int32)
    ids = np.array([11, 41, 71, 200, 201], np.int32)
    bias = np.array([-3, 3, 1, -np.inf, np.inf], np.float32)
    masks = np.zeros((2, (V + 31) // 32), np.uint32)
    masks[0] = 0x5A5A5A5A
    rows = [gpu.LogitsRow(repetition=1.5, frequency=0.5, n_generated=len(hist), n_bias=5, mask=m) for m in (-1, 0, 1)]
    got = process(gpu, x, V, rows, hist, ids, bias, masks, ld_out=V)
    check(got, *reference(x, rows, hist, ids, bias, masks))
    assert np.all(np.isneginf(got[2]))


def test_serving_step(gpu, oracle):
    """A step as a user runs it: append, attention, logits, draw.  The attention of a lone
    sequence is that of ms_attention on a contiguous cache, and the drawn token follows the
    grammar."""
    ms = gpu
    say("a serving step")
    H, kv, hd, rot, n0 = 8, 2, 128, 128, 90
    st = Setup(ms, [(20, n0), (1, 50)], H, kv, hd, "f32", 16, rot=rot, seed=11)
    nq, nkv = H * hd, kv * hd
    rng = np.random.default_rng(12)
    qkv = rng.standard_normal((21, nq + 2 * nkv)).astype(np.float32)
    d = ms.DeviceBuffer.from_array(qkv)

    class At:
        def __init__(self, off):
            self.ptr = d.ptr + 4 * off

    c, s = ms.rope_table(rot, 1e4, n0)
    ld = nq + 2 * nkv
    out = ms.DeviceBuffer(21 * nq * 4)
    ms.paged_append(st.layer, st.batch, At(nq), At(nq + nkv), ld, d, ld, d, ld, c, s, n0)
    ms.paged_attention(st.layer, st.batch, d, ld, out, nq)
    got = out.download(np.float32, (21, nq))
    # the same rows through ms_rope and ms_attention
    L = ms.LayerDesc(q_dim=nq, kv_dim=nkv, head_dim=hd, n_heads=H, n_kv_heads=kv, rot_dim=rot, theta=1e4,
                     cache_kind=ms.MS_CACHE_LINEAR, cache_len=128, clamp_reads=0)
    g = st.slots(0, 0, n0 - 20)
    cache = [np.zeros((128, nkv), np.float32) for _ in range(2)]
    for x, n in zip(cache, "kv"):
        x[:n0 - 20] = st.pool[n][g].reshape(-1, nkv)
    dc = [ms.DeviceBuffer.from_array(x) for x in cache]
    parts = [ms.DeviceBuffer.from_array(np.ascontiguousarray(qkv[:20, a:b])) for a, b in
             ((0, nq), (nq, nq + nkv), (nq + nkv, ld))]
    for p, n in zip(parts[:2], (H, kv)):
        ms.check(ms.lib().ms_rope(p.ptr, 20, n * hd, n, hd, rot, 1e4, n0 - 20))
    ref = ms.DeviceBuffer(20 * nq * 4)
    import ctypes as C
    ms.check(ms.lib().ms_attention(C.byref(L), parts[0].ptr, parts[1].ptr, parts[2].ptr, dc[0].ptr, dc[1].ptr, 20,
                                   n0 - 20, ref.ptr))
    want = ref.download(np.float32, (20, nq))
    st.pool.update(st.download())
    _, tol = st.attend(d.download(np.float32, (21, ld))[:, :nq])
    assert np.all(np.abs(got[:20] - want) <= 2 * tol[:20])  # both within tol of 64 bits
    # logits of the last rows: the attention's output as they are, a grammar and a draw
    V = nq
    masks = np.zeros((1, V // 32), np.uint32)
    masks[0, 5] = 0x10
    masks[0, 9] = 0x1
    rows = [ms.LogitsRow(repetition=1.2, n_generated=2, mask=0), ms.LogitsRow()]
    hist = np.array([5 * 32 + 4, 9], np.int32)
    dl = ms.DeviceBuffer.from_array(got[[19, 20]])
    dh, dm = ms.DeviceBuffer.from_array(hist), ms.DeviceBuffer.from_array(masks)
    ms.logits_process(dl, V, dl, V, V, rows, dh, 2, masks=dm, n_masks=1)
    x = dl.download(np.float32, (2, V))
    allowed = [5 * 32 + 4, 9 * 32]
    assert np.array_equal(np.flatnonzero(np.isfinite(x[0])), sorted(allowed)) and np.array_equal(x[1], got[20])
    for seed in range(5):
        dl.upload(x)
        tok = ms.sample(dl, V, 0.7, dh, 0, 1.0, seed)
        assert tok in allowed and tok == oracle.sample(x[0], 0.7, np.zeros(0, np.int32), 1.0, seed)[0]
