"""Helpers of the tests of 8-bit pools, normed heads and capped scores: the codes, and the operators
in 64 bits."""
import numpy as np

from tests.paged_ref import HALF, Setup, decode

CODES = {"e4m3": 4, "i8": 5}
TOP = {"e4m3": 448.0, "i8": 127.0}
MAX32 = float(np.finfo(np.float32).max)


def _e4m3_values():
    """The value of every code: sign, four bits of exponent (offset 7), three of mantissa."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c >> 7, -v, v)


E4M3 = _e4m3_values()
VALUE = {"e4m3": E4M3, "i8": np.arange(256).astype(np.uint8).view(np.int8).astype(np.float64)}


def nearest(y, dtype):
    """Codes nearest to y, even where two are as near, and whether y is so near a middle that 64 bits
    do not say which."""
    y = np.asarray(y, np.float64)
    if dtype == "i8":
        c = np.rint(y)
        return c.astype(np.int8).view(np.uint8), np.abs(np.abs(y - np.trunc(y)) - 0.5) < 1e-9
    table = E4M3[:127]
    a = np.abs(y)
    hi = np.clip(np.searchsorted(table, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = table[hi] - a, a - table[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    near = (np.abs(up - down) < 1e-9 * np.maximum(a, 2.0 ** -9)) & (up != down)
    return (code | np.where(y < 0, 128, 0)).astype(np.uint8), near


def scale_of(x, dtype):
    """The scale of rows x [..][hd] (64 bits)."""
    with np.errstate(over="ignore", invalid="ignore"):
        s = np.maximum((np.abs(x).max(-1) / TOP[dtype]).astype(np.float32), np.float32(2.0 ** -126))
        s = np.where(np.abs(x).max(-1) > MAX32, np.float32(np.nan), s)
        over = np.isfinite(s) & (s.astype(np.float64) * TOP[dtype] > MAX32)
        s = np.where(over, np.nextafter(s, np.float32(0)), s)
    return np.where(np.isfinite(s), s, np.float32(np.nan))


class SetupExt(Setup):
    """Setup over any pool, with a cap: 8-bit pools hold the codes of its random values; in
    every slot that no sequence owns the scales are NaN and the codes the type's worst."""

    def __init__(self, ms, seqs, heads, kv, hd, dtype="e4m3", page=16, page_rows=0, window=0,
                 cap=0.0, spread=0.0, norm=0, eps=1e-6, gamma=False, pairs=False, **more):
        self.cap, self.kind, self.eight = cap, dtype, dtype in CODES
        super().__init__(ms, seqs, heads, kv, hd, "f32" if self.eight else dtype, page, page_rows,
                         window, **more)
        base = self.layer
        self.scales = self.gammas = None
        if self.eight:
            self.raw, self.scales = {}, {}
            rng = np.random.default_rng(99)
            for n in "kv":
                x = self.pool[n].astype(np.float64)
                x *= 2.0 ** (spread * rng.standard_normal(x.shape[:3] + (1,)))
                self.fill(n, x)
            self.dk, self.dv = (ms.DeviceBuffer.from_array(self.raw[n]) for n in "kv")
            self.dks, self.dvs = (ms.DeviceBuffer.from_array(self.scales[n]) for n in "kv")
            base = ms.PagedLayer(n_heads=heads, n_kv_heads=kv, head_dim=hd, rot_dim=self.rot, window=window,
                                 dtype=CODES[dtype], page_rows=page_rows, scale=self.scale, k=self.dk.ptr,
                                 v=self.dv.ptr)
        self.norm, self.eps, self.pairs = norm, np.float32(eps), pairs
        if gamma:
            g = np.random.default_rng(7)
            self.gammas = [(1 + 0.3 * g.standard_normal(hd)).astype(np.float32) for _ in range(2)]
            self.dg = [ms.DeviceBuffer.from_array(x) for x in self.gammas]
        self.layer = ms.PagedLayerExt(
            base=base, k_scale=self.dks.ptr if self.eight else None, v_scale=self.dvs.ptr if self.eight else None,
            score_cap=cap, norm=norm, norm_eps=eps, q_gamma=self.dg[0].ptr if gamma else None,
            k_gamma=self.dg[1].ptr if gamma else None, rope=int(pairs))

    def fill(self, n, x):
        """Pool n from the values x [pages][rows][kv][hd]; NaN: a slot that nobody owns."""
        owned = ~np.isnan(x[..., 0])
        s = scale_of(np.nan_to_num(x), self.kind)
        with np.errstate(invalid="ignore"):
            c, _ = nearest(np.nan_to_num(x) / s[..., None], self.kind)
        s[~owned] = np.nan
        c[~owned] = 0x7F if self.kind == "e4m3" else 0x80
        self.raw[n], self.scales[n] = c, np.ascontiguousarray(s.transpose(0, 2, 1))
        self.pool[n] = self.values(n)

    def values(self, n):
        """The pool's values in 64 bits."""
        return VALUE[self.kind][self.raw[n]] * self.scales[n].transpose(0, 2, 1)[..., None].astype(np.float64)

    def upload(self):
        if not self.eight:
            return super().upload()
        for n, d, ds in (("k", self.dk, self.dks), ("v", self.dv, self.dvs)):
            d.upload(self.raw[n])
            ds.upload(self.scales[n])
            self.pool[n] = self.values(n)

    def download8(self):
        """Codes and scales of both pools: {"k": .., "v": ..}, the same."""
        return ({n: d.download(np.uint8, self.raw[n].shape) for n, d in (("k", self.dk), ("v", self.dv))},
                {n: d.download(np.float32, self.scales[n].shape) for n, d in (("k", self.dks), ("v", self.dvs))})

    def attend(self, q, only=None):
        """The rows' attention in 64 bits, capped, and per value how far an fp32 result may be off: what
        Setup.attend derives (an 8-bit key's scale is one more rounding of its score, q's 22 bits four: its eight spare
        ones), and with a cap what tanh adds.  tanh never grows an error; its own: below 0.6 2^-23 of it; above, from
        t = e^-2|z| <= 0.3 with an argument off by 2^-23, so (1 - t) / (1 + t) by at most 2^-21 of it; z itself is off by 2^-22 of it, which
        moves tanh by less than 2^-22 of it: 2^-20 of the capped score in all.
        An 8-bit value's probability times its scale is taken in two fp16 parts: off by 2^-22 of itself (eight spare
        ones hold that) or, where that is less, by half of fp16's smallest step, 2^-25, in units of 2^-7 of a power of two that
        is at most twice the largest scale the row attends to, the best key having a probability of 1 at least: 2^-31 of that
        scale for each key, times its code.
        only: of these rows."""
        G = self.heads // self.kv
        out, tol = (np.zeros((self.rows, self.heads, self.hd)) for _ in range(2))
        q = q.reshape(self.rows, self.heads, self.hd).astype(np.float64)
        sc = self.scale or 1 / np.sqrt(self.hd)
        cache = {}
        for r, (s, p) in enumerate(self.row_of()):
            if only is not None and r not in only:
                continue
            if s not in cache:
                g = self.slots(s, 0, self.len[s])
                cache = {s: [decode(self.pool[n][g], self.dtype) for n in "kv"]}
                if self.eight:
                    cache[s] += [np.abs(VALUE[self.kind][self.raw["v"][g]]), self.scales["v"].transpose(0, 2, 1)[g]]
            lo = max(0, p - self.window + 1) if self.window else 0
            k, v = (x[lo:p + 1] for x in cache[s][:2])
            for h in range(self.heads):
                kk, vv = k[:, h // G], v[:, h // G]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = kk @ q[r, h] * sc
                    d = (self.hd + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[r, h])).max() * abs(sc) + 2.0 ** -22
                    if self.cap:
                        x = self.cap * np.tanh(x / self.cap)
                        d += 2.0 ** -20 * np.abs(x).max()
                    e = np.exp(x - x.max())
                    w = e / e.sum()
                    out[r, h] = w @ vv
                    tol[r, h] = 2 * (d + (p - lo + 9) * 2.0 ** -24) * (w @ np.abs(vv)) + 1e-30
                    if self.eight:
                        code, scale = (x[lo:p + 1, h // G] for x in cache[s][2:])
                        tol[r, h] += 2.0 ** -31 * np.float64(scale.max()) * code.sum(0)
        return out.reshape(self.rows, -1), tol.reshape(self.rows, -1)

    def check(self, seed=1, pad=0, scale=1.5, only=None):
        q = (np.random.default_rng(seed).standard_normal((self.rows, self.heads * self.hd)) * scale).astype(np.float32)
        want, tol = self.attend(q, only)
        got = self.run_attention(q, pad)
        at = slice(None) if only is None else list(only)
        bad = ~(np.abs(got - want)[at] <= tol[at])
        assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got - want).max(), bad.sum())
        return q, got


def append_in_64(st, q, k, v, cos, sin):
    """What ms_paged_append_ext computes before it rounds, in 64 bits: q, k, v [rows][heads][hd], and how far fp32
    may be off (q, and k and v of pools that are not 8-bit)."""
    pos = np.array([p for _, p in st.row_of()])
    out, tol = [], []
    for i, x in enumerate((q, k, v)):
        x = x.reshape(st.rows, -1, st.hd).astype(np.float64)
        t = np.zeros_like(x)
        if st.norm >> i & 1:
            with np.errstate(invalid="ignore", divide="ignore"):
                x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(st.eps))
            if st.gammas and i < 2:
                x = x * st.gammas[i].astype(np.float64)
            t = 3 * 2.0 ** -24 * np.abs(x)  # the factor, its product, gamma's
        if i < 2 and st.rot:
            h = st.rot // 2
            a, b = (np.arange(0, st.rot, 2), np.arange(1, st.rot, 2)) if st.pairs else (np.arange(h), np.arange(h, st.rot))
            c, s = cos[pos][:, None].astype(np.float64), sin[pos][:, None].astype(np.float64)
            xa, xb, ta, tb = x[..., a], x[..., b], t[..., a], t[..., b]
            y, u = x.copy(), t.copy()
            y[..., a], y[..., b] = xa * c - xb * s, xa * s + xb * c
            # (two products and a sum: three roundings at most)
            u[..., a] = np.abs(c) * ta + np.abs(s) * tb + 2.0 ** -23 * (np.abs(xa * c) + np.abs(xb * s))
            u[..., b] = np.abs(s) * ta + np.abs(c) * tb + 2.0 ** -23 * (np.abs(xa * s) + np.abs(xb * c))
            x, t = y, u
        out.append(x)
        tol.append(t)
    return out, tol


__all__ = ["CODES", "E4M3", "HALF", "MAX32", "SetupExt", "TOP", "VALUE", "append_in_64", "decode", "nearest", "scale_of"]
