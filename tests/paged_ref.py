"""Helpers of the paged-cache tests: pools of every type, random page tables, and the
operators in 64 bits."""
import numpy as np

NAMES = {"f32": 0, "bf16": 1, "f16": 2}
# half a step of a rounding, relative to the value
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def encode(x, dtype):
    """fp32 values as the pool's elements, rounded to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x.copy()
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def decode(raw, dtype):
    if dtype == "bf16":
        return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return raw.astype(np.float64)


def raw_type(dtype):
    return {"f32": np.float32, "bf16": np.uint16, "f16": np.float16}[dtype]


class Setup:
    """A batch: sequences (new, length), pages in random order, pools with `fill` (NaN) in
    every slot that no sequence owns."""

    def __init__(self, ms, seqs, heads, kv, hd, dtype="f32", page=16, page_rows=0, window=0,
                 rot=0, scale=0.0, seed=0, spare=2, max_rows=None, shared=None):
        self.ms, self.seqs, self.heads, self.kv, self.hd = ms, seqs, heads, kv, hd
        self.dtype, self.page, self.window, self.rot = dtype, page, window, rot
        self.scale = scale
        rng = self.rng = np.random.default_rng(seed)
        self.new = [s[0] for s in seqs]
        self.len = [s[1] for s in seqs]
        self.rows = sum(self.new)
        used = [-(-n // page) for n in self.len]
        self.n_pages = sum(used) + spare
        self.max_pages = max(used + [1])
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.pages = np.full((len(seqs), self.max_pages), -1, np.int32)
        at = 0
        for s, u in enumerate(used):
            self.pages[s, :u] = order[at:at + u]
            at += u
        self.pr = page_rows or page
        shape = (self.n_pages, self.pr, kv, hd)
        self.pool = {}
        for n in "kv":
            x = np.full(shape, np.nan, np.float32)
            for s, l in enumerate(self.len):
                for p in range(0, l, page):
                    c = min(page, l - p)
                    x[self.pages[s, p // page], :c] = rng.standard_normal((c, kv, hd))
            self.pool[n] = encode(x, dtype)
        self.dk = ms.DeviceBuffer.from_array(self.pool["k"])
        self.dv = ms.DeviceBuffer.from_array(self.pool["v"])
        self.layer = ms.PagedLayer(n_heads=heads, n_kv_heads=kv, head_dim=hd, rot_dim=rot,
                                   window=window, dtype=NAMES[dtype], page_rows=page_rows,
                                   scale=scale, k=self.dk.ptr, v=self.dv.ptr)
        self.batch = ms.PagedBatch(page, self.n_pages, max(len(seqs), 1), max_rows or max(self.rows, 1),
                                   self.max_pages)
        self.batch.set(self.new, self.len, self.pages)

    def upload(self):
        self.dk.upload(self.pool["k"])
        self.dv.upload(self.pool["v"])

    def download(self):
        t = raw_type(self.dtype)
        return {"k": self.dk.download(t, self.pool["k"].shape),
                "v": self.dv.download(t, self.pool["v"].shape)}

    def slots(self, s, p0, p1):
        p = np.arange(p0, p1)
        return self.pages[s, p // self.page], p % self.page

    def row_of(self):
        """(sequence, position) of every row."""
        return [(s, p) for s, (n, l) in enumerate(zip(self.new, self.len)) for p in range(l - n, l)]

    def attend(self, q):
        """The rows' attention in 64 bits and, per value, how far an fp32 result may be off.

        A score sums hd products (each sum and product off by 2^-24 of the sum of
        magnitudes at most), its factors scale and log2(e) and the exponential add a few
        roundings of it, so p is off by d = (hd + 8) 2^-24 sum|q k| scale + 2^-22; numerator and
        denominator are off by that and by one rounding a key each: 2 (d + (keys + 8) 2^-24)
        of sum p |v|."""
        G = self.heads // self.kv
        out = np.zeros((self.rows, self.heads, self.hd))
        tol = np.zeros_like(out)
        q = q.reshape(self.rows, self.heads, self.hd).astype(np.float64)
        sc = self.scale or 1 / np.sqrt(self.hd)
        cache = {}
        for r, (s, p) in enumerate(self.row_of()):
            if s not in cache:
                g = self.slots(s, 0, self.len[s])
                cache = {s: [decode(self.pool[n][g], self.dtype) for n in "kv"]}
            lo = max(0, p - self.window + 1) if self.window else 0
            k, v = (x[lo:p + 1] for x in cache[s])
            for h in range(self.heads):
                kk, vv = k[:, h // G], v[:, h // G]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = kk @ q[r, h] * sc
                    e = np.exp(x - x.max())
                    w = e / e.sum()
                    out[r, h] = w @ vv
                    d = (self.hd + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[r, h])).max() * abs(sc) + 2.0 ** -22
                    tol[r, h] = 2 * (d + (p - lo + 9) * 2.0 ** -24) * (w @ np.abs(vv)) + 1e-30
        return out.reshape(self.rows, -1), tol.reshape(self.rows, -1)

    def run_attention(self, q, pad=0, behind=3):
        """The framework's result; rows behind the last and columns between the rows keep
        what they held."""
        n, ld = self.heads * self.hd, self.heads * self.hd + pad
        mark = np.float32(-777.0)
        buf = np.full((self.rows + behind, ld), mark, np.float32)
        src = buf.copy()
        src[:self.rows, :n] = q
        dq, do = self.ms.DeviceBuffer.from_array(src), self.ms.DeviceBuffer.from_array(buf)
        self.ms.paged_attention(self.layer, self.batch, dq, ld, do, ld)
        self.ms.synchronize()
        got = do.download(np.float32, buf.shape)
        assert np.all(got[self.rows:] == mark) and np.all(got[:, n:] == mark)
        return got[:self.rows, :n]

    def check_attention(self, seed=1, pad=0, scale=1.5):
        q = (np.random.default_rng(seed).standard_normal((self.rows, self.heads * self.hd)) * scale).astype(np.float32)
        want, tol = self.attend(q)
        got = self.run_attention(q, pad)
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got - want).max(), bad.sum())
        # rounding errors of either sign: well below the bound in the mean
        assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)
        return q, got
