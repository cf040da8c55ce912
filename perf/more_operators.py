"""More operators of a serving step over a paged key/value cache: what is measured.

    append   the new rows of a ragged batch into the pages of their sequences: q and k normed
             head by head, then rotated to their positions; k and v as they are or in 8 bits with
             a scale for each position and kv head
    read     a sequence's keys and values back out of an 8-bit cache, in 32 bits
    attend   causal attention of the new rows over the pages: 8-bit pools, scores capped by a tanh
    sample   a token for each row of logits: temperature, top-k, top-p, min-p, a given random number

Where `own` is false, run() computes them in plain torch operations in 32 bits (the sampling in
64: what a token's weight adds up to decides which token it is); where it is true, through
ms_paged_append_ext, ms_paged_read, ms_paged_attention_ext and ms_sample_rows.  These calls are
asynchronous on the library's own stream, so results are read, and inputs changed, behind
mojostream_amd.synchronize() or a device-wide wait.
"""
import ctypes
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn,
       "i8": torch.int8}
_TOP = {"e4m3": 448.0, "i8": 127.0}  # the largest code of an 8-bit pool
_LEAST = 2.0 ** -126                 # the least scale
_EPS = 1e-6

# ---- the cases ---------------------------------------------------------------


def listed():
    return [
        # one user's next token in an E4B full-attention layer (512 dims a head, 128 of them
        # rotated) into an 8-bit cache; q, k and v normed: latency is all there is
        {"name": "append_e4b_full_1", "kind": "append", "heads": 8, "kv": 2, "hd": 512, "rot": 128, "pairs": False,
         "norm": "qkv", "gamma": True, "dtype": "e4m3", "page": 16, "seqs": 1, "chunks": 0, "new": 1, "ctx": 300},
        # a whole prompt of odd length at once, 14B class, q and k normed, an 8-bit cache
        {"name": "append_14b_prompt_3001", "kind": "append", "heads": 40, "kv": 8, "hd": 128, "rot": 128,
         "pairs": False, "norm": "qk", "gamma": True, "dtype": "e4m3", "page": 64, "seqs": 1, "chunks": 1,
         "new": 3001, "ctx": 3001},
        # a prefix of 700 positions of an E4B sliding layer, to be handed on
        {"name": "read_e4b_700", "kind": "read", "kv": 2, "hd": 256, "dtype": "e4m3", "page": 16, "ctx": 700},
        # a long document's cache, 14B class
        {"name": "read_14b_20011", "kind": "read", "kv": 8, "hd": 128, "dtype": "i8", "page": 32, "ctx": 20011},
        # one user's next token, E4B full attention, 8-bit cache
        {"name": "attend_e4b_full_1", "kind": "attend", "heads": 8, "kv": 2, "hd": 512, "dtype": "i8", "page": 16,
         "seqs": 1, "chunks": 0, "new": 1, "ctx": 700, "window": 0, "cap": 0.0},
        # a decode step of 48 users with contexts of very different length, 8-bit cache
        {"name": "attend_14b_48", "kind": "attend", "heads": 40, "kv": 8, "hd": 128, "dtype": "e4m3", "page": 16,
         "seqs": 48, "chunks": 0, "new": 1, "ctx": 4096, "window": 0, "cap": 0.0},
        # one user with a very long document, capped scores: the work has to be split over the keys
        {"name": "attend_demo_long", "kind": "attend", "heads": 8, "kv": 2, "hd": 128, "dtype": "i8", "page": 32,
         "seqs": 1, "chunks": 0, "new": 1, "ctx": 131065, "window": 0, "cap": 50.0},
        # a chunk of a long prompt, 14B class, 8-bit cache: the largest
        {"name": "attend_14b_chunk", "kind": "attend", "heads": 40, "kv": 8, "hd": 128, "dtype": "e4m3", "page": 64,
         "seqs": 1, "chunks": 1, "new": 4096, "ctx": 16384, "window": 0, "cap": 0.0},
        # three prompts in an E4B sliding layer, capped scores over a 16-bit cache
        {"name": "attend_e4b_sliding", "kind": "attend", "heads": 8, "kv": 2, "hd": 256, "dtype": "bf16", "page": 16,
         "seqs": 3, "chunks": 3, "new": 1000, "ctx": 5000, "window": 512, "cap": 30.0},
        # one user's next token from E4B's vocabulary
        {"name": "sample_262144_1", "kind": "sample", "rows": 1, "vocab": 262144, "pad": 0, "first": 0, "masked": 0.0},
        # a batch of users with settings of their own, every third row under a grammar
        {"name": "sample_262144_48", "kind": "sample", "rows": 48, "vocab": 262144, "pad": 0, "first": 0,
         "masked": 0.9},
        # a small vocabulary of odd size in rows of odd stride
        {"name": "sample_32003_5", "kind": "sample", "rows": 5, "vocab": 32003, "pad": 2, "first": 1, "masked": 0.5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "read", "attend", "attend", "sample"))
    if kind == "sample":
        return {"kind": kind, "rows": _log(rng, 1, 48), "vocab": _log(rng, 1000, 262144),
                "pad": rng.choice((0, 0, 1, 3)), "first": rng.randrange(len(_SETTINGS)),
                "masked": rng.choice((0.0, round(rng.uniform(0.0, 0.999), 3)))}
    hd = rng.choice((64, 128, 128, 256, 512))
    kv = rng.choice((1, 2, 4, 8) if hd <= 128 else (1, 2, 4))
    case = {"kind": kind, "kv": kv, "hd": hd, "page": rng.choice((1, 7, 16, 16, 32, 64, 128))}
    if kind == "read":
        case.update(dtype=rng.choice(("e4m3", "i8")), ctx=_log(rng, 1, 20000))
        return case
    case["heads"] = kv * rng.choice((1, 2, 4, 5, 8))
    if kind == "append":
        seqs = _log(rng, 1, 64)
        chunks = rng.choice((0, min(seqs, 1), min(seqs, 2)))
        new = _log(rng, 2, 3000) if chunks else 1
        case.update(dtype=rng.choice(("e4m3", "e4m3", "f32", "bf16", "f16")), rot=rng.choice((hd, hd, hd // 2, hd // 4)),
                    pairs=rng.choice((False, True)), norm=rng.choice(("", "qk", "qk", "qkv")),
                    gamma=rng.choice((True, True, False)), seqs=seqs, chunks=chunks, new=new,
                    ctx=max(new, _log(rng, 1, 4096)))
        return case
    dtype, how = rng.choice(("e4m3", "i8", "e4m3", "i8", "f32", "bf16", "f16")), rng.choice(("one", "batch", "chunk", "mixed"))
    cap = rng.choice((0.0, 30.0, 50.0)) if dtype in _TOP else rng.choice((20.0, 30.0, 50.0))
    window = rng.choice((0, 0, 512))
    if how == "one":
        seqs, chunks, new, ctx = 1, 0, 1, _log(rng, 1, 131072)
    elif how == "batch":
        seqs, chunks, new, ctx = _log(rng, 2, 48), 0, 1, _log(rng, 16, 4096)
    elif how == "chunk":
        seqs = chunks = rng.randint(1, 3)
        new = _log(rng, 2, 2048)
        ctx = max(new, _log(rng, 16, 8192))
    else:
        seqs, chunks, new = rng.randint(3, 24), rng.randint(1, 2), _log(rng, 2, 512)
        ctx = max(new, _log(rng, 64, 4096))
    case.update(dtype=dtype, seqs=seqs, chunks=chunks, new=new, ctx=ctx, window=window, cap=cap)
    return case


def lengths(case):
    """New tokens and tokens in all (the new ones among them) of every sequence: the first
    `chunks` bring about `new` tokens each, the others one; contexts spread from a tenth of `ctx`
    to all of it, that of the first."""
    if case["kind"] == "read":
        return [0], [case["ctx"]]
    new, total = [], []
    for b in range(case["seqs"]):
        f = 1.0 - 0.9 * ((b * 0.6180339887498949) % 1.0)
        t = max(1, int(case["new"] * (1.0 - 0.37 * (b % 3)))) if b < case["chunks"] else 1
        new.append(t)
        total.append(max(t, int(case["ctx"] * f)))
    return new, total


# What users ask for: temperature (0: the best token), top-k (0: all), top-p (1: all), min-p (0: all).
_SETTINGS = ((0.7, 0, 0.95, 0.0), (1.0, 50, 1.0, 0.0), (0.8, 40, 0.9, 0.05), (1.2, 0, 1.0, 0.02), (0.0, 0, 1.0, 0.0),
             (1.0, 0, 1.0, 0.0), (1.5, 1000, 0.6, 0.0), (1.0, 0, 0.5, 0.0))


# ---- inputs ---------------------------------------------------------------------


def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + what * 7919 + 54321) % (1 << 62))
    return g


def _randn(shape, seed, what):
    return torch.randn(shape, dtype=torch.float32, device="cuda", generator=_gen(seed, what))


def _tables(rot, n_pos):
    """cos and sin of pos * 10000^(-2i / rot), angles in 64 bits, rounded once."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    ang = torch.arange(n_pos, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-2 * i / rot)
    return ang.cos().float().contiguous(), ang.sin().float().contiguous()


def _to8(x, dtype):
    """x [..][hd] as 8-bit codes and the scale of each row of them."""
    # (by a tensor: torch divides by a number through its reciprocal, which is another rounding)
    s = (x.abs().amax(-1, keepdim=True) / torch.full((1,), _TOP[dtype], device=x.device)).clamp(min=_LEAST)
    y = x / s
    return (y.to(torch.float8_e4m3fn) if dtype == "e4m3" else y.round().clamp(-127, 127).to(torch.int8)), s[..., 0]


def _paged_inputs(case, seed):
    new, total = lengths(case)
    P, kv, hd, dtype = case["page"], case["kv"], case["hd"], case["dtype"]
    used = [-(-n // P) for n in total]
    n_pages, most = sum(used) + 3, max(used)
    order = torch.randperm(n_pages, device="cuda", generator=_gen(seed, 1)).int().cpu().numpy()
    pages = np.zeros((len(new), most), np.int32)
    at = 0
    for b, u in enumerate(used):
        pages[b, :u] = order[at:at + u]
        at += u
    st = {"case": case, "new": new, "total": total, "pages_h": pages, "n_pages": n_pages}
    for i, n in enumerate("kv"):
        x = _randn((n_pages, P, kv, hd), seed, 2 + i)
        if dtype in _TOP:
            # (rows of different size, as a model's are)
            x *= torch.exp(0.5 * _randn((n_pages, P, kv, 1), seed, 12 + i))
            st[n], s = _to8(x, dtype)
            st[n + "_scale"] = s.transpose(1, 2).contiguous()  # [page][kv head][slot]
        else:
            st[n] = x.to(_DT[dtype])
    n, t = torch.tensor(new, device="cuda"), torch.tensor(total, device="cuda")
    st["seq"] = torch.repeat_interleave(torch.arange(len(new), device="cuda"), n)
    st["start"] = torch.cumsum(n, 0) - n
    st["t"] = torch.arange(sum(new), device="cuda") - st["start"][st["seq"]]
    st["pos"] = (t - n)[st["seq"]] + st["t"]
    st["len"] = t
    st["pages"] = torch.from_numpy(pages).cuda().long()
    return st


def _append_inputs(case, seed):
    st = _paged_inputs(case, seed)
    H, kv, hd, rows = case["heads"], case["kv"], case["hd"], sum(st["new"])
    # the projections' output rows: q | k | v side by side
    st["qkv"] = _randn((rows, (H + 2 * kv) * hd), seed, 4) * torch.exp(0.5 * _randn((rows, 1), seed, 14))
    st["cos"], st["sin"] = _tables(case["rot"], max(st["total"]))
    st["gq"], st["gk"] = ((1.0 + 0.3 * _randn((hd,), seed, 5 + i)) if case["gamma"] else None for i in range(2))
    st["q_out"] = torch.zeros((rows, H * hd), device="cuda")
    return st


def _attend_inputs(case, seed):
    st = _paged_inputs(case, seed)
    # scores of standard deviation 2 and more: some keys matter more than others, and a cap bites
    st["q"] = _randn((sum(st["new"]), case["heads"] * case["hd"]), seed, 4).mul_(5.0 if case["cap"] else 2.0)
    st["out"] = torch.zeros_like(st["q"])
    return st


def _read_inputs(case, seed):
    st = _paged_inputs(case, seed)
    st["k_out"], st["v_out"] = (torch.zeros((case["ctx"], case["kv"] * case["hd"]), device="cuda") for _ in range(2))
    return st


def _sample_inputs(case, seed):
    R, V = case["rows"], case["vocab"]
    x = _randn((R, V + case["pad"]), seed, 1).mul_(2.5)
    # a few candidates above the rest
    few = torch.randint(0, V, (R, 24), device="cuda", generator=_gen(seed, 2))
    x.scatter_add_(1, few, 5.0 + 2.0 * _randn((R, 24), seed, 3))
    if case["masked"]:  # what a grammar leaves of every third row
        off = torch.rand((R, V), device="cuda", generator=_gen(seed, 4)) < case["masked"]
        off &= (torch.arange(R, device="cuda") % 3 == 2)[:, None]
        x[:, :V].masked_fill_(off, -math.inf)
    set_h = np.array([_SETTINGS[(case["first"] + r) % len(_SETTINGS)] for r in range(R)], np.float32)
    st = {"case": case, "logits": x[:, :V], "set_h": set_h,
          "u": torch.rand((R,), device="cuda", generator=_gen(seed, 5))}
    st["temp"], st["top_k"], st["top_p"], st["min_p"] = torch.from_numpy(set_h).cuda().double().T[:, :, None]
    st["ids"], st["kept"] = (torch.zeros((R,), dtype=torch.int32, device="cuda") for _ in range(2))
    st["prob"] = torch.zeros((R,), device="cuda")
    return st


_INPUTS = {"append": _append_inputs, "read": _read_inputs, "attend": _attend_inputs, "sample": _sample_inputs}


def prepare(case, seed):
    st = _INPUTS[case["kind"]](case, seed)
    if own:  # the handle that a program keeps: its batch, set once a step for all layers
        _handles(st)
    return st


# ---- the plain forms ----------------------------------------------------------------


def _rotate(x, cos, sin, rot, pairs):
    """x [rows][heads][hd], cos and sin [rows][rot / 2]"""
    c, s = cos[:, None], sin[:, None]
    if pairs:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _normed(x, on, gamma):
    if not on:
        return x
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
    return y if gamma is None else y * gamma


def _append_plain(st):
    c = st["case"]
    H, kv, hd, P = c["heads"], c["kv"], c["hd"], c["page"]
    q, k, v = (t.unflatten(1, (-1, hd)) for t in st["qkv"].split((H * hd, kv * hd, kv * hd), 1))
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    q = _rotate(_normed(q, "q" in c["norm"], st["gq"]), cos, sin, c["rot"], c["pairs"])
    k = _rotate(_normed(k, "k" in c["norm"], st["gk"]), cos, sin, c["rot"], c["pairs"])
    v = _normed(v, "v" in c["norm"], None)
    st["q_out"] = q.flatten(1)
    page, slot = st["pages"][st["seq"], st["pos"] // P], st["pos"] % P
    out = {"q": st["q_out"], "k": st["k"], "v": st["v"]}
    if c["dtype"] in _TOP:
        out.update(k_scale=st["k_scale"], v_scale=st["v_scale"])
        k, st["k_scale"][page, :, slot] = _to8(k, c["dtype"])
        v, st["v_scale"][page, :, slot] = _to8(v, c["dtype"])
        st["k"].view(torch.uint8)[page, slot] = k.view(torch.uint8)
        st["v"].view(torch.uint8)[page, slot] = v.view(torch.uint8)
    else:
        st["k"][page, slot] = k.to(st["k"].dtype)
        st["v"][page, slot] = v.to(st["v"].dtype)
    return out


def _values(st, n, pages):
    """The pool's values of `pages`, in 32 bits: [..][slots][kv][hd]"""
    if st["case"]["dtype"] not in _TOP:
        return st[n][pages].float()
    x = st[n].view(torch.uint8)[pages].view(st[n].dtype).float()
    return x * st[n + "_scale"][pages].transpose(-1, -2)[..., None]


def _read_plain(st):
    n = st["case"]["ctx"]
    k, v = (_values(st, x, st["pages"][0]).flatten(0, 1)[:n].flatten(1) for x in "kv")
    return {"k": k, "v": v}


def _attend_plain(st):
    """Every sequence padded to the longest."""
    c = st["case"]
    H, kv, hd, B = c["heads"], c["kv"], c["hd"], c["seqs"]
    G, T = H // kv, max(st["new"])
    k, v = (_values(st, x, st["pages"]).flatten(1, 2).transpose(1, 2).contiguous() for x in "kv")
    N = k.shape[2]
    j = torch.arange(T, device="cuda")
    at = torch.clamp(st["start"][:, None] + j, max=len(st["seq"]) - 1)
    q = st["q"][at].view(B, T, kv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, kv, G * T, hd)
    s = (q @ k.transpose(-1, -2)).view(B, kv, G, T, N) * (1.0 / math.sqrt(hd))
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    n = torch.arange(N, device="cuda")
    p = st["pos"][at]
    seen = (n <= p[..., None]) & (n < st["len"][:, None, None])
    if c["window"]:
        seen &= n > p[..., None] - c["window"]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    w = (e / e.sum(-1, keepdim=True)).view(B, kv, G * T, N)
    o = (w @ v).view(B, kv, G, T, hd).permute(0, 3, 1, 2, 4).reshape(B, T, H * hd)
    return o[st["seq"], st["t"]]


def _sample_plain(st):
    V = st["case"]["vocab"]
    x, by = torch.sort(st["logits"], dim=1, descending=True, stable=True)
    x = x.double()
    best = st["temp"] == 0
    w = torch.exp((x - x[:, :1]) / torch.where(best, 1.0, st["temp"]))
    rank = torch.arange(V, device="cuda")
    in_k = (x > -math.inf) & (rank < torch.where(best, 1.0, torch.where(st["top_k"] > 0, st["top_k"], float(V))))
    w = w * in_k
    upto = torch.cumsum(w, 1)
    keep = in_k & (w >= st["min_p"]) & ((st["top_p"] >= 1) | (upto - w < st["top_p"] * upto[:, -1:]))
    w = w * keep
    run_w = torch.zeros_like(w).scatter_(1, by, w)  # in the order of the ids
    upto = torch.cumsum(run_w, 1)
    total = upto[:, -1:]
    ids = torch.argmax((upto > st["u"].double()[:, None] * total).to(torch.uint8), 1, keepdim=True)
    return {"ids": ids[:, 0].int(), "kept": keep.sum(1).int(), "prob": (run_w.gather(1, ids) / total)[:, 0].float()}


# ---- the framework's calls ------------------------------------------------------------


def _handles(st):
    import mojostream_amd as ms
    ms.init(0)
    torch.cuda.synchronize()  # the library's stream does not wait for torch's, which fills the inputs
    c = st["case"]
    st["ms"] = ms
    if c["kind"] == "sample":
        st["rows"] = (ms.SampleRow * c["rows"])(*[
            ms.SampleRow(temperature=float(t), top_k=int(k), top_p=float(p), min_p=float(m)) for t, k, p, m in st["set_h"]])
        return
    st["batch"] = ms.PagedBatch(c["page"], st["n_pages"], len(st["new"]), max(1, sum(st["new"])), st["pages_h"].shape[1])
    st["batch"].set(st["new"], st["total"], st["pages_h"])
    norm, gammas = c.get("norm", ""), {n: st[n].data_ptr() if st.get(n) is not None else None for n in ("gq", "gk")}
    st["layer"] = ms.PagedLayerExt(
        base=ms.PagedLayer(n_heads=c.get("heads", c["kv"]), n_kv_heads=c["kv"], head_dim=c["hd"], rot_dim=c.get("rot", 0),
                           window=c.get("window", 0),
                           dtype={"f32": ms.MS_KV_F32, "bf16": ms.MS_KV_BF16, "f16": ms.MS_KV_F16,
                                  "e4m3": ms.MS_KV_E4M3, "i8": ms.MS_KV_I8}[c["dtype"]],
                           k=st["k"].data_ptr(), v=st["v"].data_ptr()),
        k_scale=st["k_scale"].data_ptr() if c["dtype"] in _TOP else None,
        v_scale=st["v_scale"].data_ptr() if c["dtype"] in _TOP else None, score_cap=c.get("cap", 0.0),
        norm=("q" in norm) * ms.MS_NORM_Q + ("k" in norm) * ms.MS_NORM_K + ("v" in norm) * ms.MS_NORM_V,
        norm_eps=_EPS, q_gamma=gammas["gq"], k_gamma=gammas["gk"],
        rope=ms.MS_ROPE_PAIRS if c.get("pairs") else ms.MS_ROPE_HALVES)


def _append_own(st):
    ms, c, x = st["ms"], st["case"], st["qkv"]
    H, kv, hd = c["heads"], c["kv"], c["hd"]
    p = x.data_ptr()
    ms.check(ms.lib().ms_paged_append_ext(ctypes.byref(st["layer"]), st["batch"].h, p + 4 * H * hd, p + 4 * (H + kv) * hd,
                                          x.shape[1], p, x.shape[1], st["q_out"].data_ptr(), H * hd,
                                          st["cos"].data_ptr(), st["sin"].data_ptr(), st["cos"].shape[0]))
    out = {"q": st["q_out"], "k": st["k"], "v": st["v"]}
    if c["dtype"] in _TOP:
        out.update(k_scale=st["k_scale"], v_scale=st["v_scale"])
    return out


def _read_own(st):
    ms, n = st["ms"], st["k_out"].shape[1]
    ms.check(ms.lib().ms_paged_read(ctypes.byref(st["layer"]), st["batch"].h, 0, 0, st["case"]["ctx"],
                                    st["k_out"].data_ptr(), st["v_out"].data_ptr(), n))
    return {"k": st["k_out"], "v": st["v_out"]}


def _attend_own(st):
    ms, n = st["ms"], st["q"].shape[1]
    ms.check(ms.lib().ms_paged_attention_ext(ctypes.byref(st["layer"]), st["batch"].h, st["q"].data_ptr(), n,
                                             st["out"].data_ptr(), n))
    return st["out"]


def _sample_own(st):
    ms, c, x = st["ms"], st["case"], st["logits"]
    ms.check(ms.lib().ms_sample_rows(x.data_ptr(), x.stride(0), c["rows"], c["vocab"], st["rows"], st["u"].data_ptr(),
                                     st["ids"].data_ptr(), st["prob"].data_ptr(), st["kept"].data_ptr()))
    return {"ids": st["ids"], "kept": st["kept"], "prob": st["prob"]}


def run(st):
    kind = st["case"]["kind"]
    if own:
        return {"append": _append_own, "read": _read_own, "attend": _attend_own, "sample": _sample_own}[kind](st)
    return {"append": _append_plain, "read": _read_plain, "attend": _attend_plain, "sample": _sample_plain}[kind](st)


# ---- what a pass cannot do without --------------------------------------------------


def work(case):
    if case["kind"] == "sample":
        return {"bytes": 4.0 * case["rows"] * (case["vocab"] + 4), "flops": 4.0 * case["rows"] * case["vocab"]}
    new, total = lengths(case)
    kv, hd = case["kv"], case["hd"]
    eight = case["dtype"] in _TOP
    # a position's keys and values of all heads, with their scales
    row = 2.0 * kv * ((hd + 4) if eight else hd * (4 if case["dtype"] == "f32" else 2))
    if case["kind"] == "read":
        return {"bytes": total[0] * (row + 8.0 * kv * hd), "flops": 2.0 * total[0] * kv * hd}
    H, rows = case["heads"], sum(new)
    if case["kind"] == "append":
        norms = sum(n in case["norm"] for n in "kv") * kv + ("q" in case["norm"]) * H
        return {"bytes": 4.0 * rows * ((2 * H + 2 * kv) * hd + case["rot"]) + rows * row,
                "flops": 3.0 * rows * (H + kv) * case["rot"] + 4.0 * rows * norms * hd + 4.0 * eight * rows * kv * hd}
    W = case["window"] or max(total)
    keys = sum(min(n, W + t - 1) for t, n in zip(new, total))
    pairs = sum(sum(min(p + 1, W) for p in range(n - t, n)) for t, n in zip(new, total))
    return {"bytes": keys * row + 8.0 * rows * H * hd, "flops": 4.0 * pairs * H * hd}


# ---- the same in 64 bits --------------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        if case["kind"] == "sample":
            return _sample_exact(case, seed)
        return {"append": _append_exact, "read": _read_exact, "attend": _attend_exact}[case["kind"]](case, seed)


# the values that an e4m3 code's low seven bits stand for, but NaN
_E4M3 = [math.ldexp(c & 7, -9) if c < 8 else math.ldexp(8 + (c & 7), (c >> 3) - 10) for c in range(127)]


def _nearest(x, dtype):
    """(codes' values, scales) of 64-bit rows x [..][hd]: the nearest value, an even code where two are."""
    big = x.abs().max(-1, keepdim=True).values
    s = torch.maximum((big / _TOP[dtype]).float(), torch.full_like(big, _LEAST, dtype=torch.float32))
    y = x / s.double()
    if dtype == "i8":
        return y.round(), s[..., 0]
    table = torch.tensor(_E4M3, dtype=torch.float64, device=x.device)
    mid = (table[1:] + table[:-1]) / 2
    low = torch.bucketize(y.abs().contiguous(), mid)                    # a value at a middle goes down
    high = torch.bucketize(y.abs().contiguous(), mid, right=True)       # and up here
    code = torch.where(low % 2 == 0, low, high)
    return torch.where(y < 0, -table[code], table[code]), s[..., 0]


def _norm_exact(x, on, gamma):
    if not on:
        return x
    y = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + _EPS)
    return y * (1.0 if gamma is None else gamma.double())


def _append_exact(case, seed):
    st = _append_inputs(case, seed)
    H, kv, hd, rot, P = case["heads"], case["kv"], case["hd"], case["rot"], case["page"]
    rows = st["qkv"].double()
    k, v = (st[n].to(torch.float64 if case["dtype"] in _TOP else st[n].dtype).double() for n in "kv")
    ks, vs = (st[n].double() if case["dtype"] in _TOP else None for n in ("k_scale", "v_scale"))
    cos, sin = st["cos"].double(), st["sin"].double()
    i = torch.arange(rot // 2, device="cuda")
    first, second = (2 * i, 2 * i + 1) if case["pairs"] else (i, i + rot // 2)
    q, r = torch.empty((rows.shape[0], H, hd), dtype=torch.float64, device="cuda"), 0
    for b, (t, n) in enumerate(zip(st["new"], st["total"])):
        x = rows[r:r + t].view(t, H + 2 * kv, hd)
        p = torch.arange(n - t, n, device="cuda")
        x = [_norm_exact(x[:, :H], "q" in case["norm"], st["gq"]), _norm_exact(x[:, H:H + kv], "k" in case["norm"], st["gk"]),
             _norm_exact(x[:, H + kv:], "v" in case["norm"], None)]
        turn = torch.complex(cos[p], sin[p])[:, None]
        for j in range(2):
            z = torch.complex(x[j][..., first].contiguous(), x[j][..., second].contiguous()) * turn
            x[j] = x[j].clone()
            x[j][..., first], x[j][..., second] = z.real, z.imag
        q[r:r + t] = x[0]
        page, slot = torch.from_numpy(st["pages_h"][b]).cuda().long()[p // P], p % P
        for pool, scale, y in ((k, ks, x[1]), (v, vs, x[2])):
            if scale is None:
                pool[page, slot] = y
            else:
                pool[page, slot], s = _nearest(y, case["dtype"])
                scale[page, :, slot] = s.double()
        r += t
    out = {"q": q.view(-1, H * hd), "k": k, "v": v}
    if ks is not None:
        out.update(k_scale=ks, v_scale=vs)
    return out


def _rows_exact(st, n, b):
    """A sequence's keys or values in 64 bits: [positions][kv][hd]"""
    page = torch.from_numpy(st["pages_h"][b, :-(-st["total"][b] // st["case"]["page"])]).cuda().long()
    x = st[n].to(torch.float32)[page].double()
    if st["case"]["dtype"] in _TOP:
        x = x * st[n + "_scale"][page].double().permute(0, 2, 1).unsqueeze(-1)
    return x.flatten(0, 1)[:st["total"][b]]


def _read_exact(case, seed):
    st = _paged_inputs(case, seed)
    return {n: _rows_exact(st, n, 0).flatten(1) for n in "kv"}


def _attend_exact(case, seed):
    st = _attend_inputs(case, seed)
    H, kv, hd, W = case["heads"], case["kv"], case["hd"], case["window"]
    q = st["q"].double().view(-1, H, hd)
    out = torch.zeros_like(q)
    r = 0
    for b, (t, n) in enumerate(zip(st["new"], st["total"])):
        keys, vals = _rows_exact(st, "k", b), _rows_exact(st, "v", b)
        for t0 in range(0, t, 1024):
            t1 = min(t, t0 + 1024)
            p = torch.arange(n - t + t0, n - t + t1, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")
            off = (j > p) | (j <= p - W) if W else j > p
            for h in range(H):
                g = h * kv // H
                s = torch.matmul(q[r + t0:r + t1, h], keys[:, g].t().contiguous()) / math.sqrt(hd)
                if case["cap"]:
                    s = torch.tanh(s / case["cap"]) * case["cap"]
                out[r + t0:r + t1, h] = torch.softmax(s.masked_fill(off, -math.inf), -1) @ vals[:, g].contiguous()
        r += t
    return out.view(-1, H * hd)


def _sample_exact(case, seed):
    st = _sample_inputs(case, seed)
    logits, u = st["logits"].double().cpu().numpy(), st["u"].double().cpu().numpy()
    R, V = logits.shape
    ids, kept, prob = np.zeros(R, np.int32), np.zeros(R, np.int32), np.zeros(R)
    for r in range(R):
        x, (temp, k, p, least) = logits[r], st["set_h"][r].astype(np.float64)
        order = np.lexsort((np.arange(V), -x))
        order = order[:1 if temp == 0 else int(k) if k else V]
        order = order[np.isfinite(x[order])]
        w = np.exp((x[order] - x[order[0]]) / (temp or 1.0))
        n = len(w)
        if p < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(w), p * w.sum())))
        n = min(n, int(np.count_nonzero(w >= least)))
        by_id = np.argsort(order[:n], kind="stable")
        upto = np.cumsum(w[:n][by_id])
        at = min(n - 1, int(np.searchsorted(upto, u[r] * upto[-1], side="right")))
        ids[r], kept[r], prob[r] = order[:n][by_id][at], n, w[by_id[at]] / upto[-1]
    return {"ids": ids, "kept": kept, "prob": prob}
