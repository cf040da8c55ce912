"""The operators of a serving step over a paged key/value cache: what is measured.

    append   the new rows of a ragged batch: q and k rotated to their positions, k and v
             written into the pages of their sequences
    attend   causal attention of those rows over the pages, all keys or a sliding window
    logits   penalties for tokens that occurred, biases, and grammar masks on the logits

Where `own` is false, run() computes them in plain torch operations in 32 bits; where it
is true, through ms_paged_append, ms_paged_attention and ms_logits_process: these calls are
asynchronous on the library's own stream, so results are read, and inputs changed, behind
mojostream_amd.synchronize() or a device-wide wait.
"""
import ctypes
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# ---- the cases ---------------------------------------------------------------


def listed():
    return [
        # one user's next token in an E4B full-attention layer (512 dims a head, 128 of
        # them rotated), a cache of the activations' own type: latency is all there is
        {"name": "append_e4b_full_1", "kind": "append", "heads": 8, "kv": 2, "hd": 512, "rot": 128,
         "dtype": "f32", "page": 16, "seqs": 1, "chunks": 0, "new": 1, "ctx": 300},
        # a decode step of 37 users on a 14B-class layer
        {"name": "append_14b_37", "kind": "append", "heads": 40, "kv": 8, "hd": 128, "rot": 128,
         "dtype": "bf16", "page": 32, "seqs": 37, "chunks": 0, "new": 1, "ctx": 2500},
        # a whole prompt of odd length at once
        {"name": "append_14b_prompt_3001", "kind": "append", "heads": 40, "kv": 8, "hd": 128,
         "rot": 128, "dtype": "bf16", "page": 64, "seqs": 1, "chunks": 1, "new": 3001, "ctx": 3001},
        # one user's next token, E4B full attention
        {"name": "attend_e4b_full_1", "kind": "attend", "heads": 8, "kv": 2, "hd": 512,
         "dtype": "f32", "page": 16, "seqs": 1, "chunks": 0, "new": 1, "ctx": 700, "window": 0},
        # a decode step of 48 users with contexts of very different length
        {"name": "attend_14b_48", "kind": "attend", "heads": 40, "kv": 8, "hd": 128,
         "dtype": "bf16", "page": 16, "seqs": 48, "chunks": 0, "new": 1, "ctx": 4096, "window": 0},
        # one user with a very long document: the work has to be split over the keys
        {"name": "attend_demo_long", "kind": "attend", "heads": 8, "kv": 2, "hd": 128,
         "dtype": "f16", "page": 32, "seqs": 1, "chunks": 0, "new": 1, "ctx": 131065, "window": 0},
        # a chunk of a long prompt, 14B class: the largest
        {"name": "attend_14b_chunk", "kind": "attend", "heads": 40, "kv": 8, "hd": 128,
         "dtype": "bf16", "page": 64, "seqs": 1, "chunks": 1, "new": 4096, "ctx": 16384, "window": 0},
        # three prompts in an E4B sliding layer, cache of the activations' own type
        {"name": "attend_e4b_sliding", "kind": "attend", "heads": 8, "kv": 2, "hd": 256,
         "dtype": "f32", "page": 16, "seqs": 3, "chunks": 3, "new": 1000, "ctx": 5000, "window": 512},
        # chunked prefill beside decoding, E4B full attention: three chunks among single tokens
        {"name": "attend_e4b_mixed", "kind": "attend", "heads": 8, "kv": 2, "hd": 512,
         "dtype": "bf16", "page": 32, "seqs": 15, "chunks": 3, "new": 301, "ctx": 2300, "window": 0},
        # one user's next token from E4B's vocabulary: penalties, biases and a grammar
        {"name": "logits_262144_1", "kind": "logits", "rows": 1, "vocab": 262144, "pad": 0,
         "history": 600, "bias": 40, "mask": 0.02},
        # a batch of users with long histories, half of them under a grammar
        {"name": "logits_262144_48", "kind": "logits", "rows": 48, "vocab": 262144, "pad": 0,
         "history": 4000, "bias": 300, "mask": 0.3},
        # a small vocabulary of odd size in rows of odd stride
        {"name": "logits_32003_5", "kind": "logits", "rows": 5, "vocab": 32003, "pad": 2,
         "history": 150, "bias": 5, "mask": 0.5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "logits"))
    if kind == "logits":
        vocab = _log(rng, 1000, 262144)
        return {"kind": kind, "rows": _log(rng, 1, 48), "vocab": vocab, "pad": rng.choice((0, 0, 1, 3)),
                "history": _log(rng, 1, 8000), "bias": rng.choice((0, _log(rng, 1, 300))),
                "mask": rng.choice((0.0, round(math.exp(rng.uniform(math.log(0.001), 0)), 4)))}
    hd = rng.choice((64, 128, 128, 256, 512))
    kv = rng.choice((1, 2, 4, 8) if hd <= 128 else (1, 2, 4))
    case = {"kind": kind, "heads": kv * rng.choice((1, 2, 4, 5, 8)), "kv": kv, "hd": hd,
            "dtype": rng.choice(("f32", "bf16", "bf16", "f16")), "page": rng.choice((16, 32, 64, 128))}
    if kind == "append":
        seqs = _log(rng, 1, 64)
        chunks = rng.choice((0, min(seqs, 1), min(seqs, 2)))
        new = _log(rng, 2, 3000) if chunks else 1
        case.update(rot=rng.choice((hd, hd, hd // 2, hd // 4)), seqs=seqs, chunks=chunks, new=new,
                    ctx=max(new, _log(rng, 1, 4096)))
        return case
    how = rng.choice(("one", "batch", "chunk", "mixed"))
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
    case.update(seqs=seqs, chunks=chunks, new=new, ctx=ctx, window=window)
    return case


def lengths(case):
    """New tokens and tokens in all (the new ones among them) of every sequence: the first
    `chunks` bring about `new` tokens each, the others one; contexts spread from a tenth of `ctx`
    to all of it, that of the first."""
    new, total = [], []
    for b in range(case["seqs"]):
        f = 1.0 - 0.9 * ((b * 0.6180339887498949) % 1.0)
        t = max(1, int(case["new"] * (1.0 - 0.37 * (b % 3)))) if b < case["chunks"] else 1
        new.append(t)
        total.append(max(t, int(case["ctx"] * f)))
    return new, total


# ---- inputs ---------------------------------------------------------------------


def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + what * 7919 + 12345) % (1 << 62))
    return g


def _randn(shape, seed, what):
    return torch.randn(shape, dtype=torch.float32, device="cuda", generator=_gen(seed, what))


def _tables(rot, n_pos):
    """cos and sin of pos * 10000^(-2i / rot), angles in 64 bits, rounded once."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    ang = torch.arange(n_pos, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-2 * i / rot)
    return ang.cos().float().contiguous(), ang.sin().float().contiguous()


def _paged_inputs(case, seed):
    new, total = lengths(case)
    P, kv, hd = case["page"], case["kv"], case["hd"]
    used = [-(-n // P) for n in total]
    n_pages, most = sum(used) + 3, max(used)
    order = torch.randperm(n_pages, device="cuda", generator=_gen(seed, 1)).int().cpu().numpy()
    pages = np.zeros((len(new), most), np.int32)
    at = 0
    for b, u in enumerate(used):
        pages[b, :u] = order[at:at + u]
        at += u
    dt = _DT[case["dtype"]]
    st = {"case": case, "new": new, "total": total, "pages_h": pages, "n_pages": n_pages,
          "k": _randn((n_pages, P, kv, hd), seed, 2).to(dt), "v": _randn((n_pages, P, kv, hd), seed, 3).to(dt)}
    n, t = torch.tensor(new, device="cuda"), torch.tensor(total, device="cuda")
    st["seq"] = torch.repeat_interleave(torch.arange(len(new), device="cuda"), n)
    st["start"] = torch.cumsum(n, 0) - n
    st["t"] = torch.arange(sum(new), device="cuda") - st["start"][st["seq"]]
    st["pos"] = (t - n)[st["seq"]] + st["t"]
    st["len"] = t
    st["pages"] = torch.from_numpy(pages).cuda().long()
    return st


def prepare(case, seed):
    kind = case["kind"]
    if kind == "logits":
        st = _logits_inputs(case, seed)
    else:
        st = _paged_inputs(case, seed)
        rows = sum(st["new"])
        if kind == "append":
            # the projections' output rows: q | k | v side by side
            st["qkv"] = _randn((rows, (case["heads"] + 2 * case["kv"]) * case["hd"]), seed, 4)
            st["cos"], st["sin"] = _tables(case["rot"], max(st["total"]))
            st["q_out"] = torch.zeros((rows, case["heads"] * case["hd"]), device="cuda")
        else:
            # scores of standard deviation 2: some keys matter more than others
            st["q"] = _randn((rows, case["heads"] * case["hd"]), seed, 4).mul_(2.0)
            st["out"] = torch.zeros_like(st["q"])
    if own:  # the handle that a program keeps: its batch, set once a step for all layers
        _handles(st)
    return st


def _logits_inputs(case, seed):
    R, V, H, NB = case["rows"], case["vocab"], case["history"], case["bias"]
    ld = V + case["pad"]
    rng = np.random.RandomState(seed % (1 << 31))
    st = {"case": case, "logits": _randn((R, ld), seed, 1).mul_(3.0)[:, :V], "out": torch.zeros((R, V), device="cuda")}
    # text repeats itself: half of the history comes from a few hundred tokens
    hist = rng.randint(0, V, (R, H))
    few = rng.randint(0, V, 200)
    hist = np.where(rng.rand(R, H) < 0.5, few[rng.randint(0, 200, (R, H))], hist)
    ids = rng.randint(0, V, (R, NB))
    if NB > 3:
        ids[:, NB // 2] = ids[:, 0]
    st["hist"] = torch.from_numpy(hist.astype(np.int32)).cuda()
    st["bias_ids"] = torch.from_numpy(ids.astype(np.int32)).cuda()
    st["bias"] = torch.from_numpy(rng.uniform(-5, 5, (R, NB)).astype(np.float32)).cuda()
    st["prompt"] = [H // 3 if r % 3 else 0 for r in range(R)]
    st["rep"] = np.array([(1.2, 1.0, 1.05)[r % 3] for r in range(R)], np.float32)
    st["freq"] = np.array([(0.1, 0.3, 0.0)[r % 3] for r in range(R)], np.float32)
    st["pres"] = np.array([(0.0, 0.5, 0.2)[r % 3] for r in range(R)], np.float32)
    # every second row is under a grammar; two grammars at most
    words = -(-V // 32)
    n_masks = 0 if case["mask"] == 0 else 1 if R < 3 else 2
    bits = torch.rand((max(n_masks, 1), words * 32), device="cuda", generator=_gen(seed, 5)) < case["mask"]
    w = (bits.view(-1, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
    st["masks"] = torch.where(w >= 1 << 31, w - (1 << 32), w).int().contiguous()
    st["mask_row"] = [-1 if n_masks == 0 or r % 2 else (r // 2) % n_masks for r in range(R)]
    dev = {k: torch.from_numpy(st[k]).cuda()[:, None] for k in ("rep", "freq", "pres")}
    st.update(rep_d=dev["rep"], freq_d=dev["freq"], pres_d=dev["pres"],
              prompt_d=torch.tensor(st["prompt"], device="cuda")[:, None],
              mask_d=torch.tensor(st["mask_row"], device="cuda"))
    return st


# ---- the plain forms ----------------------------------------------------------------


def _rotate(x, cos, sin, rot):
    """x [rows][heads][hd], cos and sin [rows][rot / 2]"""
    h = rot // 2
    a, b, c, s = x[..., :h], x[..., h:rot], cos[:, None], sin[:, None]
    return torch.cat((a * c - b * s, a * s + b * c, x[..., rot:]), -1)


def _append_plain(st):
    c = st["case"]
    H, kv, hd, P = c["heads"], c["kv"], c["hd"], c["page"]
    q, k, v = st["qkv"].split((H * hd, kv * hd, kv * hd), 1)
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    st["q_out"] = _rotate(q.unflatten(1, (H, hd)), cos, sin, c["rot"]).flatten(1)
    slot = st["pages"][st["seq"], st["pos"] // P] * P + st["pos"] % P
    st["k"].view(-1, kv, hd)[slot] = _rotate(k.unflatten(1, (kv, hd)), cos, sin, c["rot"]).to(st["k"].dtype)
    st["v"].view(-1, kv, hd)[slot] = v.unflatten(1, (kv, hd)).to(st["v"].dtype)
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _attend_plain(st):
    """Every sequence padded to the longest."""
    c = st["case"]
    H, kv, hd, B = c["heads"], c["kv"], c["hd"], c["seqs"]
    G, T = H // kv, max(st["new"])
    keys = [st[n][st["pages"]].float().flatten(1, 2).transpose(1, 2).contiguous() for n in ("k", "v")]
    N = keys[0].shape[2]
    j = torch.arange(T, device="cuda")
    at = torch.clamp(st["start"][:, None] + j, max=len(st["seq"]) - 1)
    q = st["q"][at].view(B, T, kv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, kv, G * T, hd)
    s = (q @ keys[0].transpose(-1, -2)).view(B, kv, G, T, N) * (1.0 / math.sqrt(hd))
    n = torch.arange(N, device="cuda")
    p = st["pos"][at]
    seen = (n <= p[..., None]) & (n < st["len"][:, None, None])
    if c["window"]:
        seen &= n > p[..., None] - c["window"]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    w = (e / e.sum(-1, keepdim=True)).view(B, kv, G * T, N)
    o = (w @ keys[1]).view(B, kv, G, T, hd).permute(0, 3, 1, 2, 4).reshape(B, T, H * hd)
    return o[st["seq"], st["t"]]


def _logits_plain(st):
    c = st["case"]
    R, V, H = c["rows"], c["vocab"], c["history"]
    x, ids = st["logits"], st["hist"].long()
    made = (torch.arange(H, device="cuda") >= st["prompt_d"]).float()
    count = torch.zeros((R, V), device="cuda").scatter_add_(1, ids, made)
    seen = torch.zeros((R, V), dtype=torch.bool, device="cuda").scatter_(1, ids, True)
    y = torch.where(seen, torch.where(x > 0, x / st["rep_d"], x * st["rep_d"]), x)
    y = y - st["freq_d"] * count - st["pres_d"] * (count > 0)
    y = y.scatter_add(1, st["bias_ids"].long(), st["bias"])
    bits = (st["masks"][:, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
    allowed = bits.flatten(1)[:, :V].bool()[st["mask_d"].clamp(min=0)] | (st["mask_d"] < 0)[:, None]
    return y.masked_fill(~allowed, -math.inf)


# ---- the framework's calls ------------------------------------------------------------


def _handles(st):
    import mojostream_amd as ms
    ms.init(0)
    torch.cuda.synchronize()  # the library's stream does not wait for torch's, which fills the inputs
    c = st["case"]
    st["ms"] = ms
    if c["kind"] == "logits":
        st["rows"] = (ms.LogitsRow * c["rows"])(*[
            ms.LogitsRow(repetition=float(st["rep"][r]), frequency=float(st["freq"][r]),
                         presence=float(st["pres"][r]), mask=st["mask_row"][r], history=r * c["history"],
                         n_prompt=st["prompt"][r], n_generated=c["history"] - st["prompt"][r],
                         bias=r * c["bias"], n_bias=c["bias"]) for r in range(c["rows"])])
        return
    st["batch"] = ms.PagedBatch(c["page"], st["n_pages"], c["seqs"], sum(st["new"]), st["pages_h"].shape[1])
    st["batch"].set(st["new"], st["total"], st["pages_h"])
    st["layer"] = ms.PagedLayer(n_heads=c["heads"], n_kv_heads=c["kv"], head_dim=c["hd"], rot_dim=c.get("rot", 0),
                                window=c.get("window", 0), dtype={"f32": ms.MS_KV_F32, "bf16": ms.MS_KV_BF16,
                                                                  "f16": ms.MS_KV_F16}[c["dtype"]],
                                k=st["k"].data_ptr(), v=st["v"].data_ptr())


def _append_own(st):
    ms, c, x = st["ms"], st["case"], st["qkv"]
    H, kv, hd = c["heads"], c["kv"], c["hd"]
    p = x.data_ptr()
    ms.check(ms.lib().ms_paged_append(ctypes.byref(st["layer"]), st["batch"].h, p + 4 * H * hd, p + 4 * (H + kv) * hd,
                                      x.shape[1], p, x.shape[1], st["q_out"].data_ptr(), H * hd,
                                      st["cos"].data_ptr(), st["sin"].data_ptr(), st["cos"].shape[0]))
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _attend_own(st):
    ms, n = st["ms"], st["q"].shape[1]
    ms.check(ms.lib().ms_paged_attention(ctypes.byref(st["layer"]), st["batch"].h, st["q"].data_ptr(), n,
                                         st["out"].data_ptr(), n))
    return st["out"]


def _logits_own(st):
    ms, c, x = st["ms"], st["case"], st["logits"]
    ms.check(ms.lib().ms_logits_process(x.data_ptr(), x.stride(0), st["out"].data_ptr(), c["vocab"], c["rows"],
                                        c["vocab"], st["rows"], st["hist"].data_ptr(), st["hist"].numel(),
                                        st["bias_ids"].data_ptr(), st["bias"].data_ptr(), st["bias"].numel(),
                                        st["masks"].data_ptr(), st["masks"].shape[0]))
    return st["out"]


def run(st):
    kind = st["case"]["kind"]
    if kind == "append":
        return _append_own(st) if own else _append_plain(st)
    if kind == "attend":
        return _attend_own(st) if own else _attend_plain(st)
    return _logits_own(st) if own else _logits_plain(st)


# ---- what a pass cannot do without --------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "logits":
        R, V = case["rows"], case["vocab"]
        under = 0 if case["mask"] == 0 else (R + 1) // 2  # rows under a grammar: only what it allows is read
        read = 4.0 * V * (R - under + under * min(1.0, case["mask"])) + (min(under, 2) * V / 8)
        return {"bytes": read + 4.0 * R * V + R * (4.0 * case["history"] + 8.0 * case["bias"]),
                "flops": 2.0 * R * (case["history"] + case["bias"])}
    new, total = lengths(case)
    H, kv, hd = case["heads"], case["kv"], case["hd"]
    es = 4 if case["dtype"] == "f32" else 2
    rows = sum(new)
    if kind == "append":
        return {"bytes": 4.0 * rows * ((2 * H + 2 * kv) * hd + case["rot"]) + 2.0 * es * rows * kv * hd,
                "flops": 3.0 * rows * (H + kv) * case["rot"]}
    W = case["window"] or max(total)
    keys = sum(min(n, W + t - 1) for t, n in zip(new, total))
    pairs = sum(sum(min(p + 1, W) for p in range(n - t, n)) for t, n in zip(new, total))
    return {"bytes": 2.0 * es * keys * kv * hd + 8.0 * rows * H * hd, "flops": 4.0 * pairs * H * hd}


# ---- the same in 64 bits --------------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        if case["kind"] == "logits":
            return _logits_exact(case, seed)
        st = _paged_inputs(case, seed)
        return _append_exact(case, st, seed) if case["kind"] == "append" else _attend_exact(case, st, seed)


def _append_exact(case, st, seed):
    H, kv, hd, rot, P = case["heads"], case["kv"], case["hd"], case["rot"], case["page"]
    rows = _randn((sum(st["new"]), (H + 2 * kv) * hd), seed, 4).double()
    k, v, q = st["k"].double(), st["v"].double(), torch.empty((rows.shape[0], H, hd), dtype=torch.float64, device="cuda")
    f = torch.exp(-math.log(10000.0) * 2.0 / rot * torch.arange(rot // 2, dtype=torch.float64, device="cuda"))
    r = 0
    for b, (t, n) in enumerate(zip(st["new"], st["total"])):
        x = rows[r:r + t].view(t, H + 2 * kv, hd)
        p = torch.arange(n - t, n, device="cuda")
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), p.double()[:, None] * f)[:, None]
        z = torch.complex(x[:, :H + kv, :rot // 2].contiguous(), x[:, :H + kv, rot // 2:rot].contiguous()) * turn
        y = torch.cat((z.real, z.imag, x[:, :H + kv, rot:]), -1)
        q[r:r + t] = y[:, :H]
        page = torch.from_numpy(st["pages_h"][b]).cuda().long()[p // P]
        k[page, p % P] = y[:, H:]
        v[page, p % P] = x[:, H + kv:]
        r += t
    return {"q": q.view(-1, H * hd), "k": k, "v": v}


def _attend_exact(case, st, seed):
    H, kv, hd, W = case["heads"], case["kv"], case["hd"], case["window"]
    q = _randn((sum(st["new"]), H * hd), seed, 4).mul_(2.0).double().view(-1, H, hd)
    out = torch.zeros_like(q)
    r = 0
    for b, (t, n) in enumerate(zip(st["new"], st["total"])):
        page = torch.from_numpy(st["pages_h"][b, :-(-n // case["page"])]).cuda().long()
        keys, vals = (st[x][page].flatten(0, 1)[:n].double() for x in ("k", "v"))
        for t0 in range(0, t, 1024):
            t1 = min(t, t0 + 1024)
            p = torch.arange(n - t + t0, n - t + t1, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")
            off = (j > p) | (j <= p - W) if W else j > p
            for h in range(H):
                g = h * kv // H
                s = torch.matmul(q[r + t0:r + t1, h], keys[:, g].t().contiguous()) / math.sqrt(hd)
                out[r + t0:r + t1, h] = torch.softmax(s.masked_fill(off, -math.inf), -1) @ vals[:, g].contiguous()
        r += t
    return out.view(-1, H * hd)


def _logits_exact(case, seed):
    st = _logits_inputs(case, seed)
    x = st["logits"].double().cpu().numpy()
    hist, ids, bias = (st[n].cpu().numpy() for n in ("hist", "bias_ids", "bias"))
    masks = st["masks"].cpu().numpy().view(np.uint32)
    for r in range(case["rows"]):
        made = np.bincount(hist[r, st["prompt"][r]:], minlength=case["vocab"])
        seen = np.unique(hist[r])
        x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / st["rep"][r], x[r, seen] * np.float64(st["rep"][r]))
        x[r] -= np.float64(st["freq"][r]) * made + np.float64(st["pres"][r]) * (made > 0)
        np.add.at(x[r], ids[r], bias[r].astype(np.float64))
        if st["mask_row"][r] >= 0:
            bits = np.unpackbits(masks[st["mask_row"][r]].view(np.uint8), bitorder="little")[:case["vocab"]]
            x[r, bits == 0] = -np.inf
    return x
