"""The operators of many-stream decoding over a paged key-value cache, as calls that can be timed and checked.

A case is a dict of plain values; its "kind" says which operator it calls:

  append    block tables, slots and positions of a step's tokens from the requests' lengths
  qk        RMS norm of every query and key head, then the rotation; with "store" the keys and values go into the cache
  attn      attention of one new token a request over its pages
  logp      log probabilities of given tokens, the entropy, the best alternatives

prepare() makes what a serving loop holds before the call, run() is one pass (own: the library's entry points; else the
same from elementary torch operations in 32 bits), exact() the definition in 64 bits.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16}
SIZE = {"f32": 4, "f16": 2}


def listed():
    return [
        # a decode step's bookkeeping for 64 streams of the 2048-position backbone: the smallest call
        {"name": "append_decode", "kind": "append", "n": 64, "past": 1900, "new": 1, "page": 64, "short": False},
        # the prompts of many requests admitted at once, some on a cached prefix, a pool that runs out before the last ones
        {"name": "append_prompts", "kind": "append", "n": 500, "past": 300, "new": 1500, "page": 16, "short": True},
        # a 64-stream decode step of the backbone's 16 heads in F16, keys and values into their pages
        {"name": "qk_decode", "kind": "qk", "tok": 64, "hq": 16, "hkv": 16, "d": 64, "nd": 64, "mode": 2, "base": 1e4,
         "dt": "f16", "store": True, "cdt": "f16", "page": 64},
        # a batch of prompts, shared heads, F32 activations into an F16 cache with pages of an odd size
        {"name": "qk_prompts", "kind": "qk", "tok": 9001, "hq": 24, "hkv": 8, "d": 128, "nd": 128, "mode": 2, "base": 5e5,
         "dt": "f32", "store": True, "cdt": "f16", "page": 50},
        # a whole text scored in one pass, without a cache: adjacent pairs, a part of each head rotated
        {"name": "qk_partial", "kind": "qk", "tok": 1500, "hq": 20, "hkv": 5, "d": 96, "nd": 48, "mode": 0, "base": 1e4,
         "dt": "f16", "store": False, "cdt": "f16", "page": 64},
        # one stream of the backbone a few hundred tokens in, F32 activations: latency
        {"name": "attn_one", "kind": "attn", "n": 1, "lo": 300, "hi": 300, "hkv": 16, "g": 1, "d": 64, "page": 64,
         "dt": "f32", "cdt": "f16", "cap": 0.0, "window": 0},
        # 64 streams of the backbone anywhere in its 2048 positions
        {"name": "attn_streams", "kind": "attn", "n": 64, "lo": 1, "hi": 2048, "hkv": 16, "g": 1, "d": 64, "page": 64,
         "dt": "f16", "cdt": "f16", "cap": 0.0, "window": 0},
        # long requests with shared heads
        {"name": "attn_long", "kind": "attn", "n": 8, "lo": 1500, "hi": 65000, "hkv": 8, "g": 4, "d": 128, "page": 32,
         "dt": "f16", "cdt": "f16", "cap": 0.0, "window": 0},
        # an F32 cache with pages of an odd size, capped scores, a sliding window, five heads to a key head
        {"name": "attn_f32_window", "kind": "attn", "n": 23, "lo": 0, "hi": 7001, "hkv": 4, "g": 5, "d": 80, "page": 24,
         "dt": "f32", "cdt": "f32", "cap": 30.0, "window": 4001},
        # the speech tokens of a 64-stream step, four alternatives each
        {"name": "logp_step", "kind": "logp", "rows": 64, "vocab": 8194, "dt": "f32", "top": 4, "scale": 1.0, "masked": False},
        # one stream over a large vocabulary
        {"name": "logp_one", "kind": "logp", "rows": 1, "vocab": 151936, "dt": "f16", "top": 20, "scale": 1.25, "masked": False},
        # scoring whole texts: every position's logits, some tokens masked out
        {"name": "logp_texts", "kind": "logp", "rows": 4000, "vocab": 8194, "dt": "f32", "top": 8, "scale": 0.8, "masked": True},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["append", "qk", "qk", "attn", "attn", "attn", "logp", "logp"])
    if kind == "append":
        n = _log(rng, 1, 1500)
        new = rng.choice([1, 1, _log(rng, 2, max(2, min(4000, 750000 // n)))])
        return {"kind": kind, "n": n, "past": _log(rng, 1, 4000), "new": new, "page": rng.choice([1, 7, 16, 32, 50, 64, 128]),
                "short": rng.random() < 0.3}
    if kind == "qk":
        d, g, hkv = rng.choice([32, 64, 64, 80, 96, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 8, 16])
        nd = rng.choice([d, d, d // 2])
        tok = _log(rng, 1, max(2, min(9001, 9001 * 40 * 128 // (d * hkv * (g + 2)))))
        return {"kind": kind, "tok": tok, "hq": g * hkv, "hkv": hkv, "d": d, "nd": nd, "mode": rng.choice([0, 2, 2]),
                "base": rng.choice([1e4, 5e5, 1e6]), "dt": rng.choice(["f16", "f32"]), "store": rng.random() < 0.6,
                "cdt": rng.choice(["f16", "f16", "f32"]), "page": rng.choice([1, 10, 16, 32, 50, 64, 128])}
    if kind == "attn":
        d, hkv, g = rng.choice([32, 64, 64, 80, 96, 128, 128, 256]), rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
        dt = rng.choice(["f16", "f16", "f32"])
        cdt = "f16" if dt == "f16" else rng.choice(["f16", "f32"])
        n = _log(rng, 1, 256)
        hi = _log(rng, 1, max(2, min(130000, 260000 * 8 * 128 * 2 // (n * hkv * d * SIZE[cdt]))))
        lo = rng.choice([hi, 0, hi // 8])
        return {"kind": kind, "n": n, "lo": lo, "hi": hi, "hkv": hkv, "g": g, "d": d, "page": rng.choice([5, 8, 16, 24, 32, 64, 64, 128, 256]),
                "dt": dt, "cdt": cdt, "cap": rng.choice([0.0, 0.0, 0.0, 20.0]), "window": rng.choice([0, 0, 0, max(1, hi // 3)])}
    vocab = _log(rng, 60, 260000)
    dt = rng.choice(["f16", "f32"])
    return {"kind": kind, "rows": _log(rng, 1, max(2, min(8000, 32000000 // vocab))), "vocab": vocab, "dt": dt,
            "top": rng.choice([0, 1, 4, 20, 32]), "scale": rng.choice([1.0, 0.7, 1.25]), "masked": rng.random() < 0.4}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _spread(lo, hi, n):
    """n whole numbers evenly spread over [lo, hi] (hi alone for one)."""
    return np.linspace(hi if n == 1 else lo, hi, n).round().astype(np.int64)


def _lengths(case):
    """(past, new) of an append case's requests, before the seed's shuffle: a few pasts of 0, a few requests with nothing new."""
    n = case["n"]
    past = _spread(0, case["past"], n)
    new = np.full(n, 1, dtype=np.int64) if case["new"] == 1 else _spread(1, case["new"], n)
    new[15::16] = 0
    return past, new


def _tables(n, counts, width, perm):
    """[n, width] page tables: the first counts[s] entries of row s taken from perm in order, -1 behind them."""
    idx = torch.arange(width, device="cuda").expand(n, width)
    first = torch.cumsum(counts, 0) - counts
    src = (first[:, None] + idx).clamp(max=max(0, perm.numel() - 1))
    return torch.where(idx < counts[:, None], perm[src], torch.full_like(src, -1)).to(torch.int32)


def _angles(npos, nd, base):
    """theta of every position and pair: the position times theta_scale again and again, each product rounded to f32."""
    ts = np.float32(float(np.float32(base)) ** float(np.float32(-2.0) / np.float32(nd)))
    th = np.empty((npos, nd // 2), dtype=np.float32)
    t = np.arange(npos, dtype=np.float32)
    for i in range(nd // 2):
        th[:, i] = t
        t = t * ts
    return th.astype(np.float64)


POSITIONS = 4096


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    host = np.random.RandomState(int(seed) % (1 << 31))
    kind = case["kind"]
    randn = lambda *s, dt="f32": torch.randn(*s, device="cuda", generator=g, dtype=TYPES[dt])  # noqa: E731
    perm = lambda n: torch.randperm(n, device="cuda", generator=g)  # noqa: E731
    ints = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda().to(torch.int32)  # noqa: E731

    if kind == "append":
        n, page = case["n"], case["page"]
        past, new = _lengths(case)
        past, new = past[host.permutation(n)], new[host.permutation(n)]
        have, width = -(-past // page), -(-int((case["past"] + case["new"])) // page)
        need = -(-(past + new) // page) - have
        free = int(need.sum()) * 3 // 4 if case["short"] else int(need.sum()) + 100
        pages = perm(int(have.sum()) + free)
        counts = ints(have).long()
        stack = torch.full((pages.numel(),), -1, dtype=torch.int32, device="cuda")
        stack[:free] = pages[int(have.sum()):].to(torch.int32)
        return {"case": case, "n_past": ints(past), "n_new": ints(new), "free": stack,
                "n_free": torch.tensor([free], dtype=torch.int32, device="cuda"),
                "tables": _tables(n, counts, width, pages), "slots": int(new.sum()) + int(new.sum()) // 32 + 1}

    if kind == "qk":
        tok, hq, hkv, d = case["tok"], case["hq"], case["hkv"], case["d"]
        width = (hq + 2 * hkv) * d
        rows = randn(tok, width + 64, dt=case["dt"]) * 1.5
        cut = lambda a, h: rows[:, a * d:(a + h) * d].unflatten(1, (h, d))  # noqa: E731
        st = {"case": case, "q": cut(0, hq), "k": cut(hq, hkv), "v": cut(hq + hkv, hkv), "gq": 1 + 0.1 * randn(d),
              "gk": 1 + 0.1 * randn(d), "pos": torch.randint(0, POSITIONS, (tok,), device="cuda", generator=g, dtype=torch.int32)}
        theta = torch.from_numpy(_angles(POSITIONS, case["nd"], case["base"]))
        st["cos"], st["sin"] = theta.cos().float().cuda(), theta.sin().float().cuda()   # the rotation table a program keeps
        if own:
            from chatterbox_amdvulkan_amd import cbxops as C
            st["rope"] = C.RopeCache(case["nd"], mode=case["mode"], freq_base=case["base"], n_pos=POSITIONS)
        if case["store"]:
            page = case["page"]
            pages = -(-(tok + 100) // page)
            slots = perm(pages * page)[:tok].to(torch.int32)
            slots[tok - tok // 20:] = -1                        # a padded batch: its last rows belong to no request
            st["slots"] = slots
            st["kc"] = randn(pages, hkv, page, d, dt=case["cdt"])
            st["vc"] = randn(pages, hkv, page, d, dt=case["cdt"])
        return st

    if kind == "attn":
        n, hkv, d, page = case["n"], case["hkv"], case["d"], case["page"]
        lens = _spread(case["lo"], case["hi"], n)[host.permutation(n)]
        counts = -(-lens // page)
        pages = int(counts.sum()) + 3
        width = max(1, -(-case["hi"] // page))
        return {"case": case, "q": randn(n, hkv * case["g"], d, dt=case["dt"]) * 2, "lens": ints(lens), "scale": d ** -0.5,
                "tables": _tables(n, ints(counts).long(), width, perm(pages)),
                "kc": randn(pages, hkv, page, d, dt=case["cdt"]), "vc": randn(pages, hkv, page, d, dt=case["cdt"])}

    rows, vocab = case["rows"], case["vocab"]
    x = (randn(rows, vocab) * 2.5).to(TYPES[case["dt"]])
    ids = torch.randint(0, vocab, (rows,), device="cuda", generator=g, dtype=torch.int32)
    if case["masked"]:                                          # tokens that may not come next: never the given one
        gone = torch.rand(rows, vocab, device="cuda", generator=g) < 0.2
        gone.scatter_(1, ids.long()[:, None], False)
        x.masked_fill_(gone, float("-inf"))
    return {"case": case, "x": x, "ids": ids}


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from chatterbox_amdvulkan_amd import cbxops as C
        if kind == "append":
            lens, n_free, start, slots, pos = C.paged_append(st["n_past"], st["n_new"], st["free"], st["n_free"], st["tables"],
                                                             case["page"], st["slots"])
            return {"lens": lens, "n_free": n_free, "start": start, "slots": slots, "pos": pos, "tables": st["tables"]}
        if kind == "qk" and case["store"]:
            q = C.qk_norm_rope_store(st["q"], st["k"], st["v"], st["gq"], st["gk"], EPS, st["pos"], st["rope"], st["slots"],
                                     st["kc"], st["vc"])
            return {"q": q, "kc": st["kc"], "vc": st["vc"]}
        if kind == "qk":
            q, k = C.qk_norm_rope(st["q"], st["k"], st["gq"], st["gk"], EPS, st["pos"], st["rope"])
            return {"q": q, "k": k}
        if kind == "attn":
            return C.paged_attention(st["q"], st["kc"], st["vc"], st["tables"], st["lens"], st["scale"], softcap=case["cap"],
                                     window=case["window"])
        logp, entropy, top_ids, top_logp = C.token_log_probs(st["x"], st["ids"], top_n=case["top"], scale=case["scale"])
        return {"logp": logp, "entropy": entropy, "top_ids": top_ids, "top_logp": top_logp}
    if kind == "append":
        return _append(st)
    if kind == "qk":
        return _qk(st)
    if kind == "attn":
        return _attention(st)
    return _log_probs(st)


def _append(st):
    page, tables, m = st["case"]["page"], st["tables"], st["slots"]
    past, new = st["n_past"].long(), st["n_new"].long()
    n, width = tables.shape
    have = (past + page - 1) // page
    end = torch.cumsum(new, 0)
    fits = (past + new <= width * page) & (end <= m)
    need = torch.where(fits, (past + new + page - 1) // page - have, torch.zeros_like(have))
    off = torch.cumsum(need, 0) - need
    ok = fits & ((need == 0) | (off + need <= st["n_free"]))
    i = torch.arange(width, device="cuda")[None]
    fresh = ok[:, None] & (i >= have[:, None]) & (i < (have + need)[:, None])
    at = (st["n_free"].long() - 1 - off[:, None] - (i - have[:, None])).clamp(0, st["free"].numel() - 1)
    tables.copy_(torch.where(fresh, st["free"][at], tables))
    lens = torch.where(ok, past + new, past)
    n_free = st["n_free"] - torch.where(ok, need, torch.zeros_like(need)).sum()
    start = torch.cat([torch.zeros_like(end[:1]), end])
    j = torch.arange(m, device="cuda")
    s = torch.searchsorted(end, j, right=True).clamp(max=n - 1)
    inside = j < end[-1]
    pos = torch.where(inside, past[s] + j - start[s], torch.zeros_like(j))
    p = tables[s, (pos // page).clamp(max=width - 1)].long() * page + pos % page
    slots = torch.where(inside & ok[s], p, torch.full_like(p, -1))
    i32 = lambda t: t.to(torch.int32)  # noqa: E731
    return {"lens": i32(lens), "n_free": i32(n_free), "start": i32(start), "slots": i32(slots), "pos": i32(pos), "tables": tables}


def _norm_rope(x, w, cos, sin, nd, mode):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w
    a, b = (y[..., :nd // 2], y[..., nd // 2:nd]) if mode == 2 else (y[..., 0:nd:2], y[..., 1:nd:2])
    c, s = cos[:, None], sin[:, None]
    u, v = a * c - b * s, a * s + b * c
    r = torch.cat([u, v], -1) if mode == 2 else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([r, y[..., nd:]], -1)


def _qk(st):
    case = st["case"]
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    q = _norm_rope(st["q"], st["gq"], cos, sin, case["nd"], case["mode"]).to(st["q"].dtype)
    k = _norm_rope(st["k"], st["gk"], cos, sin, case["nd"], case["mode"])
    if not case["store"]:
        return {"q": q, "k": k.to(st["k"].dtype)}
    kc, vc, page = st["kc"], st["vc"], case["page"]
    rows = torch.nonzero(st["slots"] >= 0)[:, 0]
    slots = st["slots"][rows].long()
    kc[slots // page, :, slots % page] = k[rows].to(kc.dtype)
    vc[slots // page, :, slots % page] = st["v"][rows].to(vc.dtype)
    return {"q": q, "kc": kc, "vc": vc}


def _attention(st):
    case = st["case"]
    n, hkv, g, d = case["n"], case["hkv"], case["g"], case["d"]
    t = st["tables"].long().clamp(min=0)
    k, v = (c[t].float().permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d) for c in (st["kc"], st["vc"]))
    i = torch.arange(k.shape[2], device="cuda")[None]
    lens = st["lens"].long()[:, None]
    seen = i < lens
    if case["window"]:
        seen = seen & (i >= lens - case["window"])
    seen = seen[:, None, None]
    s = torch.matmul(st["q"].float().reshape(n, hkv, g, d), k.transpose(2, 3).contiguous()) * st["scale"]
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    s = torch.where(seen, s, torch.full_like(s, float("-inf")))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    y = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return y.reshape(n, hkv * g, d).to(st["q"].dtype)


def _log_probs(st):
    case = st["case"]
    x = st["x"].float() * case["scale"]
    z = x - x.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1)
    lse = torch.log(total)
    logp = z.gather(1, st["ids"].long()[:, None])[:, 0] - lse
    ez = torch.where(e > 0, e * z, torch.zeros_like(e))
    entropy = lse - ez.sum(-1) / total
    top = torch.sort(st["x"], dim=-1, descending=True, stable=True)[1][:, :case["top"]]
    return {"logp": logp, "entropy": entropy, "top_ids": top.to(torch.int32), "top_logp": z.gather(1, top) - lse[:, None]}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "append":
        past, new = _lengths(case)
        have = -(-past // case["page"])
        fresh = int((-(-(past + new) // case["page"]) - have).sum())
        # lengths in and out, the token starts, the pages taken and noted, each request's open page, slots and positions
        return {"bytes": 4 * (4 * case["n"] + 2 * fresh + int((past % case["page"] > 0).sum()) + 2 * int(new.sum()) + 3), "flops": 0}
    if kind == "qk":
        tok, d, heads = case["tok"], case["d"], case["hq"] + case["hkv"]
        if not case["store"]:
            return {"bytes": 2 * tok * heads * d * SIZE[case["dt"]] + tok * 4 + POSITIONS * case["nd"] * 4 * min(1, tok / POSITIONS),
                    "flops": 8 * tok * heads * d}
        kept = tok - tok // 20
        read = (tok * case["hq"] + 2 * kept * case["hkv"]) * d * SIZE[case["dt"]]
        wrote = tok * case["hq"] * d * SIZE[case["dt"]] + 2 * kept * case["hkv"] * d * SIZE[case["cdt"]]
        return {"bytes": read + wrote + tok * 8 + POSITIONS * case["nd"] * 4 * min(1, tok / POSITIONS),
                "flops": 8 * (tok * case["hq"] + kept * case["hkv"]) * d}
    if kind == "attn":
        lens = _spread(case["lo"], case["hi"], case["n"])
        if case["window"]:
            lens = np.minimum(lens, case["window"])
        keys, hq = int(lens.sum()), case["hkv"] * case["g"]
        return {"bytes": 2 * keys * case["hkv"] * case["d"] * SIZE[case["cdt"]] + 2 * case["n"] * hq * case["d"] * SIZE[case["dt"]],
                "flops": 4 * keys * hq * case["d"]}
    cells = case["rows"] * case["vocab"]
    return {"bytes": cells * SIZE[case["dt"]] + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * cells}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    kind = case["kind"]
    if kind == "append":
        return None                                             # whole numbers only
    st = prepare(case, seed)
    if kind == "qk":
        nd, half = case["nd"], case["nd"] // 2
        theta = torch.from_numpy(_angles(POSITIONS, nd, case["base"])).cuda()[st["pos"].long()][:, None]
        turn = torch.complex(theta.cos(), theta.sin())

        def heads(x, w):
            y = x.double() / (x.double().pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
            if case["mode"] == 2:
                z = torch.complex(y[..., :half].contiguous(), y[..., half:nd].contiguous()) * turn
                y[..., :half], y[..., half:nd] = z.real, z.imag
            else:
                z = torch.complex(y[..., 0:nd:2].contiguous(), y[..., 1:nd:2].contiguous()) * turn
                y[..., 0:nd:2], y[..., 1:nd:2] = z.real, z.imag
            return y

        q, k = heads(st["q"], st["gq"]), heads(st["k"], st["gk"])
        if not case["store"]:
            return {"q": q, "k": k}
        kc, vc = st["kc"].double(), st["vc"].double()
        flat = lambda c: c.transpose(1, 2).reshape(-1, case["hkv"], case["d"])  # noqa: E731
        fk, fv = flat(kc).clone(), flat(vc).clone()
        live = st["slots"] >= 0
        fk[st["slots"][live].long()] = k[live]
        fv[st["slots"][live].long()] = st["v"][live].double()
        back = lambda f: f.reshape(kc.shape[0], case["page"], case["hkv"], case["d"]).transpose(1, 2)  # noqa: E731
        return {"q": q, "kc": back(fk), "vc": back(fv)}
    if kind == "attn":
        hkv, g, d = case["hkv"], case["g"], case["d"]
        q = st["q"].double().reshape(case["n"], hkv, g, d)
        y = torch.zeros(case["n"], hkv * g, d, dtype=torch.float64, device="cuda")
        for s, length in enumerate(st["lens"].tolist()):
            if not length:
                continue
            rows = st["tables"][s, :-(-length // case["page"])].long()
            a = max(0, length - case["window"]) if case["window"] else 0
            for h in range(hkv):
                k, v = (c[rows, h].double().reshape(-1, d)[a:length] for c in (st["kc"], st["vc"]))
                w = (q[s, h] * st["scale"]) @ k.T
                if case["cap"]:
                    w = case["cap"] * torch.tanh(w / case["cap"])
                y[s, h * g:(h + 1) * g] = torch.softmax(w, -1) @ v
        return y
    x, ids = st["x"], st["ids"].long()
    logp, entropy, tops = [], [], []
    order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :case["top"]]
    for r in range(0, case["rows"], 512):                       # a few rows at a time: 64-bit copies of a large case are large
        lp = torch.log_softmax(x[r:r + 512].double() * case["scale"], -1)
        logp.append(lp.gather(1, ids[r:r + 512, None])[:, 0])
        entropy.append(torch.special.entr(lp.exp()).sum(-1))
        tops.append(lp.gather(1, order[r:r + 512]))
    return {"logp": torch.cat(logp), "entropy": torch.cat(entropy), "top_ids": None, "top_logp": torch.cat(tops)}
