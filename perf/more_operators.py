"""Prompts, shared prefixes and an 8-bit cache over key-value pages, as calls that can be timed and checked.

A case is a dict of plain values; its "kind" says which operator it calls:

  cache8    keys and values of a step's tokens into 8-bit pages with a scale for each row, and read back
  attn8     attention of one new token a request over 8-bit pages
  prompt    causal attention of all new tokens of packed requests over their pages, cached keys before them
  shared    attention of one new token a request, where groups of requests begin with the same pages

prepare() makes what a serving loop holds before the call, run() is one pass (own: the library's entry points; else the
same from elementary torch operations in 32 bits), exact() the definition in 64 bits.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

LOWEST = 127 * 2.0 ** -126                                      # a row's largest element counts as this at least: normal scales
TYPES = {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "i8": 1}


def listed():
    return [
        # a 64-stream decode step of the backbone's 16 heads, F32 activations: the smallest
        {"name": "cache8_decode", "kind": "cache8", "tok": 64, "hkv": 16, "d": 64, "dt": "f32", "page": 64},
        # a batch of prompts with few key heads, F16 activations, pages of an odd size
        {"name": "cache8_prompts", "kind": "cache8", "tok": 9001, "hkv": 8, "d": 128, "dt": "f16", "page": 50},
        # 64 streams of the backbone anywhere in its 2048 positions, F32 activations over 8-bit pages
        {"name": "attn8_streams", "kind": "attn8", "n": 64, "lo": 1, "hi": 2048, "hkv": 16, "g": 1, "d": 64, "page": 64,
         "dt": "f32", "cdt": "i8", "cap": 0.0, "window": 0},
        # long requests with shared heads, the cache in 8 bits
        {"name": "attn8_long", "kind": "attn8", "n": 8, "lo": 1500, "hi": 65000, "hkv": 8, "g": 4, "d": 128, "page": 32,
         "dt": "f16", "cdt": "i8", "cap": 0.0, "window": 0},
        # a few short texts admitted to the backbone, F32 activations: latency
        {"name": "prompt_texts", "kind": "prompt", "n": 4, "past_lo": 0, "past_hi": 0, "new_lo": 20, "new_hi": 150, "hkv": 16,
         "g": 1, "d": 64, "page": 64, "dt": "f32", "cdt": "f16", "cap": 0.0, "window": 0, "pad": 12},
        # many texts of all lengths at once, some on cached beginnings
        {"name": "prompt_batch", "kind": "prompt", "n": 48, "past_lo": 0, "past_hi": 700, "new_lo": 1, "new_hi": 2047, "hkv": 16,
         "g": 1, "d": 64, "page": 64, "dt": "f16", "cdt": "f16", "cap": 0.0, "window": 0, "pad": 100},
        # one long text with shared heads: the largest
        {"name": "prompt_long", "kind": "prompt", "n": 1, "past_lo": 0, "past_hi": 0, "new_lo": 16000, "new_hi": 16000, "hkv": 8,
         "g": 4, "d": 128, "page": 32, "dt": "f16", "cdt": "f16", "cap": 0.0, "window": 0, "pad": 0},
        # a few drafted tokens a request checked against a long 8-bit cache
        {"name": "prompt_draft8", "kind": "prompt", "n": 8, "past_lo": 900, "past_hi": 32000, "new_lo": 1, "new_hi": 9, "hkv": 8,
         "g": 4, "d": 128, "page": 32, "dt": "f16", "cdt": "i8", "cap": 0.0, "window": 0, "pad": 0},
        # an F32 cache with pages of an odd size, capped scores, a sliding window, five heads to a key head
        {"name": "prompt_f32_window", "kind": "prompt", "n": 5, "past_lo": 0, "past_hi": 1500, "new_lo": 300, "new_hi": 1301,
         "hkv": 4, "g": 5, "d": 80, "page": 24, "dt": "f32", "cdt": "f32", "cap": 30.0, "window": 1001, "pad": 3},
        # 64 takes of one text by the backbone: the conditioning and the text are shared, the speech so far is each take's own
        {"name": "shared_takes", "kind": "shared", "groups": 1, "n": 64, "pre_lo": 1150, "pre_hi": 1150, "own_lo": 1, "own_hi": 800,
         "hkv": 16, "g": 1, "d": 64, "page": 64, "dt": "f16", "cdt": "f16", "cap": 0.0, "window": 0},
        # long documents, many questions to each
        {"name": "shared_documents", "kind": "shared", "groups": 4, "n": 96, "pre_lo": 5000, "pre_hi": 30000, "own_lo": 10,
         "own_hi": 1500, "hkv": 8, "g": 4, "d": 128, "page": 32, "dt": "f16", "cdt": "f16", "cap": 0.0, "window": 0},
        # F32 activations over an 8-bit cache, a window that ends inside the shared part for some requests, groups of one among them
        {"name": "shared_window8", "kind": "shared", "groups": 7, "n": 33, "pre_lo": 0, "pre_hi": 3500, "own_lo": 0, "own_hi": 900,
         "hkv": 4, "g": 3, "d": 96, "page": 16, "dt": "f32", "cdt": "i8", "cap": 20.0, "window": 2500},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["cache8", "cache8", "attn8", "attn8", "prompt", "prompt", "prompt", "prompt", "shared", "shared", "shared"])
    d, hkv = rng.choice([32, 64, 64, 80, 96, 128, 128, 256]), rng.choice([1, 2, 4, 8, 16])
    if kind == "cache8":
        return {"kind": kind, "tok": _log(rng, 1, max(2, min(60000, 9001 * 40 * 128 // (d * hkv * 3)))), "hkv": hkv, "d": d,
                "dt": rng.choice(["f16", "f32"]), "page": rng.choice([1, 10, 16, 32, 50, 64, 128])}
    g, page = rng.choice([1, 1, 2, 3, 4, 7, 8, 16]), rng.choice([5, 8, 16, 24, 32, 64, 64, 128, 256])
    dt = rng.choice(["f16", "f16", "f32"])
    cdt = rng.choice(["f16", "f16", "i8"] if dt == "f16" else ["f16", "f32", "i8"])
    rest = {"hkv": hkv, "g": g, "d": d, "page": page, "dt": dt, "cdt": cdt, "cap": rng.choice([0.0, 0.0, 0.0, 20.0])}
    if kind == "attn8":
        n = _log(rng, 1, 256)
        hi = _log(rng, 1, max(2, min(130000, 260000 * 8 * 128 // (n * hkv * d))))
        return {"kind": kind, "n": n, "lo": rng.choice([hi, 0, hi // 8]), "hi": hi, **rest, "cdt": "i8",
                "window": rng.choice([0, 0, 0, max(1, hi // 3)])}
    if kind == "shared":
        n = _log(rng, 1, 200)
        groups = rng.choice([1, 1, min(n, 3), max(1, n // 8)])
        pre = _log(rng, 1, max(2, min(30000, 60000 * 8 * 128 // (hkv * d * groups))))
        mine = _log(rng, 1, max(2, min(3000, 70000 * 8 * 128 // (hkv * d * n))))
        return {"kind": kind, "groups": groups, "n": n, "pre_lo": rng.choice([pre, 0, pre // 6]), "pre_hi": pre,
                "own_lo": rng.choice([0, 1, mine]), "own_hi": mine, **rest, "window": rng.choice([0, 0, 0, max(1, pre // 2)])}
    n = _log(rng, 1, 64)
    new = rng.choice([_log(rng, 1, 16), _log(rng, 1, max(2, 16000 // n)), _log(rng, 100, max(200, 16000 // n))])
    past = rng.choice([0, 0, _log(rng, 1, max(2, min(30000, 120000 * 8 * 128 // (n * hkv * d))))])
    # queries times keys times heads, an eighth of the largest listed case's in F32 pages
    most = 16000 * 16000 // 2 * 32 * 128 // (8 if cdt == "f32" else 2)
    while new > 1 and n * new * (past + new) * hkv * g * d > most:
        new = max(1, new // 2)
    return {"kind": kind, "n": n, "past_lo": rng.choice([past, 0]), "past_hi": past, "new_lo": rng.choice([0, 1, new]), "new_hi": new,
            **rest, "window": rng.choice([0, 0, 0, max(1, (past + new) // 3)]), "pad": rng.choice([0, 0, 1, 33])}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _spread(lo, hi, n):
    """n whole numbers evenly spread over [lo, hi] (hi alone for one)."""
    return np.linspace(hi if n == 1 else lo, hi, n).round().astype(np.int64)


def _groups(case):
    """The first request of every group and their number behind the last; the groups' sizes go up."""
    n, groups = case["n"], case["groups"]
    size = np.ones(groups, dtype=np.int64) if n >= groups else np.zeros(groups, dtype=np.int64)
    rest = n - int(size.sum())
    share = np.arange(1, groups + 1, dtype=np.float64)
    size += (share / share.sum() * rest).astype(np.int64)
    size[-1] += n - int(size.sum())
    return np.concatenate([[0], np.cumsum(size)])


def _prefixes(case):
    """Keys that each group shares: whole pages."""
    return _spread(case["pre_lo"], case["pre_hi"], case["groups"]) // case["page"] * case["page"]


def _tables(n, counts, width, perm):
    """[n, width] page tables: the first counts[s] entries of row s taken from perm in order, -1 behind them."""
    idx = torch.arange(width, device="cuda").expand(n, width)
    first = torch.cumsum(counts, 0) - counts
    src = (first[:, None] + idx).clamp(max=max(0, perm.numel() - 1))
    return torch.where(idx < counts[:, None], perm[src], torch.full_like(src, -1)).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    host = np.random.RandomState(int(seed) % (1 << 31))
    kind, hkv, d, page = case["kind"], case["hkv"], case["d"], case["page"]
    randn = lambda *s, dt="f32": torch.randn(*s, device="cuda", generator=g, dtype=TYPES[dt])  # noqa: E731
    perm = lambda n: torch.randperm(n, device="cuda", generator=g)  # noqa: E731
    ints = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda().to(torch.int32)  # noqa: E731

    def cache(pages):
        """Keys or values of so many pages, and the scale of every row of an 8-bit one."""
        if case["cdt"] != "i8":
            return randn(pages, hkv, page, d, dt=case["cdt"]), None
        x = randn(pages, hkv, page, d, dt="f16").float()
        top = x.abs().amax(-1).clamp(min=LOWEST)
        return torch.round(x * 127 / top[..., None]).to(torch.int8), top / 127

    if kind == "cache8":
        tok = case["tok"]
        rows = randn(tok, 2 * hkv * d + 64, dt=case["dt"]) * 1.5   # views of one projection's output
        pages = -(-(tok + 100) // page)
        slots = perm(pages * page)[:tok].to(torch.int32)
        slots[tok - tok // 20:] = -1                            # a padded batch: its last rows belong to no request
        zeros = lambda *s, dt: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
        return {"case": case, "k": rows[:, :hkv * d].unflatten(1, (hkv, d)), "v": rows[:, hkv * d:2 * hkv * d].unflatten(1, (hkv, d)),
                "slots": slots, "kc": zeros(pages, hkv, page, d, dt=torch.int8), "vc": zeros(pages, hkv, page, d, dt=torch.int8),
                "ks": zeros(pages, hkv, page, dt=torch.float32), "vs": zeros(pages, hkv, page, dt=torch.float32)}

    n, hq = case["n"], hkv * case["g"]
    st = {"case": case, "scale": d ** -0.5}
    if kind == "attn8":
        lens = _spread(case["lo"], case["hi"], n)[host.permutation(n)]
        st["q"] = randn(n, hq, d, dt=case["dt"]) * 2
    elif kind == "prompt":
        past = _spread(case["past_lo"], case["past_hi"], n)[host.permutation(n)]
        new = _spread(case["new_lo"], case["new_hi"], n)[host.permutation(n)]
        lens = past + new
        start = np.concatenate([[0], np.cumsum(new)])
        st["q"] = randn(int(start[-1]) + case["pad"], hq, d, dt=case["dt"]) * 2
        st["y"] = torch.zeros_like(st["q"])                     # rows behind the last request stay as they are
        st["start"], st["past"], st["new"] = ints(start), past.tolist(), new.tolist()
    else:
        first, pre = _groups(case), _prefixes(case)
        mine = _spread(case["own_lo"], case["own_hi"], n)[host.permutation(n)]
        lens = np.repeat(pre, np.diff(first)) + mine
        st["q"] = randn(n, hq, d, dt=case["dt"]) * 2
        st["first"], st["pre"] = ints(first), ints(pre)
        st["groups"], st["shared"] = first.tolist(), pre.tolist()
    counts = -(-lens // page)
    width = max(1, int(counts.max()))
    pages = int(counts.sum()) + 3
    st["tables"] = _tables(n, ints(counts).long(), width, perm(pages))
    if kind == "shared":                                        # a group's shared pages are its first request's
        for a, b, p in zip(st["groups"], st["groups"][1:], st["shared"]):
            if b > a:
                st["tables"][a:b, :p // page] = st["tables"][a, :p // page].clone()
    st["lens"], st["host_lens"] = ints(lens), lens.tolist()
    (st["kc"], st["ks"]), (st["vc"], st["vs"]) = cache(pages), cache(pages)
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from chatterbox_amdvulkan_amd import cbxops as C
        if kind == "cache8":
            C.paged_store(st["k"], st["v"], st["slots"], st["kc"], st["vc"], k_scale=st["ks"], v_scale=st["vs"])
            k, v = C.paged_load(st["slots"], st["kc"], st["vc"], k_scale=st["ks"], v_scale=st["vs"], dtype=TYPES[case["dt"]])
            return {"k": k, "v": v}
        more = {"softcap": case["cap"], "window": case["window"], "k_scale": st["ks"], "v_scale": st["vs"]}
        if kind == "attn8":
            return C.paged_attention(st["q"], st["kc"], st["vc"], st["tables"], st["lens"], st["scale"], **more)
        if kind == "prompt":
            return C.paged_prompt_attention(st["q"], st["kc"], st["vc"], st["tables"], st["lens"], st["start"], st["scale"],
                                            out=st["y"], **more)
        return C.paged_shared_attention(st["q"], st["kc"], st["vc"], st["tables"], st["lens"], st["first"], st["pre"], st["scale"],
                                        **more)
    return {"cache8": _cache8, "attn8": _attn8, "prompt": _prompt, "shared": _shared}[kind](st)


def _cache8(st):
    page = st["case"]["page"]
    live = st["slots"] >= 0
    rows = torch.nonzero(live)[:, 0]
    slots, at = st["slots"][rows].long(), st["slots"].long().clamp(min=0)
    back = []
    for x, c, sc in ((st["k"], st["kc"], st["ks"]), (st["v"], st["vc"], st["vs"])):
        x64 = x.double()                                        # 64 bits: half the largest element lies on a border
        top = x64.abs().amax(-1).clamp(min=LOWEST)
        c[slots // page, :, slots % page] = torch.round(x64 * 127 / top[..., None])[rows].to(torch.int8)
        sc[slots // page, :, slots % page] = (top / 127)[rows].float()
        y = c[at // page, :, at % page].float() * sc[at // page, :, at % page][..., None]
        back.append(torch.where(live[:, None, None], y, torch.zeros_like(y)).to(x.dtype))
    return {"k": back[0], "v": back[1]}


def _values(c, s, pages):
    """The keys or values of a table's pages in 32 bits."""
    x = c[pages].float()
    return x if s is None else x * s[pages][..., None]


def _capped(s, cap):
    return cap * torch.tanh(s / cap) if cap else s


def _weights(s):
    """exp of the scores less the row's largest, and its sums: a row of nothing but -inf has zeros."""
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    return p, p.sum(-1, keepdim=True).clamp(min=1e-30)


def _attn8(st):
    case = st["case"]
    n, hkv, g, d = case["n"], case["hkv"], case["g"], case["d"]
    t = st["tables"].long().clamp(min=0)
    k, v = (_values(c, s, t).permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d) for c, s in ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
    i = torch.arange(k.shape[2], device="cuda")[None]
    lens = st["lens"].long()[:, None]
    seen = i < lens
    if case["window"]:
        seen = seen & (i >= lens - case["window"])
    s = torch.matmul(st["q"].float().reshape(n, hkv, g, d), k.transpose(2, 3).contiguous()) * st["scale"]
    s = torch.where(seen[:, None, None], _capped(s, case["cap"]), torch.full_like(s, float("-inf")))
    p, total = _weights(s)
    return (torch.matmul(p, v) / total).reshape(n, hkv * g, d).to(st["q"].dtype)


def _prompt(st):
    case, y = st["case"], st["y"]
    hkv, g, d, page, window = (case[x] for x in ("hkv", "g", "d", "page", "window"))
    at = 0
    for r, (past, new) in enumerate(zip(st["past"], st["new"])):
        if not new:
            continue
        t = st["tables"][r, :-(-(past + new) // page)].long()
        k, v = (_values(c, s, t).transpose(0, 1).reshape(hkv, -1, d)[:, :past + new] for c, s in ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
        kt = k.transpose(1, 2).contiguous()
        step = max(1, (1 << 28) // (hkv * g * (past + new)))    # some rows at a time: the scores of a long text are large
        for a in range(0, new, step):
            b = min(new, a + step)
            q = st["q"][at + a:at + b].float().reshape(b - a, hkv, g, d).permute(1, 0, 2, 3).reshape(hkv, -1, d)
            i = torch.arange(past + new, device="cuda")[None]
            pos = past + torch.arange(a, b, device="cuda").repeat_interleave(g)[:, None]
            seen = i <= pos
            if window:
                seen = seen & (i > pos - window)
            s = torch.matmul(q, kt) * st["scale"]
            s = torch.where(seen, _capped(s, case["cap"]), torch.full_like(s, float("-inf")))
            p, total = _weights(s)
            o = (torch.matmul(p, v) / total).reshape(hkv, b - a, g, d).permute(1, 0, 2, 3)
            y[at + a:at + b] = o.reshape(b - a, hkv * g, d).to(y.dtype)
        at += new
    return y


def _shared(st):
    case = st["case"]
    hkv, g, d, page, window = (case[x] for x in ("hkv", "g", "d", "page", "window"))
    out = []
    for a, b, pre in zip(st["groups"], st["groups"][1:], st["shared"]):
        n = b - a
        if not n:
            continue
        q = st["q"][a:b].float().reshape(n, hkv, g, d)
        t0 = st["tables"][a, :pre // page].long()
        longest = max(st["host_lens"][a:b])
        t1 = st["tables"][a:b, pre // page:max(1, -(-longest // page))].long().clamp(min=0)
        k0, v0 = (_values(c, s, t0).transpose(0, 1).reshape(hkv, pre, d) for c, s in ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
        k1, v1 = (_values(c, s, t1).permute(0, 2, 1, 3, 4).reshape(n, hkv, t1.shape[1] * page, d)
                  for c, s in ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
        s0 = torch.matmul(q.permute(1, 0, 2, 3).reshape(hkv, n * g, d), k0.transpose(1, 2).contiguous())
        s1 = torch.matmul(q, k1.transpose(2, 3).contiguous())
        s = torch.cat([s0.reshape(hkv, n, g, pre).permute(1, 0, 2, 3), s1], -1) * st["scale"]
        i = torch.arange(s.shape[-1], device="cuda")[None]
        lens = st["lens"][a:b].long()[:, None]
        seen = i < lens
        if window:
            seen = seen & (i >= lens - window)
        s = torch.where(seen[:, None, None], _capped(s, case["cap"]), torch.full_like(s, float("-inf")))
        p, total = _weights(s)
        o = torch.matmul(p[..., :pre].permute(1, 0, 2, 3).reshape(hkv, n * g, pre), v0).reshape(hkv, n, g, d).permute(1, 0, 2, 3)
        o = (o + torch.matmul(p[..., pre:].contiguous(), v1)) / total
        out.append(o.reshape(n, hkv * g, d).to(st["q"].dtype))
    return torch.cat(out)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def _key_bytes(case):
    """Of one key and value of one key head."""
    return 2 * (case["d"] * SIZE[case["cdt"]] + (4 if case["cdt"] == "i8" else 0))


def work(case):
    kind, hkv, d, window = case["kind"], case["hkv"], case["d"], case.get("window", 0)
    if kind == "cache8":
        tok, kept = case["tok"], case["tok"] - case["tok"] // 20
        # rows in and back (no rows of padding in), held values and their scales written and read, slots twice
        return {"bytes": 2 * (tok + kept) * hkv * d * SIZE[case["dt"]] + 4 * kept * hkv * (d + 4) + tok * 8,
                "flops": 8 * kept * hkv * d}
    hq = hkv * case["g"]
    if kind == "prompt":
        # lengths are dealt by the seed: the sizes that the sorted ones give
        past, new = _spread(case["past_lo"], case["past_hi"], case["n"]), _spread(case["new_lo"], case["new_hi"], case["n"])
        keys = pairs = 0
        for p, m in zip(past.tolist(), new.tolist()):
            pos = np.arange(p, p + m, dtype=np.int64)
            pairs += int((np.minimum(pos + 1, window) if window else pos + 1).sum())
            keys += 0 if not m else min(p + m, m + window - 1) if window else p + m
        rows = int(new.sum())
        return {"bytes": keys * hkv * _key_bytes(case) + 2 * rows * hq * d * SIZE[case["dt"]], "flops": 4 * pairs * hq * d}
    if kind == "attn8":
        lens = _spread(case["lo"], case["hi"], case["n"])
        read = pairs = int((np.minimum(lens, window) if window else lens).sum())
    else:
        first, pre = _groups(case), _prefixes(case)
        of = np.repeat(pre, np.diff(first))
        lens = of + _spread(case["own_lo"], case["own_hi"], case["n"])
        from_ = np.maximum(0, lens - window) if window else np.zeros_like(lens)
        pairs = int((lens - from_).sum())
        read = int((lens - np.maximum(of, from_)).sum())
        for a, b, p in zip(first.tolist(), first.tolist()[1:], pre.tolist()):
            if b > a:
                read += max(0, p - int(from_[a:b].min()))
    return {"bytes": read * hkv * _key_bytes(case) + 2 * case["n"] * hq * d * SIZE[case["dt"]], "flops": 4 * pairs * hq * d}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    kind = case["kind"]
    st = prepare(case, seed)
    if kind == "cache8":
        def held(x):
            x = x.double()
            top = x.abs().amax(-1, keepdim=True).clamp(min=LOWEST)
            n = x * 127 / top
            whole = torch.floor(n.abs())                        # the nearest whole number, of two the even one
            rest = n.abs() - whole
            n = torch.sign(n) * (whole + ((rest > 0.5) | ((rest == 0.5) & (whole % 2 == 1))).double())
            return torch.where((st["slots"] >= 0)[:, None, None], n * top / 127, torch.zeros_like(x))

        return {"k": held(st["k"]), "v": held(st["v"])}

    hkv, g, d, page, window, cap = (case[x] for x in ("hkv", "g", "d", "page", "window", "cap"))
    y = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for r, length in enumerate(st["host_lens"]):
        new = st["new"][r] if kind == "prompt" else 1
        if length and new:
            rows = st["tables"][r, :-(-length // page)].long()
            for h in range(hkv):
                k, v = (c[rows, h].double() * (1 if s is None else s[rows, h].double()[..., None]) for c, s in
                        ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
                k, v = k.reshape(-1, d)[:length], v.reshape(-1, d)[:length]
                for a in range(0, new, 2048):
                    b = min(new, a + 2048)
                    w = torch.einsum("thd,kd->htk", st["q"][at + a:at + b, h * g:(h + 1) * g].double() * st["scale"], k)
                    if cap:
                        w = cap * torch.tanh(w / cap)
                    last = length - new + torch.arange(a, b, device="cuda")[:, None]
                    i = torch.arange(length, device="cuda")
                    w.masked_fill_((i > last) | ((i <= last - window) if window else (i < 0)), float("-inf"))
                    y[at + a:at + b, h * g:(h + 1) * g] = (torch.softmax(w, -1) @ v).transpose(0, 1)
        at += new
    return y
