"""Plain 64-bit forms of the paged-cache operators and their error bounds."""
from __future__ import annotations

import numpy as np
import torch

U32 = 2.0 ** -24                       # half a step of f32, relative


def half_step(dtype) -> float:
    return float(torch.finfo(dtype).eps) / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def page_tables(lens, page, width, n_pages, seed, fill=-1):
    """int32 [n, width] page tables over a shuffled pool: request s's first
    ceil(lens[s] / page) entries, `fill` behind them."""
    order = np.random.RandomState(seed).permutation(n_pages)
    t = np.full((len(lens), width), fill, dtype=np.int32)
    at = 0
    for s, length in enumerate(lens):
        k = -(-max(0, length) // page)
        t[s, :k] = order[at:at + k]
        at += k
    assert at <= n_pages
    return torch.from_numpy(t)


def attention_ref(q, kc, vc, tables, lens, scale, softcap=0.0, window=0):
    """(y, bound) in float64 on q's device: the definition, and how far an f32
    evaluation may be from it.

    A score is a product of D terms (each product and sum one rounding, in
    any order: D + 1 of them against sum |q k|), times scale, in the exponent
    times log2(e) and less the maximum (4 roundings of |s| or |m|), the cap's
    division, tanh and product 4 more of at most |cap|; an exponential is 4
    roundings off.  A relative error d of every p changes y by at most 2 d
    sum p |v|, n sums by n roundings of it, the division one."""
    n, hq, d = q.shape
    page, hkv = kc.shape[2], kc.shape[1]
    g = hq // hkv
    y = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(y)
    for s, length in enumerate(lens):
        a = max(0, length - window) if window else 0
        if length <= 0:
            continue
        rows = tables[s, :-(-length // page)].long().to(q.device)
        ok = (rows >= 0) & (rows < kc.shape[0])
        rows = rows.clamp(0, kc.shape[0] - 1)
        keep = ok.repeat_interleave(page)[a:length]
        if not bool(keep.any()):
            continue
        k = kc[rows].transpose(0, 1).reshape(hkv, -1, d)[:, a:length][:, keep].double()
        v = vc[rows].transpose(0, 1).reshape(hkv, -1, d)[:, a:length][:, keep].double()
        qs = q[s].double().reshape(hkv, g, d)
        raw = torch.matmul(qs, k.transpose(1, 2).contiguous()) * scale
        size = torch.matmul(qs.abs(), k.abs().transpose(1, 2).contiguous()) * abs(scale)
        w = softcap * torch.tanh(raw / softcap) if softcap else raw
        p = torch.softmax(w, -1)
        y[s] = torch.matmul(p, v).reshape(hq, d)
        top = w.abs().amax(-1, keepdim=True)
        err = U32 * ((d + 1) * size.amax(-1, keepdim=True) + 4 * top + (4 * softcap if softcap else 0) + 4)
        pv = torch.matmul(p, v.abs())
        # two parts of an f16 pair hold 22 bits of p: 2^-22 is 4 U32
        bound[s] = ((2 * err + (k.shape[1] + 8) * U32) * pv).reshape(hq, d)
    return y, bound + half_step(q.dtype) * y.abs()


def assert_within(got, ref, bound, what=""):
    d = (got.double() - ref).abs()
    assert bool(torch.isfinite(d).all()), f"{what}: not finite"
    over = d > bound + 1e-30
    if bool(over.any()):
        i = int((d - bound).argmax())
        raise AssertionError(f"{what}: {int(over.sum())} of {d.numel()} past the bound; worst {d.flatten()[i]:.3e} "
                             f"allowed {bound.flatten()[i]:.3e}")


def append_ref(past, new, free, n_free, tables, page, n_slots):
    """paged_append by a loop over the requests; lists and a copied table."""
    tables = [list(r) for r in tables]
    width = len(tables[0]) if tables else 0
    lens, start, slots, pos = [], [0], [-1] * n_slots, [0] * n_slots
    top, dry = n_free, False
    for s, (p, w) in enumerate(zip(past, new)):
        t = start[-1]
        start.append(t + w)
        fits = p + w <= width * page and t + w <= n_slots
        need = -(-(p + w) // page) + (-p // page) if fits else 0
        if need > 0 and (dry or need > top):
            dry, fits = True, False
        if fits:
            for i in range(need):
                top -= 1
                tables[s][-(-p // page) + i] = free[top]
        lens.append(p + w if fits else p)
        for j in range(w):
            if t + j < n_slots:
                pos[t + j] = p + j
                if fits:
                    slots[t + j] = tables[s][(p + j) // page] * page + (p + j) % page
    return lens, top, start, slots, pos, tables
