"""Plain 64-bit forms of prompt attention, shared beginnings and 8-bit rows, and their error bounds."""
from __future__ import annotations

import numpy as np
import torch

from tests._paged import U32, gen, half_step, page_tables

LOWEST = 127 * 2.0 ** -126


def ints(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


def q8_ref(x):
    """(elements, scales) of rows in 8 bits: int8 and float32, decided in whole numbers."""
    x64 = x.double()
    top = x64.abs().amax(-1).clamp(min=LOWEST)
    n = x64 * 127 / top[..., None]              # 127 x exact, the quotient a tie only where the true one is
    return torch.round(n).to(torch.int8), (top / 127).float()


def make_cache(pages, hkv, page, d, cdt, g, permuted=False):
    """(k, v, k_scale, v_scale) with random pages; permuted: [n_pages, page, hkv, d] memory."""
    shape = (pages, page, hkv, d) if permuted else (pages, hkv, page, d)
    out, scales = [], []
    for _ in range(2):
        x = torch.randn(*shape, device="cuda", generator=g)
        s = None
        if cdt == torch.int8:
            x, s = q8_ref(x)
            s = s.transpose(1, 2) if permuted else s
        else:
            x = x.to(cdt)
        out.append(x.transpose(1, 2) if permuted else x)
        scales.append(s)
    return out[0], out[1], scales[0], scales[1]


def values(c, s, rows):
    """Pages in 64 bits, with their scales."""
    x = c[rows].double()
    return x if s is None else x * s[rows].double()[..., None]


def rows_ref(q, kc, vc, ks, vs, tables, lens, start, scale, softcap=0.0, window=0, fill=0.0, p_err=0.0):
    """(y, bound) in float64: every row of q attends over its own keys alone,
    picked before anything is multiplied.  start: packed tokens; None: a row a
    request.  Rows of no request hold `fill`.

    The bound is attention_ref's (a score D + 1 roundings of sum |q k|, 4 of
    the exponent's parts, the cap's 4, n + 8 roundings of sum p |v|), with two
    more a score and one more a value for an 8-bit row's scale; p_err: the
    relative rounding of each probability for its product, which moves a weight
    p / sum p by twice that."""
    t, hq, d = q.shape
    page, hkv = kc.shape[2], kc.shape[1]
    g = hq // hkv
    y = torch.full((t, hq, d), fill, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(y)
    for s, length in enumerate(lens):
        a, b = (start[s], start[s + 1]) if start is not None else (s, s + 1)
        y[a:b] = 0
        if length <= 0 or b <= a:
            continue
        rows = tables[s, :-(-length // page)].long().to(q.device)
        ok = ((rows >= 0) & (rows < kc.shape[0])).repeat_interleave(page)[:length]
        rows = rows.clamp(0, kc.shape[0] - 1)
        k = values(kc, ks, rows).transpose(0, 1).reshape(hkv, -1, d)[:, :length]
        v = values(vc, vs, rows).transpose(0, 1).reshape(hkv, -1, d)[:, :length]
        for i in range(a, b):
            end = length - (b - 1 - i)
            first = max(0, end - window) if window else 0
            if end <= 0:
                continue
            keep = ok[first:end]
            if not bool(keep.any()):
                continue
            ki, vi = k[:, first:end][:, keep], v[:, first:end][:, keep]
            qi = q[i].double().reshape(hkv, g, d)
            kt = ki.transpose(1, 2).contiguous()
            raw = torch.matmul(qi, kt) * scale
            size = torch.matmul(qi.abs(), kt.abs()) * abs(scale)
            w = softcap * torch.tanh(raw / softcap) if softcap else raw
            p = torch.softmax(w, -1)
            y[i] = torch.matmul(p, vi).reshape(hq, d)
            top = w.abs().amax(-1, keepdim=True)
            err = U32 * ((d + 3) * size.amax(-1, keepdim=True) + 4 * top + (4 * softcap if softcap else 0) + 6) + p_err
            bound[i] = ((2 * err + (ki.shape[1] + 9) * U32) * torch.matmul(p, vi.abs())).reshape(hq, d)
    # below the smallest normal number a step is that number's: eps * tiny
    return y, bound + half_step(q.dtype) * y.abs().clamp(min=torch.finfo(q.dtype).tiny)


def packed(past, new, page, seed, extra=2, width=None):
    """(lens, start, tables, n_pages) of packed requests with shuffled pages."""
    lens = [p + n for p, n in zip(past, new)]
    n_pages = sum(-(-x // page) for x in lens) + extra
    width = width or max(1, max(-(-x // page) for x in lens))
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    return lens, start, page_tables(lens, page, width, n_pages, seed).cuda(), n_pages


__all__ = ["LOWEST", "U32", "gen", "half_step", "ints", "make_cache", "packed", "page_tables", "q8_ref", "rows_ref", "values"]
