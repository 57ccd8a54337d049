"""Prompt attention and attention of shared beginnings at the ends of the
ranges: values near f32's largest, scores of millions, infinite keys that have
no weight, caps and scales of any size, tables of the largest capacity."""
import numpy as np
import pytest
import torch

from tests._paged import assert_within
from tests._paged_more import U32, gen, half_step, ints, make_cache, packed, rows_ref

pytestmark = pytest.mark.gpu
F16, F32, I8 = torch.float16, torch.float32, torch.int8
TYPES = [(F16, F16), (F32, F16), (F32, F32), (F16, F32), (F16, I8), (F32, I8)]
TWO_BF16 = 2.0 ** -15                  # of an F16 query over I8 pages: 16 bits of a probability times its value's scale, cut off


def test_shared_past_the_tiles_of_one_token(cbx):
    """32 requests of 4 key heads, tables of 2^31 - 2 keys (one page that all
    entries repeat): more tiles than the kernel of the requests' own keys
    counts.  The scratch holds NaN before the call."""
    n, page, width, d, window = 32, 42966, 49981, 64, 70
    kc, vc, _, _ = make_cache(1, 4, page, d, F16, gen(4))
    tables = torch.zeros(1, width, dtype=torch.int32, device="cuda").expand(n, width)
    q = torch.randn(n, 4, d, device="cuda", generator=gen(5)).half()
    lens = [page * width - 3 * s for s in range(n)]
    ws = torch.full((1 << 24,), float("nan"), device="cuda")
    y = cbx.paged_shared_attention(q, kc, vc, tables, ints(lens), ints([0, n]), ints([page * (width - 1)]), 0.125, window=window, ws=ws)
    one = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    short = [c[:, :, page - 200:].contiguous() for c in (kc, vc)]
    ref, bound = rows_ref(q, *short, None, None, one, [200 - 3 * s for s in range(n)], None, 0.125, window=window)
    assert_within(y, ref, bound)
    assert cbx.device_errors(clear=True) == 0


def shared_of(groups, own, page, seed=3):
    """(lens, tables, pages): groups [(first, behind, shared)] of whole pages, own[s] keys behind them."""
    n = len(own)
    pre, lead = [0] * n, list(range(n))
    for a, b, p in groups:
        assert p % page == 0
        for s in range(a, b):
            pre[s], lead[s] = p, a
    lens = [p + o for p, o in zip(pre, own)]
    pages = sum(-(-x // page) for x in lens) + 2
    order = iter(np.random.RandomState(seed).permutation(pages).tolist())
    tables = np.full((n, max(1, max(-(-x // page) for x in lens))), -1, dtype=np.int32)
    for s in range(n):
        whole = pre[s] // page if lead[s] < s else 0
        tables[s, :whole] = tables[lead[s], :whole]
        for i in range(whole, -(-lens[s] // page)):
            tables[s, i] = next(order)
    return lens, torch.from_numpy(tables).cuda(), pages


CALLS = {  # past, new of packed requests: pieces of pairs of waves, of whole row tiles, both undealt; shared beginnings
    "pieces": ([1500, 40], [3, 2]), "long": ([650, 900], [110, 100]), "pairs": ([0, 40], [50, 33]), "whole": ([0, 70], [130, 200]),
    "shared": None}


def call_of(which, page=16):
    """(lens, start or None, tables, pages, extra arguments) of one of CALLS."""
    if CALLS[which]:
        lens, start, tables, pages = packed(*CALLS[which], page, 3)
        return lens, start, tables, pages, None
    one = -(-192 // page) * page
    groups, own = [(0, 3, one), (3, 5, 4 * page)], [40, 1, 700, 33, 90]
    lens, tables, pages = shared_of(groups, own, page)
    return lens, None, tables, pages, (ints([0, 3, 5]), ints([one, 4 * page]))


def attend(cbx, q, kc, vc, ks, vs, tables, lens, start, groups, scale, **kw):
    kw = dict(kw, k_scale=ks, v_scale=vs)
    if groups:
        return cbx.paged_shared_attention(q, kc, vc, tables, ints(lens), *groups, scale, **kw)
    return cbx.paged_prompt_attention(q, kc, vc, tables, ints(lens), ints(start), scale, **kw)


@pytest.mark.parametrize("which", CALLS)
@pytest.mark.parametrize("d,g", [(64, 1), (128, 4)])
@pytest.mark.parametrize("up_k,up_v", [(1e6, 1.0), (1.0, 1e35), (1.0, 1e-33), (1e-30, 1.0)])
def test_large_and_small_8_bit_scales(cbx, which, d, g, up_k, up_v):
    """Scores of millions, values near f32's ends, as paged_attention takes them."""
    lens, start, tables, pages, groups = call_of(which)
    kc, vc, ks, vs = make_cache(pages, 2, 16, d, I8, gen(19))
    q = torch.randn(start[-1] if start else len(lens), 2 * g, d, device="cuda", generator=gen(1))
    k2, v2 = ks * up_k, vs * up_v
    y = attend(cbx, q, kc, vc, k2, v2, tables, lens, start, groups, 0.125)
    ref, bound = rows_ref(q, kc, vc, k2, v2, tables, lens, start, 0.125)
    assert bool(torch.isfinite(y).all())
    assert_within(y, ref, bound + 2.0 ** -149)


@pytest.mark.parametrize("which", CALLS)
@pytest.mark.parametrize("dt,cdt", [(F32, F32), (F32, I8)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_large_values_behind_a_rising_maximum(cbx, which, dt, cdt, d):
    """Values of 2^117 (in sum below 2^127 a row) whose scores are 7 powers of
    two above those of the first 64 keys."""
    lens, start, tables, pages, groups = call_of(which, 32)
    kc, vc, ks, vs = make_cache(pages, 2, 32, d, F32, gen(19))
    vc = vc.abs().clamp(0.25, 1.0) * 2.0 ** 116
    kc.zero_()
    rows = tables[:, 2:]
    kc[rows[rows >= 0].long(), ..., 3] = 1.0
    if cdt == I8:
        kc, vc = kc.to(I8), (vc * 2.0 ** -110).to(I8)        # 16 to 64
        ks, vs = torch.ones(pages, 2, 32, device="cuda"), torch.full((pages, 2, 32), 2.0 ** 110, device="cuda")
    else:
        ks = vs = None
    q = torch.zeros(start[-1] if start else len(lens), 2, d, device="cuda")
    q[..., 3] = 7.0
    scale = float(np.log(2.0))
    y = attend(cbx, q, kc, vc, ks, vs, tables, lens, start, groups, scale)
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, start, scale)
    assert bool(torch.isfinite(y).all())
    assert_within(y, ref, bound)


@pytest.mark.parametrize("which", CALLS)
@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("top", [2.0 ** 20, 1.37 * 2 ** 21, 1.83 * 2 ** 21, 1.11 * 2 ** 22, 2.0 ** 25, 1.37 * 2 ** 25, 1.01 * 2 ** 26,
                                 1.71 * 2 ** 26, 1.99 * 2 ** 28])
def test_equal_scores_of_millions(cbx, which, dt, cdt, top):
    """Scores of `top` powers of two, of both signs.  All keys alike: every
    score is rounded the same way, y is the mean of the row's values: n sums,
    8 more roundings as of paged_attention, and of the parts that are joined
    two exponentials, their products and a probability of two f16 parts (16
    more); 16 bits of a value times its probability under an F16 query over 8
    bits.  One key ahead of all others by a hundredth: y is its value."""
    d, page = 64, 16
    lens, start, tables, pages, groups = call_of(which, page)
    n = start[-1] if start else len(lens)
    kc, vc, ks, vs = make_cache(pages, 2, page, d, cdt, gen(7))
    q = torch.zeros(n, 2, d, dtype=dt, device="cuda")
    q[..., 3] = 1024.0
    last = []                                                # request and keys of every row
    for s, length in enumerate(lens):
        new = start[s + 1] - start[s] if start else 1
        last += [(s, length - (new - 1 - j)) for j in range(new)]
    v = [(vc[tables[s, :-(-x // page)].long()].double()
          * (1 if vs is None else vs[tables[s, :-(-x // page)].long()].double()[..., None])).transpose(0, 1).reshape(2, -1, d)
         for s, x in enumerate(lens)]
    more = (TWO_BF16 if dt == F16 and cdt == I8 else 0.0)
    for sign in (1.0, -1.0):
        high, low = (1000.0, 990.0) if sign > 0 else (990.0, 1000.0)
        unit = 1.0
        if cdt == I8:
            high, low, unit = high / 10, low / 10, 10.0
            ks = torch.full((pages, 2, page), unit, device="cuda")
        scale = sign * top / (1024.0 * 1000.0) * float(np.log(2.0))
        kc.zero_()
        kc[..., 3] = high
        y = attend(cbx, q, kc, vc, ks, vs, tables, lens, start, groups, scale)
        ref, size = (torch.stack([f(v[s][:, :x]).mean(1) for s, x in last]) for f in (lambda t: t, torch.abs))
        ends = torch.tensor([x for _, x in last], device="cuda")[:, None, None]
        assert_within(y, ref, ((ends + 24) * U32 + more) * size + half_step(dt) * ref.abs(), f"equal scores, sign {sign}")
        kc[..., 3] = low
        for s, x in enumerate(lens):
            best = 0 if start and start[s + 1] - start[s] >= x else x // 2 if start else x - 1
            kc[tables[s, best // page], :, best % page, 3] = high
        # of requests with a beginning in common the others' own best keys lie behind it: one key of the highest score each
        y = attend(cbx, q, kc, vc, ks, vs, tables, lens, start, groups, scale)
        best = [0 if start and start[s + 1] - start[s] >= lens[s] else lens[s] // 2 if start else lens[s] - 1 for s, _ in last]
        keep = torch.tensor([b < x for b, (_, x) in zip(best, last)], device="cuda")
        ref = torch.stack([v[s][:, min(b, x - 1)] for b, (s, x) in zip(best, last)])
        bound = (8 * U32 + more + half_step(dt)) * ref.abs()
        assert_within(y[keep], ref[keep], bound[keep], f"one score ahead, sign {sign}")


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, F32), (F16, F32)])
@pytest.mark.parametrize("d", [32, 40, 64, 72, 80, 96, 112, 128, 160, 248, 256, 60])
@pytest.mark.parametrize("which", ["long", "pairs", "whole", "shared"])
@pytest.mark.parametrize("page", [16, 10])
def test_infinite_keys_of_no_weight(cbx, dt, cdt, d, which, page):
    """A key with an infinity whose score is -inf has no weight, whatever the head_dim: as one that is next to it in f16."""
    lens, start, tables, pages, groups = call_of(which, page)
    kc, vc, _, _ = make_cache(pages, 2, page, d, cdt, gen(4))
    q = torch.randn(start[-1] if start else len(lens), 4, d, device="cuda", generator=gen(5)).to(dt)
    for dim in (1, d - 1):
        q[..., dim] = -1.0
    outs = []
    for far in (6e4, float("inf")):
        k2 = kc.clone()
        for s, key, dim in ((0, 3, 1), (0, 35, d - 1), (1, 20, 1)):
            k2[tables[s, key // page], :, key % page, dim] = far
        outs.append(attend(cbx, q, k2, vc, None, None, tables, lens, start, groups, 0.125))
    assert bool(torch.isfinite(outs[0][2:]).all()) and torch.equal(*outs)


@pytest.mark.parametrize("which", CALLS)
@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("cap", [2.0 ** 61, 2.0 ** 100, 3.3e38])
def test_caps_next_to_the_largest(cbx, which, dt, cdt, cap):
    """cap * tanh(s / cap) of a cap so far above the scores is s: the quotient
    is held to 2^-150 or 2^-24 of itself (2^-150 times the cap: at most 4
    U32), the tanh, products and the exponent's parts to 8 roundings of s."""
    lens, start, tables, pages, groups = call_of(which)
    kc, vc, ks, vs = make_cache(pages, 2, 16, 64, cdt, gen(4))
    q = torch.randn(start[-1] if start else len(lens), 4, 64, device="cuda", generator=gen(5)).to(dt)
    y = attend(cbx, q, kc, vc, ks, vs, tables, lens, start, groups, 0.125, softcap=cap)
    top = 0.125 * 64 * float(q.abs().max()) * 6              # above every |s|
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, start, 0.125, p_err=U32 * (8 * top + 4) + half_step(dt))
    assert_within(y, ref, bound)


@pytest.mark.parametrize("which", CALLS)
@pytest.mark.parametrize("cdt", [F32, I8])
@pytest.mark.parametrize("scale,up", [(0.0, 2.0 ** 62), (2.0 ** -140, 2.0 ** 62), (-(2.0 ** -130), 2.0 ** 62)])
def test_scales_next_to_nothing(cbx, which, cdt, scale, up):
    """Scales of 0 and below the smallest normal number, under products of up to 2^125."""
    lens, start, tables, pages, groups = call_of(which)
    kc, vc, ks, vs = make_cache(pages, 2, 16, 64, cdt, gen(4))
    if cdt == I8:
        ks = ks * up
    else:
        kc = kc * up
    q = torch.randn(start[-1] if start else len(lens), 2, 64, device="cuda", generator=gen(5)).clamp(-2, 2) * 2.0 ** 56
    y = attend(cbx, q, kc, vc, ks, vs, tables, lens, start, groups, scale)
    # |q . k| < 2^126; the scale times log2(e) is off by at most 2^-149 of its own: 2^-23, 2 U32, of the exponent
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, start, scale, p_err=4 * U32)
    assert_within(y, ref, bound)


@pytest.mark.parametrize("which", list(CALLS) + ["one"])
@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("scale", [3e38, -2.5e38])
def test_scales_next_to_the_largest(cbx, which, dt, cdt, scale):
    """Scales that log2(e) would take past f32: the query's elements times the
    scale lie below 2^126, and so do the scores."""
    lens, start, tables, pages, groups = call_of("shared" if which == "one" else which)
    kc, vc, ks, vs = make_cache(pages, 2, 16, 64, cdt, gen(4))
    # q 2^-14 to 2^-10; of the keys, 2^-24 to 2^-20 in F16, one element is not 0: scores of 2^90 and more are 0 or far apart
    q = torch.zeros(start[-1] if start else len(lens), 2, 64, dtype=dt, device="cuda")
    q[..., 5] = 2.0 ** -12
    kc.zero_()
    best = []
    for s, x in enumerate(lens):
        first = x - (start[s + 1] - start[s]) if start else x - 1
        best.append(first if start else x - 1)
        kc[tables[s, best[s] // 16], :, best[s] % 16, 5] = (1 if cdt == I8 else 2.0 ** -20) * (1 if scale > 0 else -1)
    if cdt == I8:
        ks = torch.full_like(ks, 2.0 ** -20)
    if which == "one":
        y = cbx.paged_attention(q, kc, vc, tables, ints(lens), scale, k_scale=ks, v_scale=vs)
    else:
        y = attend(cbx, q, kc, vc, ks, vs, tables, lens, start, groups, scale)
    of = [s for s in range(len(lens)) for _ in range(start[s + 1] - start[s] if start else 1)]
    page = [tables[s, best[s] // 16].long() for s in of]
    ref = torch.stack([vc[p, :, best[s] % 16].double() * (1 if vs is None else vs[p, :, best[s] % 16].double()[:, None])
                       for p, s in zip(page, of)])
    more = TWO_BF16 if dt == F16 and cdt == I8 else 0.0
    assert_within(y, ref, (8 * U32 + more + half_step(dt)) * ref.abs())
