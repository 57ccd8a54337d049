"""Rows in 8 bits: written into pages (alone and behind the norm and the
rotation), read back, and attended over by one new token a request."""
import math

import numpy as np
import pytest
import torch

from tests._paged import assert_within
from tests._paged_more import LOWEST, U32, gen, half_step, ints, make_cache, packed, page_tables, q8_ref, rows_ref

pytestmark = pytest.mark.gpu
F16, F32, I8 = torch.float16, torch.float32, torch.int8


def empty_cache(pages, hkv, page, d, permuted=False):
    shape = (pages, page, hkv, d) if permuted else (pages, hkv, page, d)
    kc, vc = (torch.full(shape, -128, dtype=I8, device="cuda") for _ in range(2))
    ks, vs = (torch.full(shape[:3], -1.0, device="cuda") for _ in range(2))
    out = (kc, vc, ks, vs)
    return tuple(x.transpose(1, 2) for x in out) if permuted else out


@pytest.mark.parametrize("permuted", [False, True])
@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("d,hkv,page", [(64, 16, 64), (128, 3, 50), (96, 2, 1), (32, 1, 16), (256, 2, 7), (512, 1, 4), (60, 3, 5),
                                        (1, 2, 3), (8, 5, 10)])
def test_store_is_the_definition(cbx, d, hkv, page, dt, permuted):
    tok, pages = 37, -(-60 // page) + 2
    g = gen(d * 7 + page)
    rows = torch.randn(tok, 2 * hkv * d + 5, device="cuda", generator=g).to(dt)
    if d % 8 == 0:                                         # both kernels: at the vectors' alignment and off it
        rows = rows[:, :2 * hkv * d].contiguous() if not permuted else rows
    k, v = rows[:, :hkv * d].unflatten(1, (hkv, d)), rows[:, hkv * d:2 * hkv * d].unflatten(1, (hkv, d))
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tok].to(torch.int32)
    slots[5::9] = -1
    kc, vc, ks, vs = empty_cache(pages, hkv, page, d, permuted)
    exp = [x.clone() for x in (kc, vc, ks, vs)]
    live = torch.nonzero(slots >= 0)[:, 0]
    at = slots[live].long()
    for x, c, s in ((k, exp[0], exp[2]), (v, exp[1], exp[3])):
        n, sc = q8_ref(x)
        c[at // page, :, at % page] = n[live]
        s[at // page, :, at % page] = sc[live]
    cbx.paged_store(k, v, slots, kc, vc, k_scale=ks, v_scale=vs)
    for got, want in zip((kc, vc, ks, vs), exp):
        assert torch.equal(got, want)
    for out_t in (F32, F16):
        bk, bv = cbx.paged_load(slots, kc, vc, k_scale=ks, v_scale=vs, dtype=out_t)
        for got, c, s in ((bk, exp[0], exp[2]), (bv, exp[1], exp[3])):
            want = torch.zeros(tok, hkv, d, device="cuda")
            want[live] = c[at // page, :, at % page].float() * s[at // page, :, at % page][..., None]
            assert torch.equal(got, want.to(out_t))
    assert cbx.device_errors(clear=True) == 0


def special_rows(d):
    rows = torch.zeros(14, 1, d, device="cuda")
    r = torch.randn(d, device="cuda", generator=gen(3))
    rows[1, 0] = r * 1e-40                                  # below the smallest normal number
    rows[2, 0] = r * 1e-37                                  # 127 / top past f32
    rows[3, 0] = r * 1e-30
    rows[4, 0] = r / r.abs().max() * torch.finfo(F32).max
    rows[5, 0] = r
    rows[5, 0, d // 2] = float("inf")
    rows[6, 0] = r
    rows[6, 0, 0] = float("nan")
    rows[7, 0, 0], rows[7, 0, 1:] = 2.0, 1.0                # 63.5: a tie, to the even 64
    rows[8, 0, 0], rows[8, 0, 1:] = -254.0, torch.arange(1, d, device="cuda") + 0.0   # whole and half steps
    rows[9, 0, 0] = 127 * 2.0 ** -126                       # the least largest element that counts as itself
    rows[9, 0, 1] = 0.5 * 2.0 ** -126
    rows[10, 0] = 1e5
    rows[10, 0, 1] = 1e-5
    rows[11, 0] = -r
    rows[12, 0, d - 1] = -3.0
    rows[13, 0] = float("-inf")
    return rows


@pytest.mark.parametrize("d", [64, 60])
def test_special_rows(cbx, d):
    x = special_rows(d)
    kc, vc, ks, vs = empty_cache(4, 1, 4, d)
    slots = torch.arange(14, dtype=torch.int32, device="cuda")
    cbx.paged_store(x, x.flip(0).contiguous(), slots, kc, vc, k_scale=ks, v_scale=vs)
    n, s = q8_ref(torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0))
    got_n, got_s = kc.reshape(16, 1, d)[:14], ks.reshape(16, 1)[:14]
    bad = [5, 6, 13]
    for i in range(14):
        if i in bad:
            assert bool(torch.isnan(got_s[i]).all()) and bool((got_n[i] == 0).all())
        else:
            assert torch.equal(got_n[i], n[i]) and torch.equal(got_s[i], s[i]), i
    assert got_n[7, 0, 1] == 64 and float(got_s[0, 0]) == 2.0 ** -126
    assert torch.equal(vc.reshape(16, d)[:14].flip(0), got_n[:, 0]) and float(got_s[9, 0]) == LOWEST / 127
    k, _ = cbx.paged_load(slots, kc, vc, k_scale=ks, v_scale=vs)
    assert torch.isnan(k).any(-1).any(-1).tolist() == [i in bad for i in range(14)]
    good = [i for i in range(14) if i not in bad]
    # |n S - x| <= S / 2; the scale is s = S (1 + u), the product k = n s (1 + u), |u| <= U32 each: S <= s (1 + 2 U32) and
    # |n S| <= |k| (1 + 3 U32), so |k - x| <= s / 2 (1 + 2 U32) + 2 U32 (1 + 4 U32) |k|
    k, x, s = k[good].double(), x[good].double(), s[good].double()[..., None]
    assert bool(((k - x).abs() <= s / 2 * (1 + 2 * U32) + 2 * U32 * (1 + 4 * U32) * k.abs()).all())


def test_store_slots_outside(cbx):
    d, page = 64, 8
    kc, vc, ks, vs = empty_cache(3, 2, page, d)
    keep = [x.clone() for x in (kc, vc, ks, vs)]
    x = torch.ones(4, 2, d, device="cuda")
    slots = ints([24, -1, -7, 1000000])
    cbx.paged_store(x, x, slots, kc, vc, k_scale=ks, v_scale=vs)
    assert cbx.device_errors(clear=True) == 4
    assert all(torch.equal(a, b) for a, b in zip((kc, vc, ks, vs), keep))
    k, v = cbx.paged_load(slots, kc, vc, k_scale=ks, v_scale=vs)
    assert cbx.device_errors(clear=True) == 4 and not k.any() and not v.any()
    none = x[:0]
    cbx.paged_store(none, none, slots[:0], kc, vc, k_scale=ks, v_scale=vs)
    assert cbx.paged_load(slots[:0], kc, vc, k_scale=ks, v_scale=vs)[0].shape == (0, 2, d)


@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("cdt", [F32, F16])
@pytest.mark.parametrize("d,permuted", [(64, False), (80, True), (20, False), (7, True)])
def test_load_of_float_pages(cbx, dt, cdt, d, permuted):
    page, hkv, tok = 6, 3, 21
    kc, vc, _, _ = make_cache(7, hkv, page, d, cdt, gen(d), permuted)
    slots = torch.randperm(42, device="cuda", generator=gen(2))[:tok].to(torch.int32)
    slots[3] = -1
    buf = torch.full((tok, 2, hkv, d + 3), 9.0, dtype=dt, device="cuda")
    out = buf[:, 0, :, :d], buf[:, 1, :, :d]
    k, v = cbx.paged_load(slots, kc, vc, dtype=dt, out=out)
    assert k.data_ptr() == buf.data_ptr()
    for got, c in ((k, kc), (v, vc)):
        at = slots.long().clamp(min=0)
        want = c[at // page, :, at % page].to(dt)
        want[3] = 0
        assert torch.equal(got, want)
    assert bool((buf[..., d:] == 9).all())


@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("hq,hkv,d,nd,mode", [(16, 16, 64, 64, 2), (10, 2, 96, 48, 0), (3, 1, 128, 128, 2), (2, 2, 256, 256, 0)])
def test_norm_rope_store_rounds_its_own_rows(cbx, hq, hkv, d, nd, mode, dt):
    """The keys are those that qk_norm_rope gives in F32, held in 8 bits."""
    tok, page = 29, 8
    g = gen(11)
    qkv = torch.randn(tok, hq + 2 * hkv, d, device="cuda", generator=g).to(dt)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    gq, gk = torch.rand(d, device="cuda", generator=g) + 0.5, torch.rand(d, device="cuda", generator=g) + 0.5
    rope = cbx.RopeCache(nd, mode=mode, n_pos=64)
    pos = torch.randint(0, 90, (tok,), device="cuda", generator=g).to(torch.int32)      # some past the table
    slots = torch.randperm(48, device="cuda", generator=g)[:tok].to(torch.int32)
    slots[-3:] = -1
    kc, vc, ks, vs = empty_cache(6, hkv, page, d)
    yq = cbx.qk_norm_rope_store(q, k, v, gq, gk, 1e-6, pos, rope, slots, kc, vc, k_scale=ks, v_scale=vs)
    eq, _ = cbx.qk_norm_rope(q, k, gq, gk, 1e-6, pos, rope)
    assert torch.equal(yq, eq)
    _, ek = cbx.qk_norm_rope(q.float(), k.float(), gq, gk, 1e-6, pos, rope)   # an F16 row's F32 result, before any rounding
    kc2, vc2, ks2, vs2 = empty_cache(6, hkv, page, d)
    cbx.paged_store(ek, v.float(), slots, kc2, vc2, k_scale=ks2, v_scale=vs2)
    for a, b in zip((kc, vc, ks, vs), (kc2, vc2, ks2, vs2)):
        assert torch.equal(a, b)
    yq = torch.empty_like(q.contiguous())                   # off the vectors' alignment: the same
    wide = torch.zeros(tok, hq + 2 * hkv, d + 1, device="cuda", dtype=dt)
    wide[..., :d] = qkv
    w = wide[..., :d]
    kc3, vc3, ks3, vs3 = empty_cache(6, hkv, page, d)
    cbx.qk_norm_rope_store(w[:, :hq], w[:, hq:hq + hkv], w[:, hq + hkv:], gq, gk, 1e-6, pos, rope, slots, kc3, vc3, out_q=yq,
                           k_scale=ks3, v_scale=vs3)
    # the same sums in another order: a key may be a rounding off, and an element next to a border a step
    assert torch.equal(vc3, vc) and torch.equal(vs3, vs)
    assert bool(((kc3.int() - kc.int()).abs() <= 1).all()) and bool(((ks3 - ks).abs() <= 4 * U32 * ks.abs()).all())
    rope.close()


CASES = [  # lens, hkv, g, d, page
    ([1, 63, 64, 65, 300, 0, 17], 4, 1, 64, 64),
    ([700, 5, 129], 2, 4, 128, 32),
    ([33, 2000], 1, 16, 96, 24),
    ([40, 41], 2, 20, 32, 5),
    ([257, 31], 1, 3, 256, 16),
    ([50, 99, 1], 2, 7, 80, 48),
    ([90, 33], 2, 2, 60, 16),
    ([20], 1, 1, 8, 16),
]


@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("lens,hkv,g,d,page", CASES)
@pytest.mark.parametrize("cap,window,permuted", [(0.0, 0, False), (3.0, 37, True)])
def test_attention_over_8_bit_pages(cbx, lens, hkv, g, d, page, dt, cap, window, permuted):
    lens, _, tables, pages = packed([0] * len(lens), lens, page, 5, width=max(1, -(-max(lens) // page)) + 2)
    kc, vc, ks, vs = make_cache(pages, hkv, page, d, I8, gen(d + page), permuted)
    q = (torch.randn(len(lens), hkv * g, d, device="cuda", generator=gen(1)) * 2).to(dt)
    y = cbx.paged_attention(q, kc, vc, tables, ints(lens), d ** -0.5, softcap=cap, window=window, k_scale=ks, v_scale=vs)
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, None, d ** -0.5, cap, window)
    assert_within(y, ref, bound)
    assert cbx.device_errors(clear=True) == 0


@pytest.mark.parametrize("page,d", [(16, 64), (5, 64), (16, 60)])
def test_what_lies_behind_a_request_stays_out(cbx, page, d):
    """Scales of NaN and infinity at keys behind the lengths and before the window, pages that are none."""
    lens = [3, 70, 0, 41]
    _, _, tables, pages = packed([0] * 4, lens, page, 6, width=20)
    kc, vc, ks, vs = make_cache(pages, 2, page, d, I8, gen(4))
    q = torch.randn(4, 4, d, device="cuda", generator=gen(5))
    args = (tables, ints(lens), 0.125)
    want = cbx.paged_attention(q, kc, vc, *args, window=30, k_scale=ks, v_scale=vs)
    seen = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        for i in range(max(0, n - 30), n):
            seen[tables[s, i // page], i % page] = True
    for bad in (float("nan"), float("inf")):
        k2, v2 = ks.clone(), vs.clone()
        k2[~seen[:, None].expand_as(k2)] = bad
        v2[~seen[:, None].expand_as(v2)] = bad
        assert torch.equal(cbx.paged_attention(q, kc, vc, *args, window=30, k_scale=k2, v_scale=v2), want)
    assert cbx.device_errors(clear=True) == 0
    wrong = tables.clone()
    wrong[1, 0], wrong[3, 1] = pages, -5
    y = cbx.paged_attention(q, kc, vc, wrong, ints(lens), 0.125, k_scale=ks, v_scale=vs)
    assert cbx.device_errors(clear=True) == 4
    ref, bound = rows_ref(q, kc, vc, ks, vs, wrong, lens, None, 0.125)
    assert_within(y, ref, bound)


def test_strided_scales(cbx):
    """Scales of every second float, and of one value a head."""
    page, d, lens = 16, 64, [40, 100]
    _, _, tables, pages = packed([0, 0], lens, page, 8)
    kc, vc, ks, vs = make_cache(pages, 2, page, d, I8, gen(9))
    q = torch.randn(2, 2, d, device="cuda", generator=gen(1))
    want = cbx.paged_attention(q, kc, vc, tables, ints(lens), 0.125, k_scale=ks, v_scale=vs)
    both = torch.stack([ks, vs], -1)
    y = cbx.paged_attention(q, kc, vc, tables, ints(lens), 0.125, k_scale=both[..., 0], v_scale=both[..., 1])
    assert torch.equal(y, want)
    one = torch.tensor([0.01, 0.02], device="cuda")[None, :, None].expand(pages, 2, page)
    ref, bound = rows_ref(q, kc, vc, one, one, tables, lens, None, 0.125)
    assert_within(cbx.paged_attention(q, kc, vc, tables, ints(lens), 0.125, k_scale=one, v_scale=one), ref, bound)


def test_large_and_small_scales(cbx):
    """Scores of millions, values near f32's ends."""
    page, d, lens = 16, 64, [90, 33]
    _, _, tables, pages = packed([0, 0], lens, page, 8)
    kc, vc, ks, vs = make_cache(pages, 2, page, d, I8, gen(19))
    q = torch.randn(2, 2, d, device="cuda", generator=gen(1))
    for up_k, up_v in ((1e6, 1.0), (1.0, 1e33), (1.0, 1e-33), (1e-30, 1.0)):
        k2, v2 = ks * up_k, vs * up_v
        ref, bound = rows_ref(q, kc, vc, k2, v2, tables, lens, None, 0.125)
        y = cbx.paged_attention(q, kc, vc, tables, ints(lens), 0.125, k_scale=k2, v_scale=v2)
        assert bool(torch.isfinite(y).all())
        assert_within(y, ref, bound + 2.0 ** -149)
    assert math.isclose(half_step(F16), 2.0 ** -11)


def test_8_bits_is_no_activation_type(cbx):
    x = torch.zeros(4, 64, dtype=I8, device="cuda")
    with pytest.raises(cbx.CbxError):
        cbx.silu(x)
    tables = page_tables([4], 4, 1, 1, 0).cuda()
    with pytest.raises(cbx.CbxError, match="unknown type"):
        cbx.paged_attention(x.view(1, 4, 64), x.view(1, 1, 4, 64), x.view(1, 1, 4, 64), tables, ints([4]), 1.0)


@pytest.mark.parametrize("d", [64, 60, 512])
def test_middles_at_every_size(cbx, d):
    """Elements in the middle of two whole numbers of steps, and the numbers
    next to these, in rows of every size that f32 has: the largest is 127 * 2^k,
    so that n + 1/2 steps are a number; and of largest elements that are not."""
    rows = []
    for k in range(-126, 121):
        n = torch.arange(d, dtype=torch.float64) * 5 % 127 + 0.5
        x = (n * 2.0 ** k).float()
        near = torch.where(torch.arange(d) % 3 == 0, x, torch.nextafter(x, torch.where(torch.arange(d) % 3 == 1, torch.inf, -torch.inf)))
        near = torch.where(torch.arange(d) % 2 == 0, near, -near)
        near[d // 2] = 127 * 2.0 ** k
        other = near.clone()
        other[d // 2] = float(np.nextafter(np.float32(127 * 2.0 ** k), np.float32(0)))
        rows += [near, other]
    x = torch.stack(rows).cuda()[:, None]
    t = x.shape[0]
    kc = torch.zeros(1, 1, t, d, dtype=torch.int8, device="cuda")
    vc, ks = torch.zeros_like(kc), torch.zeros(1, 1, t, device="cuda")
    vs = torch.zeros_like(ks)
    cbx.paged_store(x, -x, torch.arange(t, dtype=torch.int32, device="cuda"), kc, vc, ks, vs)
    q, s = q8_ref(x[:, 0])
    assert torch.equal(kc[0, 0], q) and torch.equal(ks[0, 0], s)
    assert torch.equal(vc[0, 0], -q) and torch.equal(vs[0, 0], s)
