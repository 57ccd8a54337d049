"""Prompt attention of F16 queries over F16 pages in calls of 4096 rows
(tokens times heads) and more, which hold a probability in one f16, and how far
the smaller calls, which hold it in two, may be off."""
import pytest
import torch

from tests._paged import assert_within
from tests._paged_more import gen, half_step, ints, make_cache, packed, rows_ref

pytestmark = pytest.mark.gpu
F16, F32, I8 = torch.float16, torch.float32, torch.int8
MOST = 4096                            # rows from which on a probability is one f16

# past, new, hkv, g: the forms of the kernel, all with 4096 rows or more
MANY = {
    "whole": ([0, 70, 0, 300], [200, 150, 0, 161], 2, 4),               # row tiles of 128, undealt
    "pieces": ([700, 0], [257, 5], 1, 16),                              # dealt in pieces and joined
    "pairs": ([(i * 13) % 90 for i in range(64)], [1 + (i * 7) % 11 for i in range(64)], 4, 3),      # many short requests
    "pair pieces": ([900 + i for i in range(20)], [13] * 20, 4, 4),
    "texts": ([0, 31, 0], [90, 170, 1], 16, 1),
}
P16 = 2.0 ** -11                       # a probability rounded to f16


def small_ones(v, keys, part):
    """What probabilities below f16's normal numbers lose: `part` of the row's largest each, in the sum and in its divisor."""
    return 2 * keys * part * float(v.float().abs().max())


def call(cbx, which, d, page, cap=0.0, window=0, scale=None, permuted=False, up=2.0):
    past, new, hkv, g = MANY[which]
    lens, start, tables, pages = packed(past, new, page, 5)
    kc, vc, _, _ = make_cache(pages, hkv, page, d, F16, gen(d + page), permuted)
    q = (torch.randn(start[-1] + 2, hkv * g, d, device="cuda", generator=gen(2)) * up).half()
    assert q.shape[0] * q.shape[1] >= MOST
    scale = d ** -0.5 if scale is None else scale
    args = (ints(lens), ints(start), scale)
    y = cbx.paged_prompt_attention(q, kc, vc, tables, *args, softcap=cap, window=window, out=torch.full_like(q, 7.0))
    return q, kc, vc, tables, lens, start, scale, y


def check(cbx, which, d, page, cap=0.0, window=0, **kw):
    q, kc, vc, tables, lens, start, scale, y = call(cbx, which, d, page, cap, window, **kw)
    ref, bound = rows_ref(q, kc, vc, None, None, tables, lens, start, scale, cap, window, fill=7.0, p_err=P16)
    assert_within(y, ref, bound + small_ones(vc, max(lens), 2.0 ** -34), f"{which} d {d} page {page}")
    assert bool((y[start[-1]:] == 7).all())
    assert cbx.device_errors(clear=True) == 0


@pytest.mark.parametrize("which", MANY)
@pytest.mark.parametrize("d,page", [(64, 64), (40, 16), (80, 24), (96, 10), (128, 32), (160, 16), (256, 50)])
def test_one_part_against_the_definition(cbx, which, d, page):
    check(cbx, which, d, page)


@pytest.mark.parametrize("which", MANY)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("cap,window,scale", [(5.0, 0, None), (0.0, 1, None), (0.0, 50, -0.1), (20.0, 133, 0.3), (0.0, 0, 0.0)])
def test_one_part_caps_windows_scales(cbx, which, d, cap, window, scale):
    check(cbx, which, d, 16, cap, window, scale=scale, permuted=d == 64)


@pytest.mark.parametrize("which", MANY)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_one_part_scores_of_millions(cbx, which, d):
    check(cbx, which, d, 16, up=3e4 / 4, scale=40.0)


@pytest.mark.parametrize("which", MANY)
@pytest.mark.parametrize("d,page", [(64, 16), (80, 10), (128, 32), (256, 16)])
def test_one_part_infinities_and_nans_of_later_tokens(cbx, which, d, page):
    """Values and keys that are no numbers reach the rows that attend over them and no other."""
    q, kc, vc, tables, lens, start, scale, want = call(cbx, which, d, page)
    past, new, hkv, g = MANY[which]
    for s, bad in ((0, float("inf")), (0, float("nan")), (1, float("-inf")), (1, float("nan"))):
        t = start[s] + new[s] // 2                           # the first token that sees the key
        key = past[s] + new[s] // 2
        for i in (0, 1):
            pages = [kc.clone(), vc.clone()]
            pages[i][tables[s, key // page], 0, key % page, 1] = bad
            y = cbx.paged_prompt_attention(q, *pages, tables, ints(lens), ints(start), scale, out=torch.full_like(q, 7.0))
            same = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
            same[t:start[s + 1]] = False
            assert torch.equal(y[same], want[same]) and torch.equal(y[:, g:], want[:, g:]), (bad, i)
            if i == 1:
                assert not bool(torch.isfinite(y[t, :g, 1]).any())
                rest = [j for j in range(d) if j != 1]
                assert bool(y[t, :g][:, rest].isfinite().all())


@pytest.mark.parametrize("which", MANY)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_one_part_bad_pages_and_lengths(cbx, which, d):
    q, kc, vc, tables, lens, start, scale, _ = call(cbx, which, d, 16)
    tables[0, 1], tables[1, 0], tables[0, 4] = -1, kc.shape[0], 1 << 30
    y = cbx.paged_prompt_attention(q, kc, vc, tables, ints(lens), ints(start), scale, out=torch.full_like(q, 7.0))
    assert cbx.device_errors(clear=True) == 4
    ref, bound = rows_ref(q, kc, vc, None, None, tables, lens, start, scale, fill=7.0, p_err=P16)
    assert_within(y, ref, bound + small_ones(vc, max(lens), 2.0 ** -34))
    few = [-7, 5] + lens[2:]                                 # less than none, fewer than tokens
    y = cbx.paged_prompt_attention(q, kc, vc, tables, ints(few), ints(start), scale, out=torch.full_like(q, 7.0))
    assert cbx.device_errors(clear=True) == 4
    ref, bound = rows_ref(q, kc, vc, None, None, tables, few, start, scale, fill=7.0, p_err=P16)
    assert_within(y, ref, bound + small_ones(vc, max(lens), 2.0 ** -34))


def test_one_part_captured_and_replayed(cbx):
    q, kc, vc, tables, lens, start, scale, want = call(cbx, "pieces", 64, 16)
    ln, st, out = ints(lens), ints(start), torch.full_like(q, 7.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cbx.paged_prompt_attention(q, kc, vc, tables, ln, st, scale, out=out)
    for i in range(3):
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        q.mul_(0.5)
        want = cbx.paged_prompt_attention(q, kc, vc, tables, ln, st, scale, out=torch.full_like(q, 7.0))


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, F16), (F32, F32), (F16, F32), (F16, I8), (F32, I8)])
@pytest.mark.parametrize("past,new", [([1500, 40], [3, 2]), ([0, 40], [50, 33]), ([0, 70], [130, 200]), ([650, 900], [110, 100])])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_two_parts_of_a_probability(cbx, dt, cdt, past, new, d):
    """Scores next to 0 and values that add up to next to nothing, so that a
    probability's rounding is the largest error: 2^-23 of it in two f16 parts
    (2^-39 of the row's largest of small ones), 2^-15 in two bf16 parts cut off
    (F16 queries over 8 bits), none in three or over F32 pages."""
    page, hkv = 16, 2
    lens, start, tables, pages = packed(past, new, page, 5)
    assert start[-1] * hkv < MOST
    kc, vc, ks, vs = make_cache(pages, hkv, page, d, cdt, gen(d))
    vc[:, :, 1::2] = -vc[:, :, ::2]
    if vs is not None:
        vs[:, :, 1::2] = vs[:, :, ::2]
    q = (torch.randn(start[-1], hkv, d, device="cuda", generator=gen(2)) * 0.05).to(dt)
    y = cbx.paged_prompt_attention(q, kc, vc, tables, ints(lens), ints(start), 0.05, k_scale=ks, v_scale=vs)
    p_err = 0.0 if cdt == F32 else 2.0 ** -23 if cdt == F16 else 2.0 ** -15 if dt == F16 else 0.0
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, start, 0.05, p_err=p_err)
    most = vc.float().abs().max() if vs is None else (vc.float().abs() * vs[..., None]).max()
    assert_within(y, ref, bound + (small_ones(most, max(lens), 2.0 ** -39) if cdt == F16 else 0.0))


def test_shared_scratch_is_asked_for(cbx):
    """Groups of long beginnings need scratch, and a call refuses less of it, or such that overlaps a tensor."""
    n, page, width = 6, 16, 100
    kc, vc, _, _ = make_cache(n * width, 2, page, 64, F16, gen(2))
    tables = torch.arange(n * width, dtype=torch.int32, device="cuda").view(n, width)
    tables[:, :80] = tables[0, :80].clone()
    q = torch.randn(n, 4, 64, device="cuda", generator=gen(1))
    start, pre, lens = ints([0, n]), ints([80 * page]), ints([81 * page] * n)
    need = cbx.paged_shared_attention_workspace(q, kc, tables, start)
    assert need > 0
    for ws, text in ((kc.view(-1), "ws must not overlap"), (torch.zeros(need // 4 - 4, device="cuda"), "ws needs")):
        with pytest.raises(cbx.CbxError, match=text):
            cbx.paged_shared_attention(q, kc, vc, tables, lens, start, pre, 0.125, ws=ws)
