"""One new token a request, where groups of requests begin with the same pages."""
import numpy as np
import pytest
import torch

from tests._paged import assert_within
from tests._paged_more import gen, ints, make_cache, rows_ref

pytestmark = pytest.mark.gpu
F16, F32, I8 = torch.float16, torch.float32, torch.int8
TYPES = [(F16, F16), (F32, F16), (F32, F32), (F16, F32), (F16, I8), (F32, I8)]


def build(groups, own, page, width=None, seed=3):
    """(lens, tables, pages) of requests: groups [(first, behind, shared)], own[s] keys behind the shared ones; requests in no group
    have own keys alone.  The shared part may end inside a page: the rest of that page then is every request's own copy."""
    n = len(own)
    pre = [0] * n
    for a, b, p in groups:
        for s in range(a, b):
            pre[s] = p
    lens = [p + o for p, o in zip(pre, own)]
    width = width or max(1, max(-(-x // page) for x in lens)) + 1
    order = iter(np.random.RandomState(seed).permutation(sum(-(-x // page) for x in lens) + 4).tolist())
    tables = np.full((n, width), -1, dtype=np.int32)
    for s in range(n):
        lead = next((a for a, b, p in groups if a <= s < b), s)
        whole = pre[s] // page if lead < s else 0
        tables[s, :whole] = tables[lead, :whole]
        for i in range(whole, -(-lens[s] // page)):
            tables[s, i] = next(order)
    return lens, torch.from_numpy(tables).cuda(), sum(-(-x // page) for x in lens) + 4


def check(cbx, dt, cdt, groups, own, hkv, g, d, page, cap=0.0, window=0, permuted=False, cut=None, width=None):
    lens, tables, pages = build(groups, own, page, width)
    kc, vc, ks, vs = make_cache(pages, hkv, page, d, cdt, gen(d + page), permuted)
    for a, b, p in groups:                                  # the page that a shared part ends in: its keys are copies
        for s in range(a + 1, b):
            if p % page:
                i, j = int(tables[a, p // page]), int(tables[s, p // page])
                if i >= 0 and j >= 0:
                    for c in (kc, vc, ks, vs):
                        if c is not None:
                            c[j, :, :p % page] = c[i, :, :p % page]
    if cut:
        lens = cut(lens)
    q = (torch.randn(len(own), hkv * g, d, device="cuda", generator=gen(1)) * 2).to(dt)
    start, pre = ints([a for a, _, _ in groups] + [groups[-1][1]]), ints([p for _, _, p in groups])
    y = cbx.paged_shared_attention(q, kc, vc, tables, ints(lens), start, pre, d ** -0.5, softcap=cap, window=window, k_scale=ks,
                                   v_scale=vs)
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, None, d ** -0.5, cap, window)
    assert_within(y, ref, bound, f"{dt} {cdt} d {d} page {page}")
    assert cbx.device_errors(clear=True) == 0
    return q, kc, vc, ks, vs, tables, lens, start, pre, y


CASES = [  # groups, own, hkv, g, d, page
    ([(0, 5, 128)], [1, 70, 0, 33, 64], 2, 1, 64, 64),
    ([(0, 3, 320), (3, 4, 64), (4, 9, 96)], [5, 0, 200, 17, 1, 2, 3, 4, 90], 1, 4, 128, 32),
    ([(0, 2, 0), (2, 2, 500), (2, 6, 45)], [10, 0, 33, 34, 35, 200], 2, 5, 80, 5),
    ([(1, 4, 30)], [50, 3, 4, 5, 60, 0], 2, 3, 96, 10),
    ([(0, 40, 1024)], [i * 3 % 50 for i in range(40)], 1, 1, 32, 16),
    ([(0, 3, 50)], [9, 8, 7], 1, 20, 256, 16),
    ([(0, 3, 50)], [9, 8, 7], 2, 2, 60, 16),
    ([(0, 2, 9)], [2, 1], 1, 3, 7, 3),
    ([(0, 17, 700), (17, 20, 700)], [i for i in range(20)], 2, 16, 64, 64),
]


@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("groups,own,hkv,g,d,page", CASES)
def test_against_the_definition(cbx, dt, cdt, groups, own, hkv, g, d, page):
    check(cbx, dt, cdt, groups, own, hkv, g, d, page)


@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("cap,window", [(4.0, 0), (0.0, 100), (10.0, 33), (0.0, 1)])
def test_caps_and_windows(cbx, dt, cdt, cap, window):
    """Windows that begin in the shared part of some requests and behind it of others."""
    check(cbx, dt, cdt, [(0, 4, 128), (4, 6, 64)], [1, 40, 90, 150, 20, 0], 2, 3, 64, 16, cap, window)
    check(cbx, dt, cdt, [(0, 4, 130), (4, 6, 64)], [1, 40, 90, 150, 20, 0], 1, 2, 128, 12, cap, window, permuted=True)


@pytest.mark.parametrize("dt,cdt", TYPES)
def test_long_beginnings(cbx, dt, cdt):
    """Shared and own keys dealt to several workgroups each."""
    check(cbx, dt, cdt, [(0, 3, 6000), (3, 4, 400)], [3000, 1, 10, 2500], 1, 2, 64, 16, width=600)
    check(cbx, dt, cdt, [(0, 3, 3000)], [1500, 1, 10], 2, 1, 128, 24, width=300)


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, I8), (F32, F32)])
@pytest.mark.parametrize("d", [64, 60])
def test_requests_shorter_than_the_shared_part(cbx, dt, cdt, d):
    """A request that sits out (length 0) or is within the shared keys still."""
    check(cbx, dt, cdt, [(0, 5, 128), (5, 7, 64)], [5, 0, 200, 17, 1, 3, 9], 2, 2, d, 32,
          cut=lambda lens: [lens[0], 0, lens[2], 77, 128, 1, lens[6]])


@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("d,page", [(64, 16), (60, 16), (128, 5)])
def test_what_lies_behind_a_request_stays_out(cbx, dt, cdt, d, page):
    groups, own = [(0, 4, 80)], [1, 40, 0, 33]
    q, kc, vc, ks, vs, tables, lens, start, pre, want = check(cbx, dt, cdt, groups, own, 2, 2, d, page,
                                                              cut=lambda n: [n[0], n[1], 50, n[3]])
    want = cbx.paged_shared_attention(q, kc, vc, tables, ints(lens), start, pre, 0.125, window=70, k_scale=ks, v_scale=vs)
    hq, keep = 4, []
    # keys 60 to 79 are seen by requests 0, 1 and 3 and lie behind request 2: infinities there are its neighbours' alone
    bad = [c.clone() if c is not None else None for c in (kc, vc, ks, vs)]
    target = bad[3] if cdt == I8 else bad[1]
    target[tables[0, 60 // page], :, 60 % page] = float("inf")
    y = cbx.paged_shared_attention(q, bad[0], bad[1], tables, ints(lens), start, pre, 0.125, window=70, k_scale=bad[2], v_scale=bad[3])
    assert torch.equal(y[2], want[2]) and not bool(torch.isfinite(y[0]).all())
    # and what no request sees at all
    seen = torch.zeros(kc.shape[0], page, dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        for i in range(max(0, n - 70), n):
            seen[tables[s, i // page], i % page] = True
    hide = ~seen[:, None].expand(kc.shape[0], 2, page)
    for x in (float("nan"), float("inf")):
        bad = [c.clone() if c is not None else None for c in (kc, vc, ks, vs)]
        for c in (bad[2:] if cdt == I8 else bad[:2]):
            c[hide] = x
        y = cbx.paged_shared_attention(q, bad[0], bad[1], tables, ints(lens), start, pre, 0.125, window=70, k_scale=bad[2],
                                       v_scale=bad[3])
        assert torch.equal(y, want)
    assert hq == q.shape[1] and not keep and cbx.device_errors(clear=True) == 0


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, I8), (F32, F32)])
@pytest.mark.parametrize("d,page", [(64, 16), (60, 16)])
def test_bad_pages(cbx, dt, cdt, d, page):
    q, kc, vc, ks, vs, tables, lens, start, pre, _ = check(cbx, dt, cdt, [(0, 4, 80)], [1, 40, 0, 33], 2, 2, d, page)
    tables[:4, 2] = kc.shape[0]
    tables[1, 6] = -1
    y = cbx.paged_shared_attention(q, kc, vc, tables, ints(lens), start, pre, 0.125, k_scale=ks, v_scale=vs)
    assert cbx.device_errors(clear=True) == 4
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, None, 0.125)
    assert_within(y, ref, bound)


@pytest.mark.parametrize("d", [64, 60])
def test_shared_lengths_outside_the_table(cbx, d):
    """Below 0: nothing is shared; past the table: all of it is."""
    q, kc, vc, ks, vs, tables, lens, start, pre, want = check(cbx, F16, F16, [(0, 2, 80)], [0, 0], 1, 1, d, 16)
    for p in (-5, 1 << 30):
        y = cbx.paged_shared_attention(q, kc, vc, tables, ints(lens), start, ints([p]), d ** -0.5)
        ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, None, d ** -0.5)
        assert_within(y, ref, bound)
    cbx.device_errors(clear=True)


def test_nothing_to_do(cbx):
    kc, vc, _, _ = make_cache(3, 2, 16, 64, F16, gen(4))
    t = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    q = torch.zeros(0, 2, 64, device="cuda")
    assert cbx.paged_shared_attention(q, kc, vc, t, ints([]), ints([0, 0]), ints([5]), 0.125).shape == (0, 2, 64)
    # no group at all: paged_attention
    t = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(1, 2, 64, device="cuda", generator=gen(1))
    y = cbx.paged_shared_attention(q, kc, vc, t, ints([40]), ints([0]), ints([]), 0.125)
    ref, bound = rows_ref(q, kc, vc, None, None, t, [40], None, 0.125)
    assert_within(y, ref, bound)


def test_captured_and_replayed(cbx):
    groups, own = [(0, 6, 128), (6, 8, 64)], [1] * 8
    lens, tables, pages = build(groups, [100] * 8, 16, width=40)
    kc, vc, _, _ = make_cache(pages, 2, 16, 64, F16, gen(2))
    q = torch.randn(8, 4, 64, device="cuda", generator=gen(5)).half()
    ln, start, pre = ints([x - 90 for x in lens]), ints([0, 6, 8]), ints([128, 64])
    args = (q, kc, vc, tables, ln, start, pre, 0.125)
    outs = [torch.zeros_like(q), torch.zeros_like(q)]
    graphs = []
    cbx.paged_shared_attention(*args)
    for o in outs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            cbx.paged_shared_attention(*args, out=o)
        graphs.append(gr)
    side = torch.cuda.Stream()
    for step in range(4):
        ln += 20
        q.copy_(torch.randn_like(q))
        if step == 2:                                      # the groups change between replays
            start.copy_(ints([0, 0, 6]))
            pre.copy_(ints([64, 64]))
        want = cbx.paged_shared_attention(*args)
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        ref, bound = rows_ref(q, kc, vc, None, None, tables, ln.tolist(), None, 0.125)
        assert_within(want, ref, bound)
    assert len(own) == 8


def test_scratch_overlaps_a_tensor(cbx):
    groups, own = [(0, 6, 1280)], [40] * 6
    lens, tables, pages = build(groups, own, 16, width=100)
    kc, vc, _, _ = make_cache(pages, 2, 16, 64, F16, gen(2))
    q = torch.randn(6, 4, 64, device="cuda")
    start, pre = ints([0, 6]), ints([1280])
    need = cbx.paged_shared_attention_workspace(q, kc, tables, start)
    if need:
        with pytest.raises(cbx.CbxError, match="ws must not overlap"):
            cbx.paged_shared_attention(q, kc, vc, tables, ints(lens), start, pre, 0.125, ws=kc.view(-1))
        with pytest.raises(cbx.CbxError, match="ws needs"):
            cbx.paged_shared_attention(q, kc, vc, tables, ints(lens), start, pre, 0.125, ws=torch.zeros(4, device="cuda"))
    ws = torch.full((need // 4 + 64,), float("nan"), device="cuda")
    y = cbx.paged_shared_attention(q, kc, vc, tables, ints(lens), start, pre, 0.125, ws=ws)   # whatever the scratch holds
    assert torch.equal(y, cbx.paged_shared_attention(q, kc, vc, tables, ints(lens), start, pre, 0.125))
