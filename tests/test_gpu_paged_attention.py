"""paged_attention against its definition in 64 bits."""
import numpy as np
import pytest
import torch

from tests._paged import assert_within, attention_ref, gen, page_tables

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16


def ints(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


def make(lens, hkv, g, d, page, dt, cdt, seed, width=None, poison=True, q_std=1.0):
    """q, caches and tables; keys past each length, and pages of no request,
    hold NaN and infinities."""
    n = len(lens)
    pages = sum(-(-max(0, x) // page) for x in lens) + 3
    width = max([1] + [-(-x // page) for x in lens]) if width is None else width
    tables = page_tables(lens, page, width, pages, seed)
    r = gen(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=r)  # noqa: E731
    q = (rnd(n, hkv * g, d) * q_std).to(dt)
    kc, vc = rnd(pages, hkv, page, d).to(cdt), rnd(pages, hkv, page, d).to(cdt)
    if poison:
        live = torch.zeros(pages, page, dtype=torch.bool)
        for s, x in enumerate(lens):
            for i in range(-(-max(0, x) // page)):
                live[tables[s, i], :max(0, min(page, x - i * page))] = True
        dead = ~live.cuda()[:, None, :, None]
        kc = torch.where(dead, torch.full_like(kc, float("nan")), kc)
        vc = torch.where(dead, torch.full_like(vc, float("inf")), vc)
    return q, kc, vc, tables.cuda()


def check(cbx, lens, hkv, g, d, page, dt, cdt, seed, softcap=0.0, window=0, scale=None, **kw):
    q, kc, vc, tables = make(lens, hkv, g, d, page, dt, cdt, seed, **kw)
    scale = d ** -0.5 if scale is None else scale
    y = cbx.paged_attention(q, kc, vc, tables, ints(lens), scale, softcap=softcap, window=window)
    ref, bound = attention_ref(q, kc, vc, tables, lens, scale, softcap, window)
    assert_within(y, ref, bound, f"{lens[:4]} {hkv}x{g} d{d} page{page}")
    for s, x in enumerate(lens):
        if x <= 0:
            assert bool((y[s] == 0).all())
    assert cbx.device_errors(clear=True) == 0
    return y


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500]


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, F16), (F32, F32), (F16, F32)])
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 256])
def test_lengths_and_pages(cbx, dt, cdt, page):
    check(cbx, LENS, 2, 2, 64, page, dt, cdt, 100 + page)


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, F16), (F32, F32), (F16, F32)])
@pytest.mark.parametrize("d", [4, 8, 24, 32, 40, 64, 72, 80, 96, 100, 128, 136, 160, 192, 256, 264, 512])
def test_head_sizes(cbx, dt, cdt, d):
    check(cbx, [7, 0, 150, 33], 2, 3, d, 16, dt, cdt, 200 + d)


@pytest.mark.parametrize("cdt", [F16, F32])
@pytest.mark.parametrize("hkv,g", [(1, 1), (16, 1), (1, 7), (2, 8), (1, 15), (1, 16), (1, 17), (2, 24), (1, 40), (3, 5)])
def test_groups(cbx, cdt, hkv, g):
    check(cbx, [200, 1, 0, 65], hkv, g, 64, 32, F32, cdt, 300 + 17 * hkv + g)


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, F16), (F32, F32), (F16, F32)])
@pytest.mark.parametrize("d", [96, 128, 256])
@pytest.mark.parametrize("g", [1, 16, 20])
def test_large_heads_and_groups(cbx, dt, cdt, d, g):
    """The largest sums a workgroup holds (16 heads of 256), split and whole."""
    check(cbx, [900, 3, 130], 1, g, d, 16, dt, cdt, 350 + d + g)
    check(cbx, [2500], 1, g, d, 24, dt, cdt, 351 + d + g)


@pytest.mark.parametrize("dt", [F16, F32])
def test_subnormal_values(cbx, dt):
    """F16 caches of subnormal numbers (below 2^-14): kept, not flushed.  The
    scale makes the scores ordinary again; products of a subnormal with a
    query of 1 are exact in f32."""
    lens = [100, 300]
    q, kc, vc, tables = make(lens, 1, 2, 64, 16, F32, F16, 615, poison=False)
    kc, vc = (kc.float() * 2.0 ** -17).half(), (vc.float() * 2.0 ** -18).half()
    q = q.to(dt)
    y = cbx.paged_attention(q, kc, vc, tables, ints(lens), 2.0 ** 14)
    ref, bound = attention_ref(q, kc, vc, tables, lens, 2.0 ** 14)
    # results below f16's smallest normal number are rounded to its spacing
    assert_within(y, ref, bound + (2.0 ** -25 if dt == F16 else 0.0), "subnormal")


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, F16), (F32, F32)])
@pytest.mark.parametrize("lens", [[5000], [1, 9000, 3], [2049, 17, 0, 4096], [130] * 40, [20000]])
def test_long_and_ragged(cbx, dt, cdt, lens):
    check(cbx, lens, 2, 4, 64, 64, dt, cdt, 400 + len(lens) + lens[0])


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, F16), (F32, F32)])
@pytest.mark.parametrize("softcap,window", [(5.0, 0), (0.0, 1), (0.0, 50), (30.0, 129), (0.0, 1000), (2.0, 64)])
def test_cap_and_window(cbx, dt, cdt, softcap, window):
    check(cbx, [0, 1, 49, 50, 51, 128, 700, 3000], 2, 2, 64, 24, dt, cdt, 500 + window, softcap=softcap, window=window)


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, F16), (F32, F32)])
def test_peaked_scores_and_rising_maximum(cbx, dt, cdt):
    """Scores of tens that keep rising along the keys (the running maximum is
    replaced again and again), then falling; a scale of 0 (the mean) and a
    negative one."""
    lens = [700, 333]
    q, kc, vc, tables = make(lens, 1, 2, 64, 16, dt, cdt, 600, q_std=1.0)
    ramp = torch.zeros_like(kc)
    for s, x in enumerate(lens):
        for i in range(x):
            ramp[tables[s, i // 16], 0, i % 16] = (i if s == 0 else -i) * 0.004
    kc = torch.where(torch.isnan(kc), kc, kc * 0.2 + ramp)
    q = q.abs()
    for scale in (0.6, 0.0, -0.3):
        y = cbx.paged_attention(q, kc, vc, tables, ints(lens), scale)
        ref, bound = attention_ref(q, kc, vc, tables, lens, scale)
        assert_within(y, ref, bound, f"scale {scale}")


@pytest.mark.parametrize("cdt", [F16, F32])
def test_large_and_small_queries(cbx, cdt):
    """F32 queries beyond f16's range, and far below it, against caches of
    ordinary values; a query of zeros."""
    lens = [90, 200, 40]
    q, kc, vc, tables = make(lens, 2, 2, 64, 16, F32, cdt, 610)
    q[0] *= 1e6
    q[1] *= 1e-9
    q[2] = 0
    for scale in (1e-7, 1.0):
        if scale == 1.0:
            q[0] *= 1e-7
        y = cbx.paged_attention(q, kc, vc, tables, ints(lens), scale)
        ref, bound = attention_ref(q, kc, vc, tables, lens, scale)
        assert_within(y, ref, bound, f"scale {scale}")


def test_many_small_probabilities(cbx):
    """One key far above 20000 others of nearly equal weight: what they add up
    to counts, though each is 2^-14 of the largest."""
    n = 20000
    q, kc, vc, tables = make([n], 1, 1, 64, 64, F32, F16, 620, poison=False)
    q.zero_()
    q[0, 0, 0] = 1.0
    kc[..., 0] = 0
    kc[tables[0, 3], 0, 5, 0] = 9.7
    y = cbx.paged_attention(q, kc, vc, tables, ints([n]), 1.0)
    ref, bound = attention_ref(q, kc, vc, tables, [n], 1.0)
    assert_within(y, ref, bound, "small probabilities")


@pytest.mark.parametrize("cdt", [F16, F32])
def test_orders_strides_and_alignment(cbx, cdt):
    """Pages with the heads inside the tokens, K and V of one allocation,
    values at an odd offset (no vector loads), strided q, y and tables."""
    lens, hkv, g, d, page = [70, 0, 129, 16], 2, 2, 64, 16
    q, kc, vc, tables = make(lens, hkv, g, d, page, F32, cdt, 700)
    ref, bound = attention_ref(q, kc, vc, tables, lens, 0.125)
    n = kc.shape[0]
    inner = torch.stack([kc, vc], 1).permute(0, 3, 1, 2, 4).contiguous()          # [pages, page, 2, hkv, d]
    orders = [(inner[:, :, 0].transpose(1, 2), inner[:, :, 1].transpose(1, 2))]
    wide = torch.zeros(n, hkv, page, 2 * d + 8, dtype=cdt, device="cuda")
    wide[..., :d], wide[..., d + 8:] = kc, vc
    orders.append((wide[..., :d], wide[..., d + 8:]))
    odd = torch.zeros(n, hkv, page, 2 * d + 3, dtype=cdt, device="cuda")
    odd[..., 1:1 + d], odd[..., d + 2:2 * d + 2] = kc, vc
    orders.append((odd[..., 1:1 + d], odd[..., d + 2:2 * d + 2]))
    qs = torch.zeros(len(lens), hkv * g + 1, d + 3, device="cuda")[:, 1:, 2:2 + d]
    qs.copy_(q)
    ts = torch.full((len(lens), tables.shape[1] + 5), 10 ** 6, dtype=torch.int32, device="cuda")[:, 2:2 + tables.shape[1]]
    ts.copy_(tables)
    for i, (k, v) in enumerate(orders):
        out = torch.full((len(lens), hkv * g, d + 7), 3.5, device="cuda")
        y = cbx.paged_attention(qs, k, v, ts, ints(lens), 0.125, out=out[:, :, 2:2 + d])
        assert_within(y, ref, bound, f"order {i}")
        assert bool((out[:, :, :2] == 3.5).all()) and bool((out[:, :, 2 + d:] == 3.5).all())
    one = q[:1].expand(len(lens), -1, -1)                                           # one query for all
    r1, b1 = attention_ref(one, kc, vc, tables, lens, 0.125)
    assert_within(cbx.paged_attention(one, kc, vc, tables, ints(lens), 0.125), r1, b1, "broadcast q")


@pytest.mark.parametrize("cdt", [F16, F32])
@pytest.mark.parametrize("page", [16, 5, 64])
def test_bad_pages_and_lengths(cbx, cdt, page):
    """Entries that are no page leave their keys out, lengths past the table
    end at it, negative ones are empty; each raises bit 2.  Entries behind a
    request's pages are never read as pages."""
    lens = [100, 60, 40, 30]
    q, kc, vc, tables = make(lens, 2, 1, 64, page, F32, cdt, 800 + page, poison=False)
    y0 = cbx.paged_attention(q, kc, vc, tables, ints(lens), 0.125)
    behind = tables.clone()
    behind[1:, -1] = 2 ** 30
    assert torch.equal(cbx.paged_attention(q, kc, vc, behind, ints(lens), 0.125), y0)
    assert cbx.device_errors(clear=True) == 0
    bad = tables.clone()
    bad[0, 1], bad[1, 0] = kc.shape[0], -1
    ref, bound = attention_ref(q, kc, vc, bad, lens, 0.125)
    assert_within(cbx.paged_attention(q, kc, vc, bad, ints(lens), 0.125), ref, bound, "bad pages")
    assert cbx.device_errors(clear=True) == 4
    cap = tables.shape[1] * page
    y = cbx.paged_attention(q, kc, vc, tables.clamp(min=0), ints([cap + 999, -5, 40, 2 ** 31 - 1]), 0.125)
    assert cbx.device_errors(clear=True) == 4
    ref, bound = attention_ref(q, kc, vc, tables.clamp(min=0), [cap, 0, 40, cap], 0.125)
    assert_within(y, ref, bound, "bad lengths")


def test_far_pages(cbx):
    """A cache of more than 2^31 elements: pages whose byte offsets pass 32 bits."""
    hkv, d, page = 4, 128, 256
    pages = 17000
    kc = torch.zeros(pages, hkv, page, d, dtype=F16, device="cuda")
    vc = torch.zeros_like(kc)
    use = [0, pages - 1, 8192, 16384, 16500]
    r = gen(810)
    for p in use:
        kc[p] = torch.randn(hkv, page, d, device="cuda", generator=r).half()
        vc[p] = torch.randn(hkv, page, d, device="cuda", generator=r).half()
    tables = ints([use, [pages - 1, 3, 4, 5, 6]])
    q = torch.randn(2, 8, d, device="cuda", generator=r).half()
    lens = [5 * page - 3, 200]
    ref, bound = attention_ref(q, kc, vc, tables, lens, 0.09)
    assert_within(cbx.paged_attention(q, kc, vc, tables, ints(lens), 0.09), ref, bound, "far pages")


def test_infinite_and_nan_values_in_use(cbx):
    """What torch makes of them: a NaN key or query gives its heads NaN, a key
    whose score is -inf has weight 0."""
    q, kc, vc, tables = make([40, 40, 40], 1, 1, 64, 16, F32, F32, 820)
    q = q.abs()
    kc[tables[0, 1], 0, 3, 7] = float("nan")
    kc[tables[1, 1], 0, 3, 7] = float("-inf")
    y = cbx.paged_attention(q, kc, vc, tables, ints([40, 40, 40]), 0.125)
    assert bool(torch.isnan(y[0]).all()) and bool(torch.isfinite(y[1:]).all())
    rows = tables[1, :3].long()
    k, v = (c[rows, 0].reshape(-1, 64)[:40].double() for c in (kc, vc))
    exp = torch.softmax((q[1].double() @ k.T) * 0.125, -1) @ v
    assert float((y[1].double() - exp).abs().max()) < 1e-5


def test_refusals_and_nothing_to_do(cbx):
    q, kc, vc, tables = make([20], 2, 2, 64, 16, F16, F16, 830)
    lens = ints([20])
    assert cbx.paged_attention(q[:0], kc, vc, tables[:0], lens[:0], 0.125).shape == (0, 4, 64)
    need = cbx.paged_attention_workspace(q, kc, tables.expand(1, -1))
    if need:
        with pytest.raises(cbx.CbxError, match="ws needs"):
            cbx.paged_attention(q, kc, vc, tables, lens, 0.125, ws=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    with pytest.raises(cbx.CbxError, match="tensors on"):
        cbx.paged_attention(q, kc, vc, tables.cpu(), lens, 0.125)
    with pytest.raises(cbx.CbxError, match="overlap"):
        cbx.paged_attention(q, kc, vc, tables, lens, 0.125, out=q)


def test_captured_step_follows_the_lengths(cbx):
    """One graph, replayed as the device-side lengths and tables change, with
    eager work between; two graphs over one workspace replayed in turn; a
    stream of its own."""
    n, hkv, g, d, page, width = 6, 2, 2, 64, 16, 40
    q, kc, vc, tables = make([width * page] * n, hkv, g, d, page, F16, F16, 840)
    lens = ints([1] * n)
    ws = torch.empty(max(16, cbx.paged_attention_workspace(q, kc, tables)), dtype=torch.uint8, device="cuda")
    outs = [torch.zeros_like(q) for _ in range(2)]
    cbx.paged_attention(q, kc, vc, tables, lens, 0.125, ws=ws)
    side = torch.cuda.Stream()
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cbx.paged_attention(q, kc, vc, tables, lens, 0.125, window=0 if i == 0 else 77, out=outs[i], ws=ws)
        graphs.append(graph)
    own = torch.cuda.CUDAGraph()
    with torch.cuda.graph(own):
        own_out = cbx.paged_attention(q, kc, vc, tables, lens, 0.125)          # scratch of the graph's pool
    for step, now in enumerate([[1] * n, [640, 0, 3, 200, 129, 1], [17, 640, 640, 640, 640, 640], [300] * n]):
        lens.copy_(ints(now))
        for i in range(2):
            outs[i].fill_(float("nan"))
            graphs[i].replay()
        own.replay()
        eager = cbx.paged_attention(q, kc, vc, tables, lens, 0.125)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = cbx.paged_attention(q, kc, vc, tables, lens, 0.125)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for i in range(2):
            ref, bound = attention_ref(q, kc, vc, tables, now, 0.125, window=0 if i == 0 else 77)
            assert_within(outs[i], ref, bound, f"step {step} graph {i}")
        for t in (eager, own_out, other):
            assert torch.equal(t, outs[0]), f"step {step}"


@pytest.mark.parametrize("lens", [LENS, [1], [129], [4000, 1], [0, 0, 300]])
def test_workspace_needs_no_preparation(cbx, lens):
    """Scratch full of NaN and of ones: nothing in it is read before it is
    written, also where there are fewer tiles than workgroups."""
    q, kc, vc, tables = make(lens, 2, 2, 64, 16, F32, F16, 845)
    need = cbx.paged_attention_workspace(q, kc, tables)
    ref, bound = attention_ref(q, kc, vc, tables, lens, 0.125)
    for fill in (float("nan"), 1.0):
        ws = torch.full((need // 4 + 4,), fill, device="cuda")
        assert_within(cbx.paged_attention(q, kc, vc, tables, ints(lens), 0.125, ws=ws), ref, bound, f"ws of {fill}")


def test_two_streams_at_once(cbx):
    """Calls on two streams without order between them, each with scratch of
    its own: the same results as one after the other."""
    lens = [[3000, 1, 777, 0], [12, 2500, 2500, 64]]
    sets = [make(n, 2, 4, 64, 16, F16, F16, 846 + i) for i, n in enumerate(lens)]
    alone = [cbx.paged_attention(*s, ints(n), 0.125) for s, n in zip(sets, lens)]
    devs = [ints(n) for n in lens]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(cbx.paged_attention(*sets[i], devs[i], 0.125))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, alone[i]) for y in got[i])


def test_same_call_same_bits(cbx):
    lens = [3000, 5, 1234, 0, 777]
    q, kc, vc, tables = make(lens, 2, 4, 128, 32, F16, F16, 850)
    first = cbx.paged_attention(q, kc, vc, tables, ints(lens), 0.09)
    for _ in range(5):
        assert torch.equal(cbx.paged_attention(q, kc, vc, tables, ints(lens), 0.09), first)
