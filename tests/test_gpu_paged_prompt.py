"""Causal attention of all new tokens of packed requests over their pages."""
import pytest
import torch

from tests._paged import assert_within
from tests._paged_more import gen, half_step, ints, make_cache, packed, rows_ref

pytestmark = pytest.mark.gpu
F16, F32, I8 = torch.float16, torch.float32, torch.int8
TYPES = [(F16, F16), (F32, F16), (F32, F32), (F16, F32), (F16, I8), (F32, I8)]


def run(cbx, dt, cdt, past, new, hkv, g, d, page, cap=0.0, window=0, pad=3, permuted=False, seed=1, scale=None, width=None):
    lens, start, tables, pages = packed(past, new, page, seed, width=width)
    kc, vc, ks, vs = make_cache(pages, hkv, page, d, cdt, gen(seed + 1), permuted)
    q = (torch.randn(start[-1] + pad, hkv * g, d, device="cuda", generator=gen(seed + 2)) * 2).to(dt)
    out = torch.full_like(q, 7.0)
    scale = d ** -0.5 if scale is None else scale
    y = cbx.paged_prompt_attention(q, kc, vc, tables, ints(lens), ints(start), scale, softcap=cap, window=window, out=out,
                                   k_scale=ks, v_scale=vs)
    assert y.data_ptr() == out.data_ptr()
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, start, scale, cap, window, fill=7.0, p_err=half_step(dt))
    assert_within(y, ref, bound, f"{dt} {cdt} d {d} page {page}")
    assert bool((y[start[-1]:] == 7).all())
    assert cbx.device_errors(clear=True) == 0
    return q, kc, vc, ks, vs, tables, lens, start, y


SHAPES = [  # past, new, hkv, g, d, page
    ([0, 0, 0], [1, 31, 33], 2, 1, 64, 16),
    ([0, 5, 64, 0], [127, 128, 129, 0], 2, 1, 64, 64),
    ([0], [300], 1, 4, 128, 32),
    ([100, 0, 250], [1, 65, 3], 2, 5, 80, 24),
    ([17, 0], [40, 130], 1, 3, 96, 48),
    ([63, 1], [70, 2], 1, 2, 256, 16),
    ([0, 900], [20, 4], 2, 16, 32, 5),
    ([33, 12], [20, 60], 1, 20, 40, 128),
    ([7, 30], [9, 64], 2, 2, 60, 16),
    ([3, 0], [10, 5], 1, 3, 7, 3),
    ([10], [40], 1, 1, 512, 8),
]


@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("past,new,hkv,g,d,page", SHAPES)
def test_against_the_definition(cbx, dt, cdt, past, new, hkv, g, d, page):
    run(cbx, dt, cdt, past, new, hkv, g, d, page)


@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("cap,window,scale", [(5.0, 0, None), (0.0, 1, None), (0.0, 50, -0.1), (20.0, 33, 0.3), (0.0, 0, 0.0)])
@pytest.mark.parametrize("d,page", [(64, 16), (80, 10)])
def test_caps_windows_scales(cbx, dt, cdt, cap, window, scale, d, page):
    run(cbx, dt, cdt, [40, 0, 130], [100, 70, 5], 2, 3, d, page, cap, window, scale=scale)


@pytest.mark.parametrize("dt,cdt", TYPES)
def test_permuted_pages(cbx, dt, cdt):
    run(cbx, dt, cdt, [40, 0], [100, 70], 2, 2, 64, 16, permuted=True)
    run(cbx, dt, cdt, [40, 0], [30, 70], 3, 1, 128, 7, permuted=True)


@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_few_tokens_behind_many_keys(cbx, dt, cdt, d):
    """The keys of a row tile dealt to several workgroups and joined."""
    run(cbx, dt, cdt, [5000, 17, 0, 1200], [3, 1, 2, 20], 1, 4, d, 32, width=400)
    run(cbx, dt, cdt, [3000, 0], [2, 1], 2, 1, d, 10, window=700, width=600)


@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("d,page", [(64, 64), (128, 20), (60, 16)])
def test_one_token_a_request_is_paged_attention(cbx, dt, cdt, d, page):
    q, kc, vc, ks, vs, tables, lens, start, y = run(cbx, dt, cdt, [0, 99, 500, 30], [1, 1, 1, 1], 2, 2, d, page, pad=0)
    one = cbx.paged_attention(q, kc, vc, tables, ints(lens), d ** -0.5, k_scale=ks, v_scale=vs)
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, None, d ** -0.5)
    assert_within(one, ref, bound)
    assert_within(y, ref, bound + half_step(dt) * ref.abs())


@pytest.mark.parametrize("cdt", [F16, F32])
@pytest.mark.parametrize("d,page,g", [(64, 16, 1), (128, 5, 3), (96, 64, 2), (256, 32, 1), (60, 16, 2)])
@pytest.mark.parametrize("dt", [F16, F32])
def test_infinities_and_nans_of_later_tokens(cbx, cdt, dt, d, page, g):
    """Values and keys that are no numbers reach the rows that attend over them and no other."""
    past, new = [30, 0], [70, 45]
    lens, start, tables, pages = packed(past, new, page, 3)
    kc, vc, _, _ = make_cache(pages, 2, page, d, cdt, gen(4))
    q = torch.randn(start[-1], 2 * g, d, device="cuda", generator=gen(5)).to(dt)
    call = lambda k, v, w=0: cbx.paged_prompt_attention(q, k, v, tables, ints(lens), ints(start), 0.125, window=w)  # noqa: E731
    want, want_w = call(kc, vc), call(kc, vc, 20)
    for s, key, bad in ((0, 60, float("inf")), (0, 99, float("nan")), (1, 44, float("-inf")), (1, 20, float("nan"))):
        for which in (0, 1):
            k2, v2 = kc.clone(), vc.clone()
            (k2, v2)[which][tables[s, key // page], 0, key % page, 1] = bad
            t = start[s] + key - past[s]                     # the token of that key: the first to see it
            for y, base, w in ((call(k2, v2), want, 0), (call(k2, v2, 20), want_w, 20)):
                same = torch.ones(start[-1], dtype=torch.bool, device="cuda")
                same[t:start[s + 1] if not w else min(start[s + 1], t + w)] = False
                assert torch.equal(y[same], base[same]), (s, key, bad, which, w)
                assert torch.equal(y[:, g:], base[:, g:])
                if which == 1:                               # the value itself, with a weight above 0
                    row = y[t, :g, 1].float()
                    assert not bool(torch.isfinite(row).any())
                    keep = [i for i in range(d) if i != 1]
                    assert_within(y[t:t + 1, :g][:, :, keep], base[t:t + 1, :g][:, :, keep].double(),
                                  base[t:t + 1, :g][:, :, keep].double().abs() * 4 * half_step(dt) + 4 * half_step(dt))


@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("d,page", [(64, 16), (64, 10), (60, 16)])
def test_what_lies_behind_a_request_stays_out(cbx, dt, cdt, d, page):
    past, new = [30, 0, 64], [70, 45, 1]
    lens, start, tables, pages = packed(past, new, page, 3, extra=4, width=20)
    kc, vc, ks, vs = make_cache(pages, 2, page, d, cdt, gen(4))
    q = torch.randn(start[-1], 2, d, device="cuda", generator=gen(5)).to(dt)
    args = (tables, ints(lens), ints(start), 0.125)
    want = cbx.paged_prompt_attention(q, kc, vc, *args, k_scale=ks, v_scale=vs)
    seen = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        for i in range(n):
            seen[tables[s, i // page], i % page] = True
    hide = ~seen[:, None].expand(pages, 2, page)
    for bad in (float("nan"), float("inf")):
        if cdt == I8:
            k2, v2 = ks.clone(), vs.clone()
            k2[hide], v2[hide] = bad, bad
            y = cbx.paged_prompt_attention(q, kc, vc, *args, k_scale=k2, v_scale=v2)
        else:
            k2, v2 = kc.clone(), vc.clone()
            k2[hide], v2[hide] = bad, bad
            y = cbx.paged_prompt_attention(q, k2, v2, *args)
        assert torch.equal(y, want)
    assert cbx.device_errors(clear=True) == 0


@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("d,page", [(64, 16), (128, 6), (60, 16)])
def test_bad_pages_and_lengths(cbx, dt, cdt, d, page):
    past, new = [30, 0, 64], [70, 45, 10]
    lens, start, tables, pages = packed(past, new, page, 3, width=20)
    kc, vc, ks, vs = make_cache(pages, 2, page, d, cdt, gen(4))
    q = torch.randn(start[-1], 2, d, device="cuda", generator=gen(5)).to(dt)
    tables[0, 1], tables[1, 0], tables[1, 1], tables[1, 2], tables[2, 3] = -1, pages, 1 << 30, -(1 << 31), -1
    y = cbx.paged_prompt_attention(q, kc, vc, tables, ints(lens), ints(start), 0.125, k_scale=ks, v_scale=vs)
    assert cbx.device_errors(clear=True) == 4
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, start, 0.125, p_err=half_step(dt))
    assert_within(y, ref, bound)
    # more keys than the table holds: those it holds; fewer than none: none
    y = cbx.paged_prompt_attention(q, kc, vc, tables[:, :2], ints([1000, -3, 20]), ints(start), 0.125, k_scale=ks, v_scale=vs)
    assert cbx.device_errors(clear=True) == 4
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables[:, :2], [2 * page, 0, min(20, 2 * page)], start, 0.125, p_err=half_step(dt))
    assert_within(y, ref, bound)


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, I8)])
@pytest.mark.parametrize("d", [64, 60])
def test_more_tokens_than_keys(cbx, dt, cdt, d):
    """A request that append refused keeps its length: its first tokens have no key to attend over."""
    lens, start = [5, 40], [0, 200, 240]
    _, _, tables, pages = packed([0, 0], lens, 16, 3)
    kc, vc, ks, vs = make_cache(pages, 1, 16, d, cdt, gen(4))
    q = torch.randn(240, 2, d, device="cuda", generator=gen(5)).to(dt)
    y = cbx.paged_prompt_attention(q, kc, vc, tables, ints(lens), ints(start), 0.125, k_scale=ks, v_scale=vs)
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, start, 0.125, p_err=half_step(dt))
    assert_within(y, ref, bound)
    assert not y[:195].any() and cbx.device_errors(clear=True) == 0


@pytest.mark.parametrize("d", [64, 60])
def test_rows_before_the_first_request(cbx, d):
    _, _, tables, pages = packed([0, 0, 0], [20, 0, 30], 16, 3)
    kc, vc, _, _ = make_cache(pages, 2, 16, d, F16, gen(4))
    q = torch.randn(70, 2, d, device="cuda", generator=gen(5)).half()
    out = torch.full_like(q, 3.0)
    start = [11, 31, 31, 61]
    cbx.paged_prompt_attention(q, kc, vc, tables, ints([20, 0, 30]), ints(start), 0.125, out=out)
    ref, bound = rows_ref(q, kc, vc, None, None, tables, [20, 0, 30], start, 0.125, fill=3.0, p_err=half_step(F16))
    assert_within(out, ref, bound)
    assert bool((out[:11] == 3).all()) and bool((out[61:] == 3).all())


def test_nothing_to_do(cbx):
    kc, vc, _, _ = make_cache(3, 2, 16, 64, F16, gen(4))
    none = torch.zeros(0, 2, 64, device="cuda")
    t = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    assert cbx.paged_prompt_attention(none, kc, vc, t, ints([0, 0]), ints([0, 0, 0]), 0.125).shape == (0, 2, 64)
    q = torch.zeros(4, 2, 64, device="cuda")
    out = torch.full_like(q, 5.0)
    cbx.paged_prompt_attention(q, kc, vc, t[:0], ints([]), ints([0]), 0.125, out=out)
    assert bool((out == 5).all())
    cbx.paged_prompt_attention(q, kc, vc, t[:, :0], ints([0, 0]), ints([0, 1, 3]), 0.125, out=out)   # tables without entries
    assert not out[:3].any() and bool((out[3] == 5).all())


@pytest.mark.parametrize("cdt", [F16, F32, I8])
@pytest.mark.parametrize("up", [3e6, 1e-20, 1e9])
def test_scores_of_any_size(cbx, cdt, up):
    """F32 queries far from 1 (to 2^100 of each other in one head), scores of millions and more."""
    past, new, d = [0, 40], [90, 33], 64
    lens, start, tables, pages = packed(past, new, 16, 3)
    kc, vc, ks, vs = make_cache(pages, 2, 16, d, cdt, gen(4))
    q = torch.randn(start[-1], 2, d, device="cuda", generator=gen(5)) * up
    y = cbx.paged_prompt_attention(q, kc, vc, tables, ints(lens), ints(start), 0.125, k_scale=ks, v_scale=vs)
    assert bool(torch.isfinite(y).all())
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, start, 0.125)
    assert_within(y, ref, bound)
    q = torch.randn(start[-1], 2, d, device="cuda", generator=gen(5))
    q[:, :, ::2] *= 2.0 ** -11 / 3                           # small elements beside large ones
    k2 = kc
    if cdt != I8:
        k2 = kc.clone()
        k2[..., ::2] *= 300
        k2[..., 1::2] *= 1 / 64
    y = cbx.paged_prompt_attention(q, k2, vc, tables, ints(lens), ints(start), 0.125, k_scale=ks, v_scale=vs)
    ref, bound = rows_ref(q, k2, vc, ks, vs, tables, lens, start, 0.125)
    assert_within(y, ref, bound)


def test_scores_of_millions_in_f16(cbx):
    past, new, d = [0, 40], [90, 33], 128
    lens, start, tables, pages = packed(past, new, 16, 3)
    kc, vc, _, _ = make_cache(pages, 2, 16, d, F16, gen(4))
    q = (torch.randn(start[-1], 2, d, device="cuda", generator=gen(5)) * 1e4).clamp(-6e4, 6e4).half()
    kc = (kc * 1e4).clamp(-6e4, 6e4)
    for scale in (0.125, 4.0, -1.0):
        y = cbx.paged_prompt_attention(q, kc, vc, tables, ints(lens), ints(start), scale)
        assert bool(torch.isfinite(y).all())
        ref, bound = rows_ref(q, kc, vc, None, None, tables, lens, start, scale, p_err=half_step(F16))
        assert_within(y, ref, bound)


@pytest.mark.parametrize("dt", [F16, F32])
def test_views_and_alignments(cbx, dt):
    """q a view of a projection's output, y one of a wider row, both off 16 bytes; tables a view of a wider table."""
    d, hkv, g, page = 64, 2, 2, 16
    lens, start, tables, pages = packed([10, 0], [50, 70], page, 3)
    kc, vc, _, _ = make_cache(pages, hkv, page, d, F16, gen(4))
    wide = torch.randn(start[-1] + 1, (hkv * g + 3) * d + 1, device="cuda", generator=gen(5)).to(dt)
    q = wide[:, 1:1 + hkv * g * d].unflatten(1, (hkv * g, d))
    buf = torch.full((start[-1] + 1, hkv * g, d + 3), 2.0, device="cuda", dtype=dt)
    big = torch.full((2, tables.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    big[:, 2:2 + tables.shape[1]] = tables
    y = cbx.paged_prompt_attention(q, kc, vc, big[:, 2:], ints(lens), ints(start), 0.2, out=buf[..., 1:1 + d])
    ref, bound = rows_ref(q, kc, vc, None, None, tables, lens, start, 0.2, fill=2.0, p_err=half_step(dt))
    assert_within(y, ref, bound)
    assert bool((buf[..., 0] == 2).all()) and bool((buf[..., 1 + d:] == 2).all()) and bool((buf[-1] == 2).all())
    odd = torch.zeros(pages * hkv * page * d + 1, dtype=F16, device="cuda")[1:].view_as(kc)
    odd.copy_(kc)
    y2 = cbx.paged_prompt_attention(q, odd, vc, tables, ints(lens), ints(start), 0.2, out=torch.full_like(y, 2.0))
    assert_within(y2, ref, bound)


def test_many_requests(cbx):
    """More requests than a wave has lanes, most of them without tokens."""
    n = 700
    new = [(i * 7) % 5 if i % 3 == 0 else 0 for i in range(n)]
    past = [(i * 13) % 90 for i in range(n)]
    run(cbx, F16, F16, past, new, 1, 2, 64, 16)
    run(cbx, F32, I8, past, new, 1, 1, 60, 16)


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, F16), (F16, I8)])
def test_a_long_prompt(cbx, dt, cdt):
    """Rows of a prompt of thousands, a sample of them checked: the last rows, and what the first tiles give."""
    n, d, page, hkv, g = 4111, 128, 32, 2, 4
    lens, start, tables, pages = packed([0], [n], page, 3)
    kc, vc, ks, vs = make_cache(pages, hkv, page, d, cdt, gen(4))
    q = torch.randn(n, hkv * g, d, device="cuda", generator=gen(5)).to(dt)
    y = cbx.paged_prompt_attention(q, kc, vc, tables, ints(lens), ints(start), d ** -0.5, k_scale=ks, v_scale=vs)
    for a, b in ((0, 40), (1000, 1030), (4080, 4111)):
        ref, bound = rows_ref(q[a:b], kc, vc, ks, vs, tables, [b], [0, b - a], d ** -0.5, p_err=half_step(dt))
        assert_within(y[a:b], ref, bound)


def test_captured_and_replayed(cbx):
    """One captured call over requests that grow, chunk after chunk, against the eager call; two graphs with scratch of their own."""
    d, page, n, width = 64, 16, 3, 40
    kc, vc, _, _ = make_cache(n * width, 2, page, d, F16, gen(4))
    tables = torch.randperm(n * width, device="cuda", generator=gen(1)).to(torch.int32).view(n, width)
    q = torch.randn(50, 4, d, device="cuda", generator=gen(5)).half()
    lens, start = ints([0] * n), ints([0] * (n + 1))
    outs = [torch.zeros_like(q), torch.zeros_like(q)]
    graphs = []
    cbx.paged_prompt_attention(q, kc, vc, tables, lens, start, 0.125)
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cbx.paged_prompt_attention(q, kc, vc, tables, lens, start, 0.125, out=o)
        graphs.append(g)
    for step in ([10, 0, 40], [1, 1, 1], [0, 48, 2], [17, 17, 16]):
        lens += ints(step)
        start.copy_(ints([0, step[0], step[0] + step[1], sum(step)]))
        q.copy_(torch.randn_like(q))
        want = cbx.paged_prompt_attention(q, kc, vc, tables, lens, start, 0.125, out=torch.zeros_like(q))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for o, g in zip(outs, graphs):
            o.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_two_streams(cbx):
    a = run(cbx, F16, F16, [2000, 0], [4, 90], 2, 2, 64, 16)
    q, kc, vc, _, _, tables, lens, start, y = a
    ln, st = ints(lens), ints(start)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(cbx.paged_prompt_attention(q, kc, vc, tables, ln, st, 64 ** -0.5, out=torch.full_like(q, 7.0)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o in outs)


@pytest.mark.parametrize("cdt,d", [(F16, 128), (I8, 128), (F16, 60)])
def test_pages_past_four_gigabytes(cbx, cdt, d):
    hkv, page, n = 2, 64, 3
    size = 2 if cdt == F16 else 1
    pages = (1 << 32) // (hkv * page * d * size) + 9
    kc = torch.zeros(pages, hkv, page, d, dtype=cdt, device="cuda")
    vc = torch.zeros_like(kc)
    ks = vs = None
    if cdt == I8:
        ks, vs = torch.ones(pages, hkv, page, device="cuda"), torch.ones(pages, hkv, page, device="cuda")
    k, v, s, t = make_cache(n, hkv, page, d, cdt, gen(4))
    for c, x in ((kc, k), (vc, v), (ks, s), (vs, t)):
        if c is not None:
            c[:n], c[-n:] = x, x
    q = torch.randn(70, hkv, d, device="cuda", generator=gen(5)).half()
    low = torch.arange(n, dtype=torch.int32, device="cuda")[None]
    call = lambda tab: cbx.paged_prompt_attention(q, kc, vc, tab, ints([190]), ints([0, 70]), 0.1, k_scale=ks, v_scale=vs)  # noqa: E731
    assert torch.equal(call(low), call(low + pages - n))


@pytest.mark.parametrize("dt,cdt", [(F16, F16), (F32, F16), (F16, I8), (F32, F32)])
def test_lengths_up_to_the_last(cbx, dt, cdt):
    """2^31 - 2 keys, the most that a table can hold, all in one page that its
    entries repeat: the window's keys are the page's last."""
    page, width, d, n, window = 42966, 49981, 64, 5, 70
    kc, vc, ks, vs = make_cache(1, 2, page, d, cdt, gen(4))
    tables = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    q = torch.randn(n, 4, d, device="cuda", generator=gen(5)).to(dt)
    last = slice(page - 200, page)
    short = [c[:, :, last].contiguous() if c is not None else None for c in (kc, vc, ks, vs)]
    one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    y = cbx.paged_prompt_attention(q, kc, vc, tables, ints([page * width]), ints([0, n]), 0.125, window=window, k_scale=ks, v_scale=vs)
    ref, bound = rows_ref(q, *short, one, [200], [0, n], 0.125, window=window, p_err=half_step(dt))
    assert_within(y, ref, bound)
    both = tables.expand(2, width)
    y = cbx.paged_shared_attention(q[:2], kc, vc, both, ints([page * width, page * width - 3]), ints([0, 2]), ints([page * width]),
                                   0.125, window=window, k_scale=ks, v_scale=vs)
    ref, bound = rows_ref(q[:2], *short, one.expand(2, 1), [200, 197], None, 0.125, window=window, p_err=half_step(dt))
    assert_within(y, ref, bound)
    assert cbx.device_errors(clear=True) == 0


@pytest.mark.parametrize("dt,cdt", TYPES)
def test_a_cap_next_to_nothing(cbx, dt, cdt):
    """softcap 2^-140: every score is 0 to f32's precision, also one that was 0 before."""
    lens, start, tables, pages = packed([100, 0], [20, 30], 16, 3)
    kc, vc, ks, vs = make_cache(pages, 2, 16, 64, cdt, gen(4))
    q = torch.randn(50, 4, 64, device="cuda", generator=gen(5)).to(dt)
    q[3], q[40] = 0, 0
    y = cbx.paged_prompt_attention(q, kc, vc, tables, ints(lens), ints(start), 0.125, softcap=2.0 ** -140, k_scale=ks, v_scale=vs)
    ref, bound = rows_ref(q, kc, vc, ks, vs, tables, lens, start, 0.125, 2.0 ** -140, p_err=half_step(dt))
    assert_within(y, ref, bound)
