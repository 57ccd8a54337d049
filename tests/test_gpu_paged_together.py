"""Prompts, shared beginnings and an 8-bit cache as a serving loop uses them:
texts cached once, requests begun on their pages, prompts, steps of one token,
drafts checked, everything given back; against 64-bit attention over what the
cache holds, and what it holds against the oracle's rows."""
import numpy as np
import pytest
import torch

from tests._paged import U32, gen, half_step
from tests._paged_more import LOWEST, ints, rows_ref

pytestmark = pytest.mark.gpu
F16, F32, I8 = torch.float16, torch.float32, torch.int8


def within(y, ref, bound, what):
    assert bool(torch.isfinite(y).all()), what
    assert bool(((y.double() - ref).abs() <= bound).all()), what


def held(x, cdt):
    """How far a cached row may be from x: its rounding; in 8 bits half a step
    of its largest element / 127, and the roundings of that quotient, of the
    row's own elements (of an F32 norm and rotation made alike) and of the
    product that reads it back: 4 of the element."""
    if cdt == F32:
        return torch.zeros_like(x.double())
    if cdt == F16:
        return half_step(F16) * x.double().abs().clamp(min=torch.finfo(F16).tiny)
    top = x.double().abs().amax(-1, keepdim=True).clamp(min=LOWEST)
    return top / 127 * (0.5 + 127 * 4 * U32)


class Server:
    def __init__(self, cbx, oracle, dt, cdt, page, hkv, g, d, pool):
        self.cbx, self.oracle, self.dt, self.cdt, self.page, self.hkv, self.g, self.d = cbx, oracle, dt, cdt, page, hkv, g, d
        self.hq, self.pool = hkv * g, pool
        self.rope = cbx.RopeCache(d, n_pos=512)
        self.gq, self.gk = torch.rand(d, device="cuda") + 0.5, torch.rand(d, device="cuda") + 0.5
        shape = (pool, hkv, page, d)
        if cdt == I8:                                    # whatever the pages held before
            self.kc = torch.full(shape, 77, dtype=I8, device="cuda")
            self.ks = torch.full(shape[:3], float("nan"), device="cuda")
            self.vs = torch.full_like(self.ks, float("inf"))
        else:
            self.kc = torch.full(shape, float("nan"), dtype=cdt, device="cuda")
            self.ks = self.vs = None
        self.vc = self.kc.clone()
        self.scales = dict(k_scale=self.ks, v_scale=self.vs)
        self.stack, self.n_free = ints(np.random.RandomState(1).permutation(pool)), ints([pool])
        self.rand = gen(7)

    def rows(self, slots):
        return torch.randn(slots, (self.hq + 2 * self.hkv) * self.d, device="cuda", generator=self.rand).to(self.dt)

    def cut(self, rows, a, h):
        return rows[:, a * self.d:(a + h) * self.d].unflatten(1, (h, self.d))

    def store(self, rows, lens, new, tables):
        """append and store of a step: (q, seq_lens, tok_start, slots, positions); lens and n_free move on."""
        ln, left, start, slots, pos = self.cbx.paged_append(lens, new, self.stack, self.n_free, tables, self.page, rows.shape[0])
        q = self.cbx.qk_norm_rope_store(self.cut(rows, 0, self.hq), self.cut(rows, self.hq, self.hkv),
                                        self.cut(rows, self.hq + self.hkv, self.hkv), self.gq, self.gk, 1e-6, pos, self.rope, slots,
                                        self.kc, self.vc, **self.scales)
        lens.copy_(ln)
        self.n_free.copy_(left)
        return q, ln, start, slots, pos

    def check_store(self, rows, q, slots, pos, n, what):
        """The first n rows reached the cache as the oracle has them."""
        k, v = self.cbx.paged_load(slots, self.kc, self.vc, **self.scales)
        assert not k[n:].any() and not v[n:].any(), what
        p = pos[:n].cpu().numpy()

        def turned(x, w):
            y = self.oracle.rms_norm_mul(x.float().cpu().numpy(), w.cpu().numpy(), 1e-6).reshape(x.shape)
            return torch.from_numpy(self.oracle.rope_ext(y, p, self.d)).cuda()

        assert torch.equal(q[:n], turned(self.cut(rows, 0, self.hq)[:n], self.gq).to(self.dt)), what
        ke = turned(self.cut(rows, self.hq, self.hkv)[:n], self.gk)
        ve = self.cut(rows, self.hq + self.hkv, self.hkv)[:n].float()
        within(k[:n], ke.double(), held(ke, self.cdt), what)
        within(v[:n], ve.double(), held(ve, self.cdt), what)

    def ref(self, q, lens, start, tables):
        return rows_ref(q, self.kc, self.vc, self.ks, self.vs, tables, lens, start, self.d ** -0.5, p_err=half_step(self.dt))

    def prompt(self, q, ln, start, tables, **kw):
        return self.cbx.paged_prompt_attention(q, self.kc, self.vc, tables, ln, start, self.d ** -0.5, **self.scales, **kw)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dt,cdt,page,hkv,g,d", [(F16, F16, 16, 2, 2, 64), (F32, F16, 16, 1, 3, 96), (F16, I8, 16, 2, 4, 128),
                                                 (F32, I8, 10, 2, 1, 64), (F32, F32, 12, 1, 2, 32), (F16, I8, 7, 1, 2, 40)])
def test_texts_takes_and_drafts(cbx, oracle, captured, dt, cdt, page, hkv, g, d):
    groups, outside, width = [(0, 3), (3, 5)], 5, 24
    n = outside + 1
    s = Server(cbx, oracle, dt, cdt, page, hkv, g, d, 8 * 2 + width * n)
    text_tables = torch.full((2, 8), -1, dtype=torch.int32, device="cuda")
    tables = torch.full((n, width), -1, dtype=torch.int32, device="cuda")

    # two texts, cached once
    texts, text_lens = [5 * page - 2, 3 * page], ints([0, 0])
    rows = s.rows(sum(texts) + 5)
    q, ln, start, slots, pos = s.store(rows, text_lens, ints(texts), text_tables)
    y = s.prompt(q, ln, start, text_tables, out=torch.full_like(q, 9.0))
    s.check_store(rows, q, slots, pos, sum(texts), "texts")
    ref, bound = s.ref(q[:sum(texts)], texts, [0, texts[0], sum(texts)], text_tables)
    within(y[:sum(texts)], ref, bound, "texts")
    assert bool((y[sum(texts):] == 9).all())

    # their whole pages are the beginnings of requests, which go on by prompts of their own
    whole = [4, 3]
    for p, (a, b) in enumerate(groups):
        tables[a:b, :whole[p]] = text_tables[p, :whole[p]]
    past = [whole[0] * page] * 3 + [whole[1] * page] * 2 + [0]
    new = [page + 3, 1, 40, 0, 2 * page, 17]
    lens = ints(past)
    rows = s.rows(sum(new) + 3)
    q, ln, start, slots, pos = s.store(rows, lens, ints(new), tables)
    y = s.prompt(q, ln, start, tables)
    s.check_store(rows, q, slots, pos, sum(new), "prompts")
    held_lens = [a + b for a, b in zip(past, new)]
    assert lens.tolist() == held_lens
    ref, bound = s.ref(q[:sum(new)], held_lens, np.concatenate([[0], np.cumsum(new)]).tolist(), tables)
    within(y[:sum(new)], ref, bound, "prompts")

    # a token a request, the beginnings read once a group
    group_start, shared = ints([0, 3, 5]), ints([w * page for w in whole])
    buf, ones = s.rows(n), ints([1] * n)

    def step():
        q, ln, start, slots, pos = s.store(buf, lens, ones, tables)
        return cbx.paged_shared_attention(q, s.kc, s.vc, tables, ln, group_start, shared, d ** -0.5, **s.scales), q, slots, pos

    graph, outs = None, None
    for i in range(page + 3):                              # past the end of a page
        buf.copy_(s.rows(n))
        if captured:
            if graph is None:
                keep = lens.clone(), s.n_free.clone(), tables.clone()
                step()                                     # warm up, then the state is set back
                lens.copy_(keep[0]), s.n_free.copy_(keep[1]), tables.copy_(keep[2])
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    outs = step()
                lens.copy_(keep[0]), s.n_free.copy_(keep[1]), tables.copy_(keep[2])
            graph.replay()
            y, q, slots, pos = outs
        else:
            y, q, slots, pos = step()
        held_lens = [x + 1 for x in held_lens]
        assert lens.tolist() == held_lens
        s.check_store(buf, q, slots, pos, n, f"step {i}")
        ref, bound = s.ref(q, held_lens, None, tables)
        within(y, ref, bound, f"step {i}")
        within(cbx.paged_attention(q, s.kc, s.vc, tables, lens, d ** -0.5, **s.scales), ref, bound, f"step {i}, alone")

    # drafts checked, some of their tokens taken back: the next ones overwrite these, and a page that this leaves empty is given back
    for taken in ([3, 1, 2, 4, 1, 2], [1, 1, 4, 2, 3, 1]):
        new = [4] * n
        rows = s.rows(4 * n)
        q, ln, start, slots, pos = s.store(rows, lens, ints(new), tables)
        y = s.prompt(q, ln, start, tables)
        s.check_store(rows, q, slots, pos, 4 * n, "drafts")
        ref, bound = s.ref(q, [x + 4 for x in held_lens], list(range(0, 4 * n + 1, 4)), tables)
        within(y, ref, bound, "drafts")
        for r in range(n):
            kept = -(-(held_lens[r] + taken[r]) // page)
            if held_lens[r] + 4 > kept * page:
                _, left = cbx.paged_release(ints([held_lens[r] + 4 - kept * page]), ints([1]), tables[r:r + 1, kept:], page, s.stack,
                                            s.n_free)
                s.n_free.copy_(left)
        held_lens = [a + b for a, b in zip(held_lens, taken)]
        lens.copy_(ints(held_lens))
        y = cbx.paged_shared_attention(q[::4], s.kc, s.vc, tables, lens, group_start, shared, d ** -0.5, **s.scales)
        ref, bound = s.ref(q[::4], held_lens, None, tables)
        within(y, ref, bound, "after drafts")

    # given back: a group's own pages behind the shared ones, the request of none, the texts
    for a, b, w in [(0, 3, whole[0]), (3, 5, whole[1]), (5, 6, 0)]:
        _, left = cbx.paged_release(lens[a:b] - w * page, ints([1] * (b - a)), tables[a:b, w:], page, s.stack, s.n_free)
        s.n_free.copy_(left)
    _, left = cbx.paged_release(text_lens, ints([1, 1]), text_tables, page, s.stack, s.n_free)
    assert left.tolist() == [s.pool] and sorted(s.stack.tolist()) == list(range(s.pool))
    assert cbx.device_errors(clear=True) == 0
    s.rope.close()


@pytest.mark.parametrize("cdt", [F16, I8])
def test_two_graphs_in_turn(cbx, cdt):
    """Two captured calls, each with scratch of its own graph's, replayed in
    turn and at once on two streams: every replay gives the eager result."""
    from tests._paged_more import make_cache, packed
    past, new = [700, 3, 1500], [3, 5, 2]
    lens, start, tables, pages = packed(past, new, 16, 3)
    kc, vc, ks, vs = make_cache(pages, 2, 16, 64, cdt, gen(4))
    kw = dict(k_scale=ks, v_scale=vs)
    ln, st, gs, sh = ints(lens), ints(start), ints([0, 1, 3]), ints([0, 0])
    q = torch.randn(10, 4, 64, device="cuda", generator=gen(5)).half()
    calls = [lambda: cbx.paged_prompt_attention(q, kc, vc, tables, ln, st, 0.125, **kw),
             lambda: cbx.paged_shared_attention(q[:3], kc, vc, tables, ln, gs, sh, 0.125, **kw),
             lambda: cbx.paged_load(ints_slots, kc, vc, **kw)[0]]
    ints_slots = (tables[:, :1].long() * 16 + torch.arange(3, device="cuda")).flatten().int()
    eager = [c() for c in calls]
    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in calls]
    for turn in range(4):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for i, g in enumerate(graphs):
            if turn % 2:
                with torch.cuda.stream(streams[i]):
                    g.replay()
            else:
                g.replay()
        torch.cuda.synchronize()
        for e, o, c in zip(eager, outs, calls):
            assert torch.equal(e, o) and torch.equal(c(), e), f"turn {turn}"
    assert cbx.device_errors(clear=True) == 0
