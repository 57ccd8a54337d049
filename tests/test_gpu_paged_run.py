"""The paged operators as a serving loop uses them: prompts admitted, decoded
token by token with requests coming and going, against attention over plain
per-request lists of keys and values."""
import numpy as np
import pytest
import torch

from tests._paged import U32, gen, half_step

pytestmark = pytest.mark.gpu


def ints(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dt,page,hkv,g,d", [(torch.float16, 16, 4, 1, 64), (torch.float32, 5, 2, 3, 32)])
def test_serving_loop(cbx, oracle, captured, dt, page, hkv, g, d):
    n, width, hq, vocab = 5, 24, hkv * g, 500
    rope = cbx.RopeCache(d, n_pos=256)
    gq, gk = torch.rand(d, device="cuda") + 0.5, torch.rand(d, device="cuda") + 0.5
    pool = n * width
    kc = torch.full((pool, hkv, page, d), float("nan"), dtype=torch.float16, device="cuda")
    vc = torch.full_like(kc, float("nan"))
    tables = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    stack, n_free = ints(np.random.RandomState(1).permutation(pool)), ints([pool])
    lens = ints([0] * n)
    hist = [[] for _ in range(n)]
    head = torch.randn(hq * d, vocab, device="cuda", generator=gen(2)) * 0.2
    qkv = torch.zeros(40, (hq + 2 * hkv) * d, device="cuda", dtype=dt)
    cut = lambda t, a, h: t[:, a * d:(a + h) * d].unflatten(1, (h, d))  # noqa: E731

    def oracle_row(x, w, p):
        y = oracle.rms_norm_mul(x.float().cpu().numpy()[None], w.cpu().numpy(), 1e-6).reshape(1, x.shape[0], d)
        return torch.from_numpy(oracle.rope_ext(y, np.array([p], dtype=np.int32), d)).cuda()[0]

    def device_step(new, slots):
        """A step's launches over the buffers (the last token of each request attends)."""
        ln, left, start, sl, pos = cbx.paged_append(lens, new, stack, n_free, tables, page, slots)
        rows = qkv[:slots]
        q = cbx.qk_norm_rope_store(cut(rows, 0, hq), cut(rows, hq, hkv), cut(rows, hq + hkv, hkv), gq, gk, 1e-6, pos, rope, sl,
                                   kc, vc)
        last = (start[1:].long() - 1).clamp(min=0)
        ql = q.index_select(0, last)
        y = cbx.paged_attention(ql, kc, vc, tables, ln, d ** -0.5)
        logits = torch.matmul(y.float().reshape(n, -1), head)
        lp, ent, ti, tl = cbx.token_log_probs(logits, ti_in, top_n=3)
        lens.copy_(ln)
        n_free.copy_(left)
        return y, ql, logits, lp, ti

    ti_in = ints([3, 1, 4, 1, 5])
    new_buf, graph, outs = ints([0] * n), None, None
    r = gen(7)
    for step in range(12):
        if step == 0:
            new, slots = [7, 0, 1, 12, 16], 40
        elif step == 4:
            new, slots = [1, 9, 0, 1, 1], 40                  # a new prompt beside decoding requests
        else:
            new, slots = [1, 1 if step > 4 else 0, 1, 1, 1], 8
        if step == 6:                                          # request 3 ends, its pages go back
            ln, left = cbx.paged_release(lens, ints([0, 0, 0, 1, 0]), tables, page, stack, n_free)
            lens.copy_(ln)
            n_free.copy_(left)
            hist[3] = []
        qkv[:slots] = torch.randn(slots, qkv.shape[1], device="cuda", generator=r).to(dt)
        new_buf.copy_(ints(new))
        before = lens.tolist()
        if captured and slots == 8:
            if graph is None:
                keep = lens.clone(), n_free.clone(), tables.clone()
                device_step(new_buf, 8)                       # warm up, then the state is set back
                lens.copy_(keep[0]), n_free.copy_(keep[1]), tables.copy_(keep[2])
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    outs = device_step(new_buf, 8)
                lens.copy_(keep[0]), n_free.copy_(keep[1]), tables.copy_(keep[2])
            graph.replay()
            y, ql, logits, lp, ti = outs
        else:
            y, ql, logits, lp, ti = device_step(new_buf, slots)
        torch.cuda.synchronize()
        assert lens.tolist() == [a + b for a, b in zip(before, new)]
        t = 0
        for s in range(n):
            for j in range(new[s]):
                row, p = qkv[t], before[s] + j
                hist[s].append((oracle_row(cut(row[None], hq, hkv)[0], gk, p).half(), cut(row[None], hq + hkv, hkv)[0].half().clone()))
                if j == new[s] - 1:
                    exp_q = oracle_row(cut(row[None], 0, hq)[0], gq, p).to(dt)
                    assert torch.equal(ql[s], exp_q), f"step {step} request {s}: q"
                t += 1
            if not hist[s]:
                assert bool((y[s] == 0).all())
                continue
            k = torch.stack([a for a, _ in hist[s]]).double().transpose(0, 1)
            v = torch.stack([b for _, b in hist[s]]).double().transpose(0, 1)
            qs = ql[s].double().reshape(hkv, g, d)
            w = torch.matmul(qs, k.transpose(1, 2).contiguous()) * d ** -0.5
            prob = torch.softmax(w, -1)
            ref = torch.matmul(prob, v).reshape(hq, d)
            size = torch.matmul(qs.abs(), k.abs().transpose(1, 2).contiguous()).amax() * d ** -0.5
            err = float(2 * U32 * ((d + 1) * size + 8 * w.abs().amax() + 4) + (len(hist[s]) + 8) * U32)
            bound = err * torch.matmul(prob, v.abs()).reshape(hq, d) + half_step(dt) * ref.abs()
            assert bool(((y[s].double() - ref).abs() <= bound + 1e-30).all()), f"step {step} request {s}"
        order = torch.argsort(logits, dim=-1, descending=True, stable=True)[:, :3]
        assert torch.equal(ti.long(), order)
        ref_lp = torch.log_softmax(logits.double(), -1).gather(1, ti_in.long()[:, None])[:, 0]
        # V exponentials and their sum: (V + 16) roundings, the logits' own size 8 more of each
        assert bool(((lp.double() - ref_lp).abs() <= U32 * (vocab + 16 + 16 * float(logits.abs().max()))).all())
    assert cbx.device_errors(clear=True) == 0
    used = int((tables >= 0).sum())
    assert used + int(n_free) == pool
    live = tables[tables >= 0].tolist() + stack[:int(n_free)].tolist()
    assert sorted(live) == list(range(pool)), "every page is in one table or on the stack"
    rope.close()
