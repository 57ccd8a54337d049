"""token_log_probs against its definition in 64 bits; tokens exactly."""
import numpy as np
import pytest
import torch

from tests._paged import U32, gen

pytestmark = pytest.mark.gpu

INF = float("inf")


def reference(x, ids, top_n, scale):
    """(logp, entropy, top ids, top logp) in float64, and the error bound of
    an f32 evaluation of each.

    z = scale x - scale max carries 3 roundings of at most |scale x| + |scale
    max|; an exponential is off by that and 4 roundings, the sum of V of them
    by at most V more (any order), the logarithm by 2 of |log T| <= log V.
    Entropy: the same relative errors on log T and on each e z / T."""
    lp = torch.log_softmax(x.double() * scale, -1)
    fin = torch.where(torch.isinf(x), torch.zeros_like(x), x).double().abs()
    m = x.amax(-1, keepdim=True).double().abs().clamp(max=1e30)
    ez = 3 * U32 * scale * (fin.amax(-1, keepdim=True) + m)
    v = x.shape[-1]
    et = ez + (4 + v) * U32 + 2 * U32 * (1 + float(np.log(v)))
    ent = torch.special.entr(lp.exp()).sum(-1)
    order = torch.argsort(x.float() + 0.0, dim=-1, descending=True, stable=True)[:, :top_n]
    out = (lp.gather(1, ids.long()[:, None])[:, 0] if ids is not None else None, ent, order, lp.gather(1, order))
    b = ez + et
    lim = lambda t: b.expand_as(t) + 2 * U32 * t.abs().nan_to_num(0, 0, 0)  # noqa: E731
    ent_b = (et[:, 0] * (1 + 2 * ent) + 3 * ez[:, 0] * (1 + ent) + 6 * U32 * (1 + ent)) + 4 * U32
    return out, (b[:, 0] + 2 * U32 * out[0].abs().nan_to_num(0, 0, 0) if ids is not None else None, ent_b, None, lim(out[3]))


def near(got, ref, bound, what):
    fin = torch.isfinite(ref)
    assert torch.equal(got[~fin].double(), ref[~fin]), f"{what}: infinities"
    d = (got.double() - ref)[fin].abs()
    assert bool((d <= bound[fin]).all()), f"{what}: {float(d.max()):.3g} past {float(bound[fin].min()):.3g}"


def check(cbx, x, ids, top_n, scale=1.0, **kw):
    logp, ent, ti, tl = cbx.token_log_probs(x, ids, top_n=top_n, scale=scale, **kw)
    ref, bound = reference(x, ids, top_n, scale)
    if ids is not None:
        near(logp, ref[0], bound[0], "logp")
    near(ent, ref[1], bound[1], "entropy")
    assert torch.equal(ti.long(), ref[2]), "top ids"
    near(tl, ref[3], bound[3], "top logp")
    assert cbx.device_errors(clear=True) == 0


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 63), (2, 64), (5, 65), (1, 255), (4, 257), (64, 8194), (1, 8194), (7, 1000),
                                        (2, 50257), (1, 151936), (300, 1031), (1100, 130)])
def test_sizes(cbx, dt, rows, vocab):
    x = (torch.randn(rows, vocab, device="cuda", generator=gen(rows + vocab)) * 3).to(dt)
    ids = torch.randint(0, vocab, (rows,), device="cuda", generator=gen(1), dtype=torch.int32)
    for top in {0, 1, min(5, vocab), min(64, vocab)}:
        check(cbx, x, ids, top, 1.0 if top else 0.7)


def test_last_chunk_of_one(cbx):
    """A row so long that its parts' rounding leaves one logit to the last."""
    x = torch.randn(1, 4096 * 1500 + 1, device="cuda", generator=gen(2))
    for last in (-50.0, 50.0):
        x[0, -1] = last
        check(cbx, x, torch.tensor([4096 * 1500], dtype=torch.int32, device="cuda"), 64)


@pytest.mark.parametrize("vocab", [100, 8194, 40000])
def test_equal_logits_go_by_number(cbx, vocab):
    """All equal; a few levels only; -0 and +0 equal."""
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.full((4, vocab), 1.5, device="cuda")
    x[1] = (torch.arange(vocab, device="cuda") % 3).float()
    x[2] = torch.where(torch.arange(vocab, device="cuda") % 2 == 0, -0.0, 0.0)
    x[3] = torch.arange(vocab, device="cuda").float() // 50 * 0.25
    for top in (1, 20, 64):
        check(cbx, x, ids, top)
        check(cbx, x.half(), ids, top)


@pytest.mark.parametrize("vocab", [300, 8194, 70000])
def test_largest_side_by_side(cbx, vocab):
    """The largest logits all next to each other, all a workgroup's width
    apart, rising and falling along the row: wherever they sit."""
    ids = torch.full((6,), 7, dtype=torch.int32, device="cuda")
    i = torch.arange(vocab, device="cuda")
    x = torch.randn(6, vocab, device="cuda", generator=gen(3))
    x[0] = -i * 0.001
    x[1] = i * 0.001
    x[2, 100:200] += 20
    x[3, ::256] += 20
    x[4, ::1024] += 20
    x[5, 3::64] += 20
    for top in (1, 17, 64):
        check(cbx, x, ids, top)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("vocab", [50, 8194, 33000])
def test_masked_tokens_and_empty_rows(cbx, dt, vocab):
    """Logits of -inf and of the type's lowest value; rows with one token left
    and with none."""
    rows = 6
    x = torch.randn(rows, vocab, device="cuda", generator=gen(5)).to(dt)
    x[0, ::2] = -INF
    x[1, 1:] = -INF
    x[2, 5:] = torch.finfo(dt).min
    x[3] = torch.finfo(dt).min
    x[4, :vocab - 1] = -INF
    ids = torch.tensor([1, 0, 3, 2, 0, 0], dtype=torch.int32, device="cuda")
    check(cbx, x[:5], ids[:5], min(40, vocab))
    x[5] = -INF
    logp, ent, ti, tl = cbx.token_log_probs(x, ids, top_n=3)
    assert float(logp[5]) == -INF and float(ent[5]) == 0.0 and tl[5].tolist() == [-INF] * 3 and ti[5].tolist() == [0, 1, 2]
    assert float(logp[4]) == -INF and float(logp[1]) == 0.0 and float(ent[1]) == 0.0


def test_nan_and_infinite_rows(cbx):
    x = torch.randn(4, 700, device="cuda", generator=gen(6))
    x[0, 333] = float("nan")
    x[1, 12] = INF
    x[3] = float("nan")
    ids = torch.tensor([5, 5, 5, 5], dtype=torch.int32, device="cuda")
    logp, ent, ti, tl = cbx.token_log_probs(x, ids, top_n=4)
    assert bool(torch.isnan(logp[[0, 1, 3]]).all()) and bool(torch.isnan(ent[[0, 1, 3]]).all()) and bool(torch.isnan(tl[[0, 1, 3]]).all())
    assert ti[0, 0] == 333 and ti[1, 0] == 12 and ti[3].tolist() == [0, 1, 2, 3]
    assert torch.equal(ti[2].long(), torch.argsort(x[2], descending=True, stable=True)[:4])
    assert bool(torch.isfinite(logp[2]))


def test_rows_at_a_stride_and_odd_alignment(cbx):
    base = torch.randn(9, 5005, device="cuda", generator=gen(7))
    ids = torch.randint(0, 4000, (9,), device="cuda", generator=gen(8), dtype=torch.int32)
    for a in (0, 1, 2, 3):
        check(cbx, base[:, a:a + 4001], ids, 6)
        check(cbx, base.half()[:, a:a + 4001], ids, 6)
    check(cbx, base[:1].expand(5, -1), ids[:5], 3)


def test_scales(cbx):
    x = torch.randn(20, 2000, device="cuda", generator=gen(9)) * 4
    ids = torch.randint(0, 2000, (20,), device="cuda", generator=gen(10), dtype=torch.int32)
    for scale in (0.01, 0.5, 2.0, 30.0):
        check(cbx, x, ids, 10, scale)


def test_optional_outputs_and_ids_out_of_range(cbx):
    x = torch.randn(5, 900, device="cuda", generator=gen(11))
    logp, ent, ti, tl = cbx.token_log_probs(x, top_n=2, entropy=False)
    assert logp is None and ent is None and torch.equal(ti.long(), torch.argsort(x, descending=True, stable=True)[:, :2])
    logp, ent, ti, tl = cbx.token_log_probs(x)
    assert logp is None and ti.shape == (5, 0) and bool(torch.isfinite(ent).all())
    bad = torch.tensor([0, -1, 900, 2 ** 31 - 1, 3], dtype=torch.int32, device="cuda")
    logp, _, _, _ = cbx.token_log_probs(x, bad)
    assert cbx.device_errors(clear=True) == 1
    assert logp[1:4].tolist() == [0.0, 0.0, 0.0] and bool((logp[[0, 4]] < 0).all())
    e = cbx.token_log_probs(x[:0], bad[:0], top_n=2)
    assert e[0].shape == (0,) and e[2].shape == (0, 2)


def test_captured_and_repeated(cbx):
    """Replays follow the logits, equal to the eager call bit for bit; a row
    long enough to be split as well as many short ones."""
    for rows, vocab in ((2, 120000), (600, 900)):
        x = torch.randn(rows, vocab, device="cuda", generator=gen(12))
        ids = torch.randint(0, vocab, (rows,), device="cuda", generator=gen(13), dtype=torch.int32)
        cbx.token_log_probs(x, ids, top_n=9)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = cbx.token_log_probs(x, ids, top_n=9, scale=0.9)
        for step in range(4):
            x.normal_(generator=gen(20 + step))
            graph.replay()
            eager = cbx.token_log_probs(x, ids, top_n=9, scale=0.9)
            torch.cuda.synchronize()
            for a, b in zip(got, eager):
                assert torch.equal(a, b)
            check(cbx, x, ids, 9, 0.9)
