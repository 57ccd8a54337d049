"""What the paged operators refuse on the host once the device is known, and
the rows that their other tests' bounds say little about."""
import pytest
import torch

from tests._paged import gen

pytestmark = pytest.mark.gpu


def test_attention_scratch_overlaps_a_tensor(cbx):
    d, page, width = 64, 64, 40
    kc = torch.zeros(width, 1, page, d, dtype=torch.float16, device="cuda")
    vc, tables = torch.zeros_like(kc), torch.arange(width, dtype=torch.int32, device="cuda")[None]
    lens, q = torch.tensor([width * page], dtype=torch.int32, device="cuda"), torch.zeros(1, 1, d, device="cuda")
    need = cbx.paged_attention_workspace(q, kc, tables)
    assert need > 0
    arena = torch.zeros(need // 4 + 64 + d, device="cuda")
    y = arena[need // 4 - 16:need // 4 - 16 + d].view(1, 1, d)
    with pytest.raises(cbx.CbxError, match="ws must not overlap"):
        cbx.paged_attention(q, kc, vc, tables, lens, 0.125, out=y, ws=arena)
    with pytest.raises(cbx.CbxError, match="ws must not overlap"):
        cbx.paged_attention(q, kc, vc, tables, lens, 0.125, ws=kc.view(-1))
    y = arena[-d:].view(1, 1, d)                   # an arena that holds more than the scratch
    assert torch.equal(cbx.paged_attention(q, kc, vc, tables, lens, 0.125, out=y, ws=arena), torch.zeros_like(y))


def test_log_prob_scratch_overlaps_a_tensor(cbx):
    x = torch.zeros(1, 40000, device="cuda")
    assert 0 < cbx.token_log_probs_workspace(x, 4) < x.numel() * 4
    with pytest.raises(cbx.CbxError, match="ws must not overlap"):
        cbx.token_log_probs(x, top_n=4, ws=x.view(-1))


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("v", [70, 8194, 40000])
def test_lowest_logits_mask_as_infinite_ones(cbx, dt, v):
    """Logits of the type's lowest value beside usual ones have p = 0 in f32 as
    those of -inf do: the other tokens' results are the same bits."""
    g = gen(31)
    x = (torch.randn(9, v, device="cuda", generator=g) * 3).to(dt)
    mask = torch.rand(9, v, device="cuda", generator=g) < 0.5
    mask[:, 5] = False
    ids = torch.full((9,), 5, dtype=torch.int32, device="cuda")
    low = cbx.token_log_probs(x.masked_fill(mask, torch.finfo(dt).min), ids, top_n=8, scale=0.7)
    inf = cbx.token_log_probs(x.masked_fill(mask, float("-inf")), ids, top_n=8, scale=0.7)
    for a, b in zip(low, inf):
        assert torch.equal(a, b) and bool(torch.isfinite(a.float()).all())


@pytest.mark.parametrize("d,page", [(128, 64), (128, 24), (60, 64)])
def test_pages_past_four_gigabytes(cbx, d, page):
    """Pages behind a 32-bit byte offset, written and read, give the bits of
    the same rows in the first pages: whole runs of 16 keys to a page, others,
    and a head size that the tiles do not take."""
    hkv, n = 2, 3
    n_pages = (1 << 32) // (hkv * page * d * 2) + 3 * n
    width = n
    kc = torch.zeros(n_pages, hkv, page, d, dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    g = gen(41)
    tok = n * page
    k, v = (torch.randn(tok, hkv, d, device="cuda", generator=g).half() for _ in range(2))
    q = torch.randn(1, 2 * hkv, d, device="cuda", generator=g).half()
    lens = torch.tensor([tok - 3], dtype=torch.int32, device="cuda")
    at = torch.arange(tok, dtype=torch.int32, device="cuda")
    out = []
    for first in (0, n_pages - n):
        cbx.paged_store(k, v, at + first * page, kc, vc)
        tables = torch.arange(first, first + width, dtype=torch.int32, device="cuda")[None]
        out.append(cbx.paged_attention(q, kc, vc, tables, lens, d ** -0.5))
        rows = kc[first:first + n].transpose(1, 2).reshape(tok, hkv, d)
        assert torch.equal(rows, k)
    assert torch.equal(out[0], out[1]) and bool(out[0].any())
    assert not bool(kc[n:n + 3].any()), "pages between stay as they were"
    assert cbx.device_errors(clear=True) == 0


def test_logits_past_four_gigabytes(cbx):
    rows, v = 140000, 8194
    x = torch.zeros(rows, v, device="cuda")
    x[-3:] = torch.randn(3, v, device="cuda", generator=gen(42))
    ids = torch.full((rows,), 11, dtype=torch.int32, device="cuda")
    got = cbx.token_log_probs(x, ids, top_n=4)
    few = cbx.token_log_probs(x[-3:].clone(), ids[-3:], top_n=4)
    for a, b in zip(got, few):
        assert torch.equal(a[-3:], b)


def test_captured_append_and_release(cbx):
    """A pair of append and release replayed as the lengths change: every
    replay as the same calls made eagerly."""
    n, page, pool, width, slots = 6, 8, 40, 9, 96
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731

    def state():
        return [ints([0] * n), ints([0] * n), ints([0] * n), ints(list(range(pool))), ints([pool]), ints([[-1] * width] * n)]

    def step(st):
        lens, new, rel, stack, left, tables = st
        ln, nf, start, sl, pos = cbx.paged_append(lens, new, stack, left, tables, page, slots)
        ln2, nf2 = cbx.paged_release(ln, rel, tables, page, stack, nf)
        lens.copy_(ln2), left.copy_(nf2)
        return start, sl, pos

    a, b = state(), state()
    keep = [t.clone() for t in b]
    step(b)
    for t, o in zip(b, keep):
        t.copy_(o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(b)
    for t, o in zip(b, keep):
        t.copy_(o)
    for new, rel in (([5, 0, 20, 1, 8, 9], [0] * n), ([1] * n, [0, 0, 1, 0, 0, 0]), ([3, 60, 1, 0, 30, 1], [1, 0, 0, 0, 0, 1]),
                     ([0] * n, [1] * n), ([16] * n, [0] * n)):
        for st in (a, b):
            st[1].copy_(ints(new)), st[2].copy_(ints(rel))
        exp = step(a)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(list(exp) + a, list(outs) + b):
            assert torch.equal(x, y)
    assert cbx.device_errors(clear=True) == 0
