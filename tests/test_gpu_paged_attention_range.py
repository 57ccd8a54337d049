"""paged_attention at scores of millions, at queries of a wide range, and with
one bad page at a time."""
import numpy as np
import pytest
import torch

from tests._paged import U32, assert_within, attention_ref, gen, half_step, page_tables

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16
TYPES = [(F16, F16), (F32, F16), (F32, F32)]


def ints(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


def caches(length, page, d, dt, seed, hkv=1):
    pages = -(-length // page) + 2
    tables = page_tables([length], page, -(-length // page), pages, seed).cuda()
    r = gen(seed)
    kc, vc = (torch.randn(pages, hkv, page, d, device="cuda", generator=r).to(dt) for _ in range(2))
    return kc, vc, tables


def rows_of(cache, tables, length):
    """[length, d] of the one request and its one key head."""
    return cache[tables[0].long(), 0].reshape(-1, cache.shape[-1])[:length]


@pytest.mark.parametrize("dt,cdt", TYPES)
@pytest.mark.parametrize("length,page", [(1, 16), (40, 16), (40, 24), (3000, 64), (3000, 24)])
@pytest.mark.parametrize("top", [2.0 ** 25, 1.37 * 2 ** 25, 1.9 * 2 ** 25, 1.01 * 2 ** 26, 1.71 * 2 ** 26, 1.3 * 2 ** 27, 1.99 * 2 ** 28])
def test_scores_of_millions(cbx, dt, cdt, length, page, top):
    """Scores of `top` powers of two, of both signs, in a whole and in a split
    key head.  One key ahead of all others by a thousandth (some 2^15 powers
    of two): y is its value, to the rounding of v times 1 / 1.  All keys
    alike: every score is rounded the same way, y is the mean of the values,
    off by n sums and 8 more roundings."""
    d = 64
    kc, vc, tables = caches(length, page, d, cdt, 30 + length + page)
    q = torch.zeros(1, 2, d, dtype=dt, device="cuda")
    q[..., 3] = 1024.0
    lens, v = ints([length]), rows_of(vc, tables, length).double()
    for sign in (1.0, -1.0):
        scale = sign * top / (1024.0 * 1000.0) * float(np.log(2.0))
        kc.zero_()
        kc[..., 3] = 1000.0
        y = cbx.paged_attention(q, kc, vc, tables, lens, scale).double()
        ref = v.mean(0).expand(2, d)[None]
        bound = (length + 8) * U32 * v.abs().mean(0) + half_step(dt) * ref.abs()
        assert_within(y, ref, bound, f"equal scores, sign {sign}")
        best = length // 2
        kc[..., 3] = 999.0 if sign > 0 else 1000.0
        kc[tables[0, best // page], 0, best % page, 3] = 1000.0 if sign > 0 else 999.0
        y = cbx.paged_attention(q, kc, vc, tables, lens, scale).double()
        ref = v[best].expand(2, d)[None]
        assert_within(y, ref, (2 * U32 + half_step(dt)) * ref.abs(), f"one score ahead, sign {sign}")


@pytest.mark.parametrize("cdt", [F16, F32])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 24), (60, 16)])
@pytest.mark.parametrize("large", [1.0, 1e4, 1e6, 1e8, 1e10])
def test_queries_of_a_wide_range(cbx, cdt, d, page, large):
    """An F32 query with one element `large` times the others, where the keys
    are 0 in that dim: the scores come from the small ones.  Three dims of the
    query are not 0, so a score is three products (all others are exact
    zeros): an element is held to 2^-23 of itself or 2^-51 of the largest, 3
    roundings of the products and sums, one of the scale."""
    length = 300
    kc, vc, tables = caches(length, page, d, cdt, 70 + d)
    q = torch.zeros(1, 1, d, device="cuda")
    q[..., 1], q[..., d - 2], q[..., 5] = 1.7, -2.3, 3.3 * large
    kc[..., 5] = 0
    k, v = rows_of(kc, tables, length).double(), rows_of(vc, tables, length).double()
    y = cbx.paged_attention(q, kc, vc, tables, ints([length]), 1.0)
    s = k @ q[0, 0].double()
    p = torch.softmax(s, -1)
    size = k.abs() @ q[0, 0].double().abs()
    err = (6 * U32 * size + 2.0 ** -51 * float(q.abs().max()) * k.abs().sum(-1) + 4 * U32 * s.abs().amax() + 4 * U32).amax()
    bound = (2 * err + (length + 8) * U32) * (p @ v.abs())
    assert_within(y[0, 0], p @ v, bound, f"{large}")


@pytest.mark.parametrize("cdt", [F16, F32])
@pytest.mark.parametrize("d", [64, 60])
@pytest.mark.parametrize("page", [1, 5, 8, 16, 24, 64])
def test_one_bad_page_alone(cbx, cdt, d, page):
    """Every entry of a table in its turn no page of the cache, below 0 or
    past the last: its keys are left out and bit 2 is raised, whichever keys
    of a step the page holds."""
    length = 100
    kc, vc, tables = caches(length, page, d, cdt, 90 + page, hkv=2)
    q = torch.randn(1, 4, d, device="cuda", generator=gen(91))
    cbx.device_errors(clear=True)
    for entry in range(tables.shape[1]):
        for value in (-1, kc.shape[0], 2 ** 31 - 1):
            bad = tables.clone()
            bad[0, entry] = value
            y = cbx.paged_attention(q, kc, vc, bad, ints([length]), 0.125)
            assert cbx.device_errors(clear=True) == 4, f"entry {entry} of {value}"
            ref, bound = attention_ref(q, kc, vc, bad, [length], 0.125)
            assert_within(y, ref, bound, f"entry {entry} of {value}")
            # the same entry behind the request's keys, or before its window: not looked at
            if entry > 0:
                cbx.paged_attention(q, kc, vc, bad, ints([entry * page]), 0.125)
            if (entry + 1) * page < length:
                cbx.paged_attention(q, kc, vc, bad, ints([length]), 0.125, window=length - (entry + 1) * page)
            assert cbx.device_errors(clear=True) == 0, f"entry {entry} of {value} is not used"
