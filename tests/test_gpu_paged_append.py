"""paged_append / paged_release / paged_store against loops over the requests:
whole numbers and copies, so everything is equal."""
import numpy as np
import pytest
import torch

from tests._paged import append_ref, page_tables

pytestmark = pytest.mark.gpu


def ints(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


def setup(n, page, max_past, max_new, seed, room=None, width=None):
    rng = np.random.RandomState(seed)
    past = rng.randint(0, max_past + 1, n)
    new = rng.randint(0, max_new + 1, n)
    have = -(-past // page)
    need = int((-(-(past + new) // page) - have).sum())
    room = need + 3 if room is None else room
    width = -(-(max_past + max_new) // page) if width is None else width
    total = int(have.sum()) + room
    order = rng.permutation(total)
    tables = np.full((n, max(1, width)), -1, dtype=np.int32)
    at = 0
    for s in range(n):
        tables[s, :have[s]] = order[at:at + have[s]]
        at += have[s]
    free = np.full(total, -7, dtype=np.int32)
    free[:room] = order[at:]
    return past, new, free, room, tables


def check(cbx, past, new, free, n_free, tables, page, n_slots):
    t = ints(tables)
    got = cbx.paged_append(ints(past), ints(new), ints(free), ints([n_free]), t, page, n_slots)
    lens, left, start, slots, pos, tab = append_ref(past.tolist(), new.tolist(), free.tolist(), n_free, tables.tolist(), page,
                                                    n_slots)
    exp = (lens, [left], start, slots, pos)
    for name, g, e in zip(("lens", "n_free", "start", "slots", "positions"), got, exp):
        assert g.tolist() == list(e), name
    assert t.tolist() == tab, "tables"
    return got, t


@pytest.mark.parametrize("n,page,max_past,max_new", [(1, 1, 0, 1), (1, 16, 5, 0), (3, 7, 20, 30), (64, 64, 1900, 1), (255, 16, 40, 3),
                                                     (256, 5, 9, 9), (257, 16, 100, 40), (1000, 32, 300, 2), (4096, 8, 20, 1)])
def test_lengths_and_pages(cbx, n, page, max_past, max_new):
    past, new, free, n_free, tables = setup(n, page, max_past, max_new, 10 + n)
    check(cbx, past, new, free, n_free, tables, page, int(new.sum()) + 5)


@pytest.mark.parametrize("room", [0, 1, 7, 40])
def test_pool_runs_out(cbx, room):
    """Requests are served in order until the stack is short; those that need
    no page go on, and the stack below is untouched."""
    past, new, free, n_free, tables = setup(90, 4, 30, 6, 77, room=room)
    got, _ = check(cbx, past, new, free, n_free, tables, 4, int(new.sum()))
    assert int(got[1]) >= 0


def test_table_and_slots_too_small(cbx):
    """A request past its table row is refused and takes no page from those
    behind it; so is one whose tokens do not all fit in the slots."""
    past, new, free, n_free, tables = setup(40, 8, 30, 20, 5, width=4)
    check(cbx, past, new, free, n_free, tables, 8, int(new.sum()))
    past, new, free, n_free, tables = setup(40, 8, 30, 20, 6)
    check(cbx, past, new, free, n_free, tables, 8, int(new.sum()) - 30)
    check(cbx, past, new, free, n_free, tables, 8, 0)


def test_no_requests_and_strided_tables(cbx):
    got = cbx.paged_append(ints([]), ints([]), ints([4, 2]), ints([2]), ints(np.zeros((0, 3))), 16, 6)
    assert got[1].tolist() == [2] and got[2].tolist() == [0] and got[3].tolist() == [-1] * 6 and got[4].tolist() == [0] * 6
    past, new, free, n_free, tables = setup(20, 4, 17, 5, 8)
    wide = torch.full((20, tables.shape[1] + 9), -5, dtype=torch.int32, device="cuda")
    view = wide[:, 3:3 + tables.shape[1]]
    view.copy_(ints(tables))
    cbx.paged_append(ints(past), ints(new), ints(free), ints([n_free]), view, 4, 70)
    exp = append_ref(past.tolist(), new.tolist(), free.tolist(), n_free, tables.tolist(), 4, 70)[5]
    assert view.tolist() == exp
    assert bool((wide[:, :3] == -5).all()) and bool((wide[:, 3 + tables.shape[1]:] == -5).all())


def test_malformed_values_raise_the_bit(cbx):
    """Lengths outside the table, a stack count outside the stack, a page
    that is none: left out, bit 2 of the device word."""
    cbx.device_errors(clear=True)
    past, new = ints([-3, 5, 100, 2]), ints([1, -1, 1, 1])
    t = ints([[-1, -1], [0, -1], [1, -1], [-1, -1]])
    lens, left, start, slots, pos = cbx.paged_append(past, new, ints([9, 8]), ints([5]), t, 4, 4)
    assert cbx.device_errors(clear=True) == 4
    assert lens.tolist() == [-3, 5, 100, 2] or lens.tolist() == [-3, 5, 100, 3]
    assert start.tolist() == [0, 1, 1, 2, 3]
    assert slots.tolist()[:2] == [-1, -1] and slots.tolist()[3] == -1
    assert slots.tolist()[2] == -1                       # its page in the table is -1
    lens, left = cbx.paged_release(ints([9, -1]), ints([1, 1]), ints([[0, 1], [2, 3]]), 4, ints([0, 0, 0]), ints([1]))
    assert cbx.device_errors(clear=True) == 4 and lens.tolist() == [0, 0] and left.tolist() == [1]


def test_release_then_append_takes_the_pages_again(cbx):
    """Pages given back are on top of the stack in order, their entries -1;
    the next append takes them from the top."""
    rng = np.random.RandomState(3)
    n, page, width = 50, 8, 6
    lens = rng.randint(0, page * width + 1, n)
    rel = rng.randint(0, 2, n)
    total = int((-(-lens // page)).sum()) + 9
    tables = page_tables(lens.tolist(), page, width, total, 4).cuda()
    used = set(tables[tables >= 0].tolist())
    rest = [p for p in range(total) if p not in used]
    stack = torch.full((total,), -1, dtype=torch.int32, device="cuda")
    stack[:len(rest)] = ints(rest)
    exp = list(rest)
    for s in range(n):
        if rel[s]:
            exp += tables[s, :-(-lens[s] // page)].tolist()
    before = tables.clone()
    out, left = cbx.paged_release(ints(lens), ints(rel), tables, page, stack, ints([len(rest)]))
    assert left.tolist() == [len(exp)] and stack[:len(exp)].tolist() == exp
    assert out.tolist() == [0 if rel[s] else int(lens[s]) for s in range(n)]
    for s in range(n):
        k = -(-lens[s] // page)
        assert tables[s].tolist() == ([-1] * k + before[s, k:].tolist() if rel[s] else before[s].tolist())
    new = np.where(rel, 3, 0)
    got = cbx.paged_append(out, ints(new), stack, left, tables, page, int(new.sum()))
    assert got[1].tolist() == [len(exp) - int((rel > 0).sum())]
    first = [s for s in range(n) if rel[s]][0]
    assert tables[first, 0].item() == exp[-1]
    assert cbx.device_errors(clear=True) == 0
    # more pages than the stack has room for: dropped, with the bit
    small = torch.zeros(2, dtype=torch.int32, device="cuda")
    _, left = cbx.paged_release(ints([24]), ints([1]), ints([[5, 6, 7]]), 8, small, ints([1]))
    assert small.tolist() == [0, 5] and left.tolist() == [2] and cbx.device_errors(clear=True) == 4


@pytest.mark.parametrize("dt,cdt", [(torch.float32, torch.float16), (torch.float16, torch.float16), (torch.float16, torch.float32),
                                    (torch.float32, torch.float32)])
@pytest.mark.parametrize("d,page,order", [(64, 16, "pages"), (40, 7, "tokens"), (129, 3, "pages")])
def test_store(cbx, dt, cdt, d, page, order):
    """Rows of strided k and v to distinct slots, padding skipped, every other
    element of the cache as it was; both page orders; any head size."""
    tok, hkv, pages = 37, 3, 20
    rows = torch.randn(tok, 2 * hkv * d + 5, device="cuda").to(dt)
    k, v = rows[:, :hkv * d].unflatten(1, (hkv, d)), rows[:, hkv * d:2 * hkv * d].unflatten(1, (hkv, d))
    make = (lambda: torch.randn(pages, hkv, page, d, device="cuda").to(cdt)) if order == "pages" else \
        (lambda: torch.randn(pages, page, hkv, d, device="cuda").to(cdt).transpose(1, 2))
    kc, vc = make(), make()
    slots = torch.randperm(pages * page, device="cuda")[:tok].to(torch.int32)
    slots[5] = slots[36] = -1
    ek, ev = kc.clone(), vc.clone()
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            ek[s // page, :, s % page], ev[s // page, :, s % page] = k[t].to(cdt), v[t].to(cdt)
    cbx.paged_store(k, v, slots, kc, vc)
    assert torch.equal(kc, ek) and torch.equal(vc, ev)
    assert cbx.device_errors(clear=True) == 0
    slots[0] = pages * page                              # one past the last slot
    cbx.paged_store(k, v, slots, kc, vc)
    assert cbx.device_errors(clear=True) == 4
    assert torch.equal(kc, ek) and torch.equal(vc, ev)
