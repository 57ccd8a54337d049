"""paged_release where tables hold entries that are no page, and what append
makes of malformed values: whole numbers, so everything is equal."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


def release_ref(lens, rel, tables, page, free, n_free):
    """paged_release by a loop: (lens, n_free, tables, free, raised)."""
    tables, free, raised = [list(r) for r in tables], list(free), False
    cap = len(tables[0]) * page if tables else 0
    out = []
    for s, length in enumerate(lens):
        if not rel[s]:
            out.append(length)
            continue
        out.append(0)
        if length < 0 or length > cap:
            raised = True
            continue
        for i in range(-(-length // page)):
            p, tables[s][i] = tables[s][i], -1
            if p < 0:
                raised = True
            elif n_free < len(free):
                free[n_free] = p
                n_free += 1
            else:
                raised = True
    return out, n_free, tables, free, raised


def check(cbx, lens, rel, tables, page, free, n_free):
    cbx.device_errors(clear=True)
    t, f = ints(tables), ints(free)
    out, left = cbx.paged_release(ints(lens), ints(rel), t, page, f, ints([n_free]))
    lens, n_free, tables, free, raised = release_ref(lens, rel, tables, page, free, n_free)
    assert out.tolist() == lens and left.tolist() == [n_free]
    assert t.tolist() == tables, "tables"
    assert f.tolist() == free, "stack"
    assert cbx.device_errors(clear=True) == (4 if raised else 0)
    return out, left, t, f


@pytest.mark.parametrize("n,page,width", [(1, 1, 1), (1, 16, 200), (3, 7, 63), (64, 64, 32), (65, 16, 64), (257, 5, 65), (1000, 16, 129),
                                          (4096, 8, 4)])
@pytest.mark.parametrize("gone", [0.0, 0.02, 0.5, 1.0])
def test_entries_that_are_no_page(cbx, n, page, width, gone):
    """Left out, the others pushed without holes, in the order of the requests
    and of their tables; lengths outside the table leave their rows alone."""
    rng = np.random.RandomState(n + width)
    tables = rng.permutation(n * width).reshape(n, width).astype(np.int32)
    tables[rng.rand(n, width) < gone] = -1
    tables[rng.rand(n, width) < gone / 4] = -7
    lens = rng.randint(0, page * width + 1, n)
    lens[rng.rand(n) < gone / 10] = -1
    lens[rng.rand(n) < gone / 10] = page * width + 1
    rel = rng.randint(0, 2, n)
    rel[n // 2] = 1
    for room in (n * width, n * width // 4):
        free = np.full(room + 5, -9)
        check(cbx, lens.tolist(), rel.tolist(), tables.tolist(), page, free.tolist(), 5)


def test_released_twice(cbx):
    """A request released again under its old length gives nothing back: the
    stack stays as it is, bit 2 is raised, and the next append gets pages."""
    lens, rel, page = [40, 17, 64], [1, 0, 1], 16
    tables = [[3, 1, 4, -1], [5, 9, -1, -1], [2, 6, 8, 7]]
    free = [0] + [-1] * 11
    _, left, t, f = check(cbx, lens, rel, tables, page, free, 1)
    assert left.tolist() == [8]
    _, again, t, f = check(cbx, lens, rel, t.tolist(), page, f.tolist(), 8)
    assert again.tolist() == [8]
    got = cbx.paged_append(ints([0, 17, 0]), ints([20, 0, 1]), f, again, t, page, 21)
    assert cbx.device_errors(clear=True) == 0
    assert got[0].tolist() == [20, 17, 1] and got[1].tolist() == [5] and min(got[3].tolist()) >= 0
    assert t[:, :2].tolist() == [[7, 8], [5, 9], [6, -1]]


def test_no_requests_empty_tables_and_strided_ones(cbx):
    cbx.device_errors(clear=True)
    out, left = cbx.paged_release(ints([]), ints([]), ints(np.zeros((0, 3))), 16, ints([4, 2]), ints([2]))
    assert out.tolist() == [] and left.tolist() == [2]
    out, left = cbx.paged_release(ints([0, 0]), ints([1, 0]), ints(np.zeros((2, 0))), 16, ints([4, 2]), ints([1]))
    assert out.tolist() == [0, 0] and left.tolist() == [1]
    wide = torch.full((3, 9), 77, dtype=torch.int32, device="cuda")
    view = wide[:, 2:6]
    view.copy_(ints([[3, -1, 5, 6], [7, 8, 9, -1], [1, 2, 0, 4]]))
    stack = ints([-9] * 12)
    _, left = cbx.paged_release(ints([9, 5, 16]), ints([1, 0, 1]), view, 4, stack, ints([0]))
    assert cbx.device_errors(clear=True) == 4
    assert left.tolist() == [6] and stack.tolist() == [3, 5, 1, 2, 0, 4] + [-9] * 6
    assert view.tolist() == [[-1, -1, -1, 6], [7, 8, 9, -1], [-1] * 4]
    assert bool((wide[:, :2] == 77).all()) and bool((wide[:, 6:] == 77).all())


def test_two_streams_at_once(cbx):
    """Releases of two pools without order between them: each as if alone."""
    rng = np.random.RandomState(9)
    n, page, width = 300, 4, 70
    sets = []
    for _ in range(2):
        a = [rng.randint(0, page * width + 1, n).tolist(), rng.randint(0, 2, n).tolist(),
             np.where(rng.rand(n, width) < 0.1, -1, rng.permutation(n * width).reshape(n, width)).tolist()]
        sets.append((a, release_ref(*a, page, [-1] * n * width, 0)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    runs = [[[ints(x) for x in a] + [ints([-1] * n * width), ints([0])] for _ in range(10)] for a, _ in sets]
    torch.cuda.synchronize()
    outs = [[], []]
    for j in range(10):
        for i in range(2):
            lens, rel, tables, stack, count = runs[i][j]
            with torch.cuda.stream(streams[i]):
                outs[i].append(cbx.paged_release(lens, rel, tables, page, stack, count))
    torch.cuda.synchronize()
    for i in range(2):
        lens, n_free, tables, free, _ = sets[i][1]
        for (out, left), run in zip(outs[i], runs[i]):
            assert [out.tolist(), left.tolist(), run[2].tolist(), run[3].tolist()] == [lens, [n_free], tables, free]
    cbx.device_errors(clear=True)


def test_captured_release(cbx):
    """Replayed as lengths and tables change, with eager calls between."""
    n, page, width = 9, 4, 12
    lens, rel, tables, stack, count = ints([0] * n), ints([0] * n), ints(np.zeros((n, width))), ints([-1] * n * width), ints([3])
    cbx.paged_release(lens, rel, tables, page, stack, count)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, left = cbx.paged_release(lens, rel, tables, page, stack, count)
    rng = np.random.RandomState(4)
    for step in range(5):
        a = [rng.randint(0, page * width + 1, n).tolist(), rng.randint(0, 2, n).tolist(),
             np.where(rng.rand(n, width) < 0.2, -1, rng.permutation(n * width).reshape(n, width)).tolist()]
        free = [-1] * n * width
        for t, x in zip((lens, rel, tables, stack), a + [free]):
            t.copy_(ints(x))
        graph.replay()
        torch.cuda.synchronize()
        exp = release_ref(*a, page, free, 3)
        assert [out.tolist(), left.tolist(), tables.tolist(), stack.tolist()] == [exp[0], [exp[1]], exp[2], exp[3]], f"step {step}"
        check(cbx, *a, page, free, 3)
        cbx.device_errors(clear=True)


def test_append_beside_malformed_requests(cbx):
    """A request that needs no page is granted beside others that are
    malformed and a stack count that is none."""
    cbx.device_errors(clear=True)
    t = ints([[-1, -1], [0, -1], [1, -1], [-1, -1]])
    got = cbx.paged_append(ints([-3, 5, 100, 2]), ints([1, -1, 1, 1]), ints([9, 8]), ints([5]), t, 4, 4)
    assert cbx.device_errors(clear=True) == 4
    assert [g.tolist() for g in got] == [[-3, 5, 100, 3], [2], [0, 1, 1, 2, 3], [-1, -1, -1, -1], [-3, 100, 2, 0]]
    assert t.tolist() == [[-1, -1], [0, -1], [1, -1], [-1, -1]]


def test_append_from_a_stack_with_entries_that_are_no_page(cbx):
    """They are handed out in their turn: noted in the table, their tokens'
    slots -1, bit 2; the other pages' tokens have theirs."""
    cbx.device_errors(clear=True)
    t = ints([[-1, -1], [-1, -1]])
    got = cbx.paged_append(ints([0, 0]), ints([5, 2]), ints([6, -4, 2]), ints([3]), t, 4, 7)
    assert cbx.device_errors(clear=True) == 4
    assert [g.tolist() for g in got] == [[5, 2], [0], [0, 5, 7], [8, 9, 10, 11, -1, 24, 25], [0, 1, 2, 3, 4, 0, 1]]
    assert t.tolist() == [[2, -4], [6, -1]]
