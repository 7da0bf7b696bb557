"""The paged cache's calls on the device against the same calls in plain Python (pages_ref.py).  Nothing is
computed, so every number has to be equal."""
import random

import numpy as np
import pytest

from whisper4j_b200._lib import IllegalStateError

from .pages_ref import PagesRef

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def new_cache(n_layer=2, n_kv=3, dim=64, n_pages=40, page=16, n_rows=8, max_tokens=100, dtype=torch.float16, seed=0):
    from whisper4j_b200 import ops
    c = ops.PagedCache(n_layer, n_kv, dim, n_pages, page, n_rows, max_tokens, dtype=dtype)
    g = torch.Generator("cuda").manual_seed(seed)
    c.pool.copy_(torch.randn(c.pool.shape, device="cuda", generator=g))
    c.table.fill_(-7)  # entries behind a row's length are neither read nor written
    return c, mirror(c)


def host(c):
    torch.cuda.synchronize()
    return (c.pool.view(torch.int16).cpu().numpy(), c.ref.cpu().numpy(), c.table.cpu().numpy(), c.len.cpu().numpy())


def mirror(c):
    return PagesRef(*host(c))


def same(c, m):
    pool, ref, table, length = host(c)
    np.testing.assert_array_equal(length, m.len)
    np.testing.assert_array_equal(table, m.table)
    np.testing.assert_array_equal(ref, m.ref)
    np.testing.assert_array_equal(pool, m.pool)
    c.check()


def starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def grow(c, m, rows, counts, seed=1):
    start = starts(counts)
    c.extend(ints(rows), ints(start))
    m.extend(rows, start)
    g = torch.Generator("cuda").manual_seed(seed)
    for layer in range(c.n_layer):
        kv = torch.randn(2, start[-1], c.n_kv_head, c.head_dim, device="cuda", generator=g).to(c.pool.dtype)
        c.write(layer, ints(rows), ints(start), kv[0], kv[1])
        k, v = kv.view(torch.int16).cpu().numpy()
        m.write(layer, rows, start, k, v)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page,dim,n_kv", [(16, 64, 3), (8, 128, 1), (24, 64, 5), (128, 64, 2)])
def test_grow_and_write(page, dim, n_kv, dtype):
    c, m = new_cache(page=page, dim=dim, n_kv=n_kv, dtype=dtype, max_tokens=4 * page, n_pages=90)
    grow(c, m, [3, 0, 5], [1, page, 2 * page + 3])
    same(c, m)
    grow(c, m, [5, 3, 7, 0], [1, page - 1, 0, 7])  # into a page, up to its end, nothing, over a border
    same(c, m)
    grow(c, m, list(range(8)), [1] * 8)  # one token each: a decode step
    same(c, m)


@pytest.mark.parametrize("lens", [(20, 33), (16, 48), (5, 0)])
@pytest.mark.parametrize("dst,src", [([2], [0]), ([2, 3, 4], [0, 0, 0]), ([0], [0]), ([0, 1], [1, 0]), ([0, 1, 2], [1, 1, 1]),
                                     ([0, 1], [0, 0]), ([1, 0, 2], [0, 0, 1]), ([0], [-1]), ([0, 4, 5], [-1, 0, 0]),
                                     ([6, 0], [7, 6])])
def test_fork(lens, dst, src):
    c, m = new_cache()
    grow(c, m, [0, 1], list(lens))
    c.fork(ints(dst), ints(src))
    m.fork(dst, src)
    same(c, m)
    grow(c, m, [0, 1, 2], [1, 2, 3], seed=5)  # what the forked rows write stays their own
    same(c, m)


@pytest.mark.parametrize("n_rows,max_tokens,n_pages", [(300, 120, 2500), (5000, 16, 9000), (40, 4000, 3000)])
def test_fork_of_many_rows(n_rows, max_tokens, n_pages):
    """Sizes that the whole cluster takes: many rows, long tables, a long free list."""
    rnd = random.Random(n_rows)
    c, m = new_cache(n_layer=1, n_kv=1, n_pages=n_pages, n_rows=n_rows, max_tokens=max_tokens, page=8)
    some = rnd.sample(range(n_rows), n_rows // 4)
    grow(c, m, some, [rnd.randint(1, max_tokens // 4) for _ in some])
    for turn in range(3):
        dst = rnd.sample(range(n_rows), n_rows // 2)
        src = [rnd.choice(some + [-1]) for _ in dst]
        c.fork(ints(dst), ints(src))
        m.fork(dst, src)
        same(c, m)


def test_free_and_compact():
    c, m = new_cache()
    grow(c, m, [0, 1, 2, 3], [40, 17, 33, 5])
    c.fork(ints([4, 5]), ints([2, 2]))
    m.fork([4, 5], [2, 2])
    c.free(ints([0, 2]))
    m.free([0, 2])
    same(c, m)
    live = c.compact()
    assert int(live) == m.compact()
    same(c, m)
    assert int(c.compact()) == m.compact()  # nothing is left to move
    same(c, m)
    grow(c, m, [0, 6], [50, 16])
    same(c, m)
    c.free(ints(list(range(8))))
    m.free(list(range(8)))
    assert int(c.compact()) == 0
    same(c, m)


@pytest.mark.parametrize("n_rows,n_pages", [(64, 1000), (700, 12000)])
def test_turnover_at_random(n_rows, n_pages):
    rnd = random.Random(n_pages)
    c, m = new_cache(n_layer=1, n_kv=2, n_pages=n_pages, n_rows=n_rows, max_tokens=200, page=16)
    for turn in range(6):
        rows = rnd.sample(range(n_rows), n_rows // 3)
        c.free(ints(rows))
        m.free(rows)
        if turn % 2:
            assert int(c.compact()) == m.compact()
        grow(c, m, rows, [rnd.randint(0, 150) for _ in rows], seed=turn)
        dst = rnd.sample(range(n_rows), n_rows // 5)
        src = [rnd.randrange(-1, n_rows) for _ in dst]
        c.fork(ints(dst), ints(src))
        m.fork(dst, src)
        same(c, m)


def refused(c, m, text, call):
    call()
    with pytest.raises(IllegalStateError, match=text):
        c.check()
    same(c, m)  # nothing has changed, and the next call goes on


@pytest.mark.parametrize("n_rows", [8, 5000, 30000])
def test_calls_that_cannot_be_done_change_nothing(n_rows):
    c, m = new_cache(n_rows=n_rows, n_pages=10)
    grow(c, m, [0, 1], [70, 20])  # 5 + 2 pages of 10
    s = [0, 1]
    refused(c, m, "free pages", lambda: c.extend(ints([2]), ints([0, 49])))
    refused(c, m, "free pages", lambda: c.extend(ints([2, 3]), ints([0, 33, 49])))
    refused(c, m, "outgrow", lambda: c.extend(ints([0]), ints([0, 100])))
    refused(c, m, "outgrow", lambda: c.extend(ints([0]), ints([0, 2 ** 31 - 1])))
    refused(c, m, "twice", lambda: c.extend(ints([2, 2]), ints([0, 1, 2])))
    refused(c, m, "out of range", lambda: c.extend(ints([n_rows]), ints(s)))
    refused(c, m, "out of range", lambda: c.extend(ints([-1]), ints(s)))
    refused(c, m, "ascend", lambda: c.extend(ints([2]), ints([1, 2])))
    refused(c, m, "ascend", lambda: c.extend(ints([2, 3]), ints([0, 2, 1])))
    refused(c, m, "free pages", lambda: c.fork(ints([2, 3, 4, 5]), ints([0, 0, 1, 1])))
    refused(c, m, "twice", lambda: c.fork(ints([2, 2]), ints([0, 1])))
    refused(c, m, "out of range", lambda: c.fork(ints([2]), ints([n_rows])))
    refused(c, m, "out of range", lambda: c.fork(ints([2]), ints([-2])))
    refused(c, m, "out of range", lambda: c.fork(ints([-1]), ints([0])))
    refused(c, m, "twice", lambda: c.free(ints([1, 0, 1])))
    refused(c, m, "out of range", lambda: c.free(ints([n_rows])))
    c.fork(ints([2, 3, 4]), ints([0, 0, 1]))  # exactly the free pages
    m.fork([2, 3, 4], [0, 0, 1])
    same(c, m)
    c.table[1, 1], m.table[1, 1] = 10, 10  # a page that is not there
    for call in (lambda: c.free(ints([1])), lambda: c.fork(ints([5]), ints([1])), lambda: c.fork(ints([1]), ints([-1])),
                 lambda: c.compact(),
                 lambda: c.write(0, ints([1]), ints(s), *torch.zeros(2, 1, 3, 64, dtype=torch.float16, device="cuda"))):
        refused(c, m, "page", call)


@pytest.mark.parametrize("n", [40, 100, 1000])
def test_forks_of_many_rows_that_cannot_be_done(n):
    """A fault in any one row, late or early, leaves all rows as they were."""
    c, m = new_cache(n_layer=1, n_kv=1, n_rows=2 * n, n_pages=4 * n, max_tokens=64)
    grow(c, m, list(range(n)), [30 + i % 3 for i in range(n)])  # 2 pages each; 32 is whole, 30 and 31 are not
    dst, src = list(range(n, 2 * n)), list(range(n))
    for at in (0, n // 2, n - 1):
        for value in (2 * n, -2):
            refused(c, m, "out of range", lambda: c.fork(ints(dst), ints(src[:at] + [value] + src[at + 1:])))
        refused(c, m, "out of range", lambda: c.fork(ints(dst[:at] + [2 * n] + dst[at + 1:]), ints(src)))
        old = int(m.table[at, 1])
        c.table[at, 1] = m.table[at, 1] = 4 * n
        refused(c, m, "page", lambda: c.fork(ints(dst), ints(src)))
        c.table[at, 1] = m.table[at, 1] = old
    refused(c, m, "twice", lambda: c.fork(ints(dst[:-1] + dst[:1]), ints(src)))
    c.fork(ints(dst), ints(src))  # a row of its own for each: full pages shared, the last one stays with the source
    m.fork(dst, src)
    grow(c, m, dst, [1] * n)
    same(c, m)
    grow(c, m, [0], [20])  # n - 2 pages are left, and n rows want one
    refused(c, m, "free pages", lambda: c.fork(ints(dst), ints([0] * n)))
    c.fork(ints(dst[2:]), ints([0] * (n - 2)))
    m.fork(dst[2:], [0] * (n - 2))
    same(c, m)


def test_write_leaves_out_what_has_no_place():
    c, m = new_cache()
    grow(c, m, [0, 1], [3, 4])
    kv = torch.ones(2, 6, 3, 64, dtype=torch.float16, device="cuda")
    refused(c, m, "out of range", lambda: c.write(0, ints([8]), ints([0, 6]), kv[0], kv[1]))
    # more tokens than start deals out: those behind the last row are left out, and reported
    c.write(1, ints([0, 1]), ints([0, 2, 5]), kv[0], kv[1])
    m.write(1, [0, 1], [0, 2, 5], *kv.view(torch.int16).cpu().numpy())
    with pytest.raises(IllegalStateError, match="ascend"):
        c.check()
    same(c, m)
    c.write(0, ints([0]), ints([0, 6]), kv[0], kv[1])  # the row holds 3 tokens: the first 3 have no place
    m.write(0, [0], [0, 3], *kv[:, 3:].view(torch.int16).cpu().numpy())
    with pytest.raises(IllegalStateError, match="fit the rows"):
        c.check()
    same(c, m)


def test_write_from_a_fused_projection():
    c, m = new_cache()
    qkv = torch.randn(7, 5 * 64 + 2 * 3 * 64, device="cuda").half()
    k, v = qkv[:, 320:512].view(7, 3, 64), qkv[:, 512:].view(7, 3, 64)
    rows, start = [2, 6, 1], [0, 3, 3, 7]
    c.extend(ints(rows), ints(start))
    m.extend(rows, start)
    c.write(1, ints(rows), ints(start), k, v)
    m.write(1, rows, start, k.contiguous().view(torch.int16).cpu().numpy(), v.contiguous().view(torch.int16).cpu().numpy())
    same(c, m)
    with pytest.raises(ValueError):
        c.write(1, ints(rows), ints(start), k.float(), v)
    with pytest.raises(ValueError):
        c.write(1, ints(rows), ints(start), k.transpose(0, 1), v)
    with pytest.raises(ValueError):
        c.extend(ints(rows), ints(start[:-1]))
    with pytest.raises(ValueError):
        c.free(ints(rows).long())


def test_captured_and_replayed():
    """A decode step's extend, write and reorder in a graph, replayed with other rows and tokens in its inputs."""
    c, m = new_cache(n_pages=64)
    grow(c, m, [0, 1, 2], [30, 15, 16])
    rows, start, dst, src = ints([0, 1, 2]), ints([0, 1, 2, 3]), ints([0, 1, 2]), ints([0, 0, 2])
    kv = torch.zeros(2, 3, 3, 64, dtype=torch.float16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.extend(rows, start)
        c.write(0, rows, start, kv[0], kv[1])
        c.fork(dst, src)
    same(c, m)  # captured, not run
    for order in ([0, 0, 2], [1, 0, 1], [2, 1, 0], [0, 1, 2]):
        kv.normal_()
        src.copy_(ints(order))
        graph.replay()
        m.extend([0, 1, 2], [0, 1, 2, 3])
        m.write(0, [0, 1, 2], [0, 1, 2, 3], *kv.view(torch.int16).cpu().numpy())
        m.fork([0, 1, 2], order)
        same(c, m)


def test_on_a_stream_of_its_own():
    c, m = new_cache()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grow(c, m, [0, 1], [25, 60])
        c.fork(ints([3]), ints([1]))
    torch.cuda.current_stream().wait_stream(side)
    m.fork([3], [1])
    same(c, m)


def tokens(c, n, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(2, n, c.n_kv_head, c.head_dim, device="cuda", generator=g).to(c.pool.dtype)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("n_rows", [8, 30000])  # planned by one block, and by a cluster
def test_writes_behind_a_refused_extension_change_nothing(n_rows, captured):
    """Rows whose last page is full and shared: the tokens of an extension that finds no page would land on it."""
    c, m = new_cache(n_pages=8, n_rows=n_rows)
    grow(c, m, [0, 6], [48, 33])  # 3 + 3 pages, 2 free
    c.fork(ints([1, 2]), ints([0, 0]))
    m.fork([1, 2], [0, 0])
    rows, start, kv = ints([0, 1, 2]), ints([0, 1, 2, 3]), tokens(c, 3, 5)

    def step():
        c.extend(rows, start)
        for layer in range(c.n_layer):
            c.write(layer, rows, start, kv[0], kv[1])

    run = step
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        run = graph.replay
    for _ in range(2):
        refused(c, m, "free pages", run)  # three rows want a page each
    refused(c, m, "free pages", lambda: c.write(0, rows, start, kv[0], kv[1]))  # also behind a status that was read
    grow(c, m, [6], [2])  # another row goes on
    c.extend(ints([1]), ints([0, 1]))  # and one of the three
    m.extend([1], [0, 1])
    more = tokens(c, 1, 6)
    for layer in range(c.n_layer):
        c.write(layer, ints([1]), ints([0, 1]), more[0], more[1])
        m.write(layer, [1], [0, 1], *more.view(torch.int16).cpu().numpy())
    same(c, m)
    c.free(ints([6]))
    m.free([6])
    run()  # there is room now
    m.extend([0, 1, 2], [0, 1, 2, 3])
    for layer in range(c.n_layer):
        m.write(layer, [0, 1, 2], [0, 1, 2, 3], *kv.view(torch.int16).cpu().numpy())
    same(c, m)


@pytest.mark.parametrize("n_rows", [8, 30000])
@pytest.mark.parametrize("rows,counts,text", [([0, 1], [1, 65], "outgrow"), ([0, 0], [1, 1], "twice"), ([0, -1], [1, 1], "out of range"),
                                              ([1, 0], [3, -1], "ascend")])
def test_writes_behind_any_refusal(n_rows, rows, counts, text):
    c, m = new_cache(n_rows=n_rows)
    grow(c, m, [0, 1], [20, 48])
    start = starts(counts)
    kv = tokens(c, max(start), 3)

    def step():
        c.extend(ints(rows), ints(start))
        c.write(1, ints(rows), ints(start), kv[0], kv[1])

    refused(c, m, text, step)
    grow(c, m, [0, 1], [2, 3])
    same(c, m)


@pytest.mark.parametrize("n", [3, 40, 700, 5000])
def test_writes_that_name_a_row_twice(n):
    """Two tokens would have one place: the row takes those at the index of its last extension, if any."""
    c, m = new_cache(n_layer=1, n_kv=1, n_rows=6000, n_pages=6100, max_tokens=32)
    rows, start = list(range(n)), starts([1 + i % 2 for i in range(n)])
    grow(c, m, rows, [3] * n)
    kv = tokens(c, start[-1], 7)
    for move in (0, 1):  # at their extension's indexes, and all of them at others
        for i, j in ((0, n - 1), (n - 1, 0), (n // 2, n // 2 + 1)):
            order = rows[move:] + rows[:move]
            order[j] = order[i]
            c.write(0, ints(order), ints(start), kv[0], kv[1])
            k, v = kv.view(torch.int16).cpu().numpy()
            for x in range(n):
                if order.count(order[x]) == 1 or x == order[x]:
                    m.write(0, [order[x]], [0, start[x + 1] - start[x]], k[start[x]:start[x + 1]], v[start[x]:start[x + 1]])
            with pytest.raises(IllegalStateError, match="twice"):
                c.check()
            same(c, m)
            kv += 1
    order = rows[1:] + rows[:1]
    c.write(0, ints(order), ints(start), kv[0], kv[1])
    m.write(0, order, start, *kv.view(torch.int16).cpu().numpy())
    same(c, m)


@pytest.mark.parametrize("n", [4, 500, 5000])
def test_writes_whose_start_descends_are_reported(n):
    """Both ends are right; the rows behind the fault get their tokens, the row that it deals none stays as it was."""
    c, m = new_cache(n_layer=1, n_kv=1, n_rows=6000, n_pages=6100, max_tokens=32)
    grow(c, m, list(range(n)), [9] * n)
    for at in sorted({0, n // 2, n - 3}):
        start = starts([2] * n)
        start[at + 1], start[at + 2] = start[at + 2] + 1, start[at + 1] + 1
        kv = tokens(c, start[-1], 7)
        c.write(0, ints(list(range(n))), ints(start), kv[0], kv[1])
        with pytest.raises(IllegalStateError, match="ascend"):
            c.check()
        k, v = kv.view(torch.int16).cpu().numpy()
        others = [x for x in range(n) if not at <= x <= at + 2]
        for x in others:
            m.write(0, [x], [0, 2], k[2 * x:2 * x + 2], v[2 * x:2 * x + 2])
        pool = c.pool.view(torch.int16).cpu().numpy()
        pages = [m.held(x)[0] for x in others + [at + 1]]
        np.testing.assert_array_equal(pool[:, pages], m.pool[:, pages])
        m.pool[:] = pool


@pytest.mark.parametrize("n_rows", [8, 400, 30000])  # one block, a cluster of blocks for a fork, the cluster's passes
def test_rows_whose_pages_nobody_holds(n_rows):
    """Such a page would be dealt out while the row reads it, or its count fall below none."""
    c, m = new_cache(n_rows=n_rows, n_layer=1, n_kv=1, n_pages=900)
    grow(c, m, [0, 1], [70, 20])
    many = list(range(2, min(n_rows, 102)))
    page = int(m.table[0, 2])
    c.ref[page] = m.ref[page] = 0
    for call in (lambda: c.free(ints([1, 0])), lambda: c.fork(ints([2]), ints([0])), lambda: c.fork(ints([0]), ints([1])),
                 lambda: c.fork(ints(many), ints([1] * (len(many) - 1) + [0])), lambda: c.compact()):
        refused(c, m, "page", call)
    c.free(ints([1]))  # a row that has all of its pages
    m.free([1])
    same(c, m)
