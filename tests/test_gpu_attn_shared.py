"""Shared-prefix attention over a paged cache against softmax(scale q K^T) V in 64 bits, row by row.

Tolerance of one output element, from the formats alone.  With u = half a step of the cache's type
(torch.finfo(t).eps / 2), A = sum p |v| / sum p the magnitude the weighted sum runs over:
  * the weights are rounded to the type before they meet the values: u A; weights below the type's normal range
    are rounded by half its smallest step t0 against a largest weight of at least 2^-0 in its part: n t0 / 2 max|v| / l,
    with l >= 1 the sum of weights relative to the largest;
  * scores are products exact in 32 bits, summed in 32 bits: an error of (D + 8) 2^-24 scale sum |q k| <= (D + 8) 2^-24 S,
    S the largest such sum, plus 2 2^-23 |exponent| for base-2 scaling and the hardware's exponential of 2 units in the
    last place: e = (D + 8) 2^-24 S + 8 2^-24 (1 + S); a weight and the sum of weights are off by e each: 2 e A;
  * sums of n weights and products in 32 bits: n 2^-24 A at most;
  * the result is rounded once: u |o|.
"""
import pytest

from whisper4j_b200._lib import IllegalStateError

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F16, BF16 = torch.float16, torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make(groups, shared, lens, nq=1, heads=4, kv=2, dim=64, page=16, dtype=F16, seed=0, layers=1, spread=1.0):
    """A cache whose rows are laid on random pages; groups: sequences of each group; lens: tokens of each sequence."""
    from whisper4j_b200 import ops
    g = torch.Generator("cuda").manual_seed(seed)
    order = torch.Generator().manual_seed(seed)
    start = [sum(groups[:i]) for i in range(len(groups) + 1)]
    n_pages = sum(-(-n // page) for n in lens) + 3
    pool = torch.full((2 * layers, n_pages, kv, page, dim), float("nan"), device="cuda", dtype=dtype)
    free = iter(torch.randperm(n_pages, generator=order).tolist())
    rows = torch.randperm(len(lens) + 2, generator=order)[:len(lens)].tolist()
    width = max(1, max(-(-n // page) for n in lens)) + 1
    table = torch.full((len(lens) + 2, width), -9, dtype=torch.int32)
    length = torch.full((len(lens) + 2,), 5, dtype=torch.int32)
    for gi in range(len(groups)):
        for i in range(start[gi], start[gi + 1]):
            r, n = rows[i], lens[i]
            length[r] = n
            first = rows[start[gi]]
            for j in range(-(-n // page)):
                if i > start[gi] and (j + 1) * page <= shared[gi]:
                    table[r, j] = table[first, j]
                    continue
                p = table[r, j] = next(free)
                k = min(page, n - j * page)
                data = torch.randn(2 * layers, kv, k, dim, device="cuda", generator=g) * spread
                same = max(0, min(k, shared[gi] - j * page)) if i > start[gi] else 0
                data = data.to(dtype)
                if same:
                    data[:, :, :same] = pool[:, table[first, j], :, :same]
                pool[:, p, :, :k] = data
    ref = torch.bincount(table[table >= 0].long(), minlength=n_pages).int()
    cache = ops.PagedCache.from_tensors(pool, ref.cuda(), table.cuda(), length.cuda())
    q = (torch.randn(len(lens), nq, heads, dim, device="cuda", generator=g) * spread).to(dtype)
    return dict(cache=cache, q=q, rows=ints(rows), start=ints(start), shared=ints(shared), lens=lens,
                max_shared=max(shared), max_own=max(n - shared[gi] for gi in range(len(groups))
                                                    for n in lens[start[gi]:start[gi + 1]]))


def attend(s, layer=0, **kw):
    return s["cache"].attend(layer, s["q"], s["rows"], s["start"], s["shared"], s["max_shared"], s["max_own"], **kw)


def verify(s, out, layer=0, scale=None, skip=()):
    c, q = s["cache"], s["q"]
    n_seq, nq, heads, dim = q.shape
    kv, page, rep = c.n_kv_head, c.page_tokens, heads // c.n_kv_head
    scale = dim ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    t0 = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    table, rows = c.table.tolist(), s["rows"].tolist()
    assert out.dtype == q.dtype
    for i, n in enumerate(s["lens"]):
        if i in skip:
            continue
        pages = table[rows[i]][:-(-n // page)]
        k, v = (c.pool[2 * layer + w, pages].transpose(0, 1).reshape(kv, len(pages) * page, dim)[:, :n].double()
                .repeat_interleave(rep, 0) for w in (0, 1))
        for t in range(nq):
            m = max(0, n - nq + t + 1)
            got = out[i, t].double()
            if m == 0:
                assert not got.any(), (i, t)
                continue
            x = q[i, t].double()
            sc = scale * torch.einsum("hd,hkd->hk", x, k[:, :m])
            S = scale * torch.einsum("hd,hkd->hk", x.abs(), k[:, :m].abs()).max()
            p = torch.softmax(sc, 1)
            o = torch.einsum("hk,hkd->hd", p, v[:, :m])
            A = torch.einsum("hk,hkd->hd", p, v[:, :m].abs())
            e = (dim + 8) * 2 ** -24 * S + 8 * 2 ** -24 * (1 + S)
            tol = A * (u + 2 * e + m * 2 ** -24) + m * t0 / 2 * v[:, :m].abs().max() + o.abs() * u + t0
            bad = (got - o).abs() > tol
            assert not bad.any(), (i, t, float(((got - o).abs() / tol).max()))
    c.check()


SHAPES = [
    dict(groups=[1], shared=[0], lens=[1]),
    dict(groups=[1], shared=[0], lens=[37]),
    dict(groups=[5], shared=[224], lens=[230, 230, 230, 230, 230], heads=8, kv=8),
    dict(groups=[5], shared=[227], lens=[228, 231, 243, 260, 500], heads=8, kv=8),
    dict(groups=[3, 1, 4], shared=[16, 0, 33], lens=[17, 40, 16, 5, 34, 33, 64, 65], heads=6, kv=2),
    dict(groups=[2, 0, 3], shared=[7, 0, 100], lens=[8, 7, 101, 130, 100]),
    dict(groups=[40], shared=[500], lens=[500 + i % 7 for i in range(40)], heads=2, kv=2),
    dict(groups=[33, 17], shared=[1029, 64], lens=[1030 + 3 * i for i in range(33)] + [64 + 5 * i for i in range(17)], heads=4,
         kv=1),
    dict(groups=[150], shared=[2047], lens=[2047 + (7 * i) % 90 for i in range(150)], heads=1, kv=1),
    dict(groups=[70], shared=[300], lens=[303 + i for i in range(70)], nq=3, heads=10, kv=2),
    dict(groups=[4, 4], shared=[60, 61], lens=[70, 64, 65, 80, 65, 66, 67, 100], nq=4, heads=4, kv=4),
    dict(groups=[2], shared=[5], lens=[30, 40], nq=20, heads=6, kv=3),
    dict(groups=[1, 2], shared=[0, 0], lens=[0, 2, 0], nq=1),
    dict(groups=[3], shared=[0], lens=[2, 0, 9], nq=5),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=range(len(SHAPES)))
def test_against_64_bits(shape, dim, dtype):
    s = make(dim=dim, dtype=dtype, **shape)
    verify(s, attend(s))


# few rows and long ones: a row's keys are shared out over the blocks of a cluster, whose size these change
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,heads,nq", [(1, 1, 1), (3, 8, 1), (4, 8, 1), (5, 8, 1), (9, 8, 1), (13, 8, 1), (5, 4, 11)])
def test_few_long_rows(n, heads, nq, dim):
    shared = 0 if n == 1 else 701
    lens = [[3017, 2100, 701, 0, 1, 640, 513][i % 7] if i else 3017 for i in range(n)]
    lens = [max(x, shared) if x > 1 else x for x in lens]
    s = make([1] * n, [shared if x > shared else 0 for x in lens], lens, nq=nq, heads=heads, kv=heads, dim=dim, page=24)
    verify(s, attend(s))


@pytest.mark.parametrize("page", [8, 24, 64, 136, 1024])
@pytest.mark.parametrize("dim", [64, 128])
def test_page_sizes(page, dim):
    s = make([3, 70], [page, 5 * page // 2], [page, page + 1, 3 * page] + [5 * page // 2 + i for i in range(70)], page=page,
             dim=dim, heads=3, kv=1)
    verify(s, attend(s))


@pytest.mark.parametrize("spread", [0.01, 4.0])
def test_flat_and_peaked_rows(spread):
    s = make([6, 140], [40, 700], [50] * 6 + [700 + i for i in range(140)], spread=spread, seed=3)
    verify(s, attend(s))


def test_layers_scale_and_strides():
    s = make([4], [70], [71, 90, 110, 75], nq=2, heads=6, kv=2, layers=3)
    wide = torch.zeros(4, 2, 904, dtype=F16, device="cuda")
    wide[..., 8:392] = s["q"].flatten(2)
    s["q"] = wide[..., 8:392].unflatten(2, (6, 64))
    place = torch.full((4, 2, 800), 7.0, dtype=F16, device="cuda")
    out = attend(s, layer=2, scale=0.3, out=place[..., :384].unflatten(2, (6, 64)))
    verify(s, out, layer=2, scale=0.3)
    assert (place[..., 384:] == 7).all()


def test_long_shared_text():
    s = make([20], [20000], [20000 + 50 * i for i in range(20)], heads=8, kv=8, page=64)
    verify(s, attend(s))
    s = make([130], [9000], [9000 + i for i in range(130)], heads=2, kv=1, page=32, dim=128, dtype=BF16)
    verify(s, attend(s))


@pytest.mark.parametrize("what", ["nan", "inf"])
def test_later_tokens_of_the_same_row_may_be_anything(what):
    """A query's future tokens hold NaN or infinities in K and V: it does not see them."""
    s = make([2], [40], [50, 61], nq=4, heads=6, kv=2)
    c = s["cache"]
    clean = attend(s)
    for i, n in enumerate(s["lens"]):
        r = int(s["rows"][i])
        p = int(c.table[r, (n - 2) // 16])
        c.pool[:, p, :, (n - 2) % 16] = float(what)  # seen by the last two queries only
    out = attend(s)
    assert torch.equal(out[:, :2], clean[:, :2])
    assert not torch.isfinite(out[:, 2:]).any()
    c.check()


def test_nan_in_one_row_stays_there():
    s = make([40], [100], [110 + i for i in range(40)], heads=4, kv=2)
    clean = attend(s)
    s["q"][3] = float("nan")
    out = attend(s)
    assert torch.isnan(out[3]).all()
    keep = [i for i in range(40) if i != 3]
    assert torch.equal(out[keep], clean[keep])


def test_the_same_twice():
    s = make([100, 30], [800, 90], [800 + i for i in range(100)] + [95] * 30, heads=4, kv=4)
    first = attend(s)
    for _ in range(3):
        assert torch.equal(attend(s), first)


def bad(s, text, rows):
    out = attend(s)
    with pytest.raises(IllegalStateError, match=text):
        s["cache"].check()
    assert torch.isnan(out[rows]).all()
    return out


@pytest.mark.parametrize("n", [4, 140])
def test_bad_sequences_are_marked(n):
    def fresh():
        return make([n, 2], [64, 33], [70 + i for i in range(n)] + [40, 50], nq=2)
    clean = attend(fresh())
    others = [i for i in range(n + 2) if i != 2]
    s = fresh()
    s["rows"][2] = n + 4
    assert torch.equal(bad(s, "out of range", [2])[others], clean[others])
    s = fresh()
    s["cache"].table[int(s["rows"][2]), 4] = 1 << 20  # the row's own page
    assert torch.equal(bad(s, "table entry", [2])[others], clean[others])
    s = fresh()
    s["cache"].len[int(s["rows"][2])] = 64  # its first query sees 63 tokens only
    assert torch.equal(bad(s, "shared", [2])[others], clean[others])
    s = fresh()
    s["shared"][1] = 65  # over max_shared
    assert torch.equal(bad(s, "shared", [n, n + 1])[:n], clean[:n])
    s = fresh()
    s["shared"][1] = -1
    bad(s, "shared", [n, n + 1])
    s = fresh()
    s["cache"].table[int(s["rows"][0]), 1] = -1  # a shared page: the whole group
    assert torch.equal(bad(s, "table entry", list(range(n)))[n:], clean[n:])
    s = fresh()
    s["start"][2] = n + 1  # the last sequence is in no group
    bad(s, "ascend", [n + 1])
    s = fresh()
    s["start"][1] = n + 5  # groups that do not ascend
    attend(s)
    with pytest.raises(IllegalStateError, match="ascend"):
        s["cache"].check()


@pytest.mark.parametrize("max_own", [0, 1])
@pytest.mark.parametrize("n,shared", [(2, 40), (30, 40), (30, 0)])
def test_rows_may_outgrow_max_own(n, shared, max_own):
    s = make([n], [shared], [40 + 97 * (i + 1) for i in range(n)], heads=8, kv=8)
    s["max_own"] = max_own
    verify(s, attend(s))


def test_a_bad_page_late_in_a_long_row():
    """Read by one of the blocks that share the row's keys: all of the row's results are marked."""
    s = make([1, 1], [0, 0], [2000, 2000], heads=8, kv=8)
    clean = attend(s)
    s["cache"].table[int(s["rows"][0]), 120] = 1 << 20
    assert torch.equal(bad(s, "table entry", [0])[1], clean[1])


def test_captured_and_replayed():
    """One graph replayed while rows grow: lengths, tables and groups are read on the device."""
    from whisper4j_b200 import ops
    c = ops.PagedCache(1, 2, 64, 64, 16, 6, 200)
    rows, start = ints([0, 1, 2]), ints([0, 1, 2, 3])
    c.extend(ints([0]), ints([0, 50]))
    kv = torch.randn(2, 50, 2, 64, device="cuda").half()
    c.write(0, ints([0]), ints([0, 50]), kv[0], kv[1])
    c.fork(ints([1, 2]), ints([0, 0]))
    q, out = torch.zeros(3, 1, 4, 64, dtype=F16, device="cuda"), torch.empty(3, 1, 4, 64, dtype=F16, device="cuda")
    new = torch.zeros(2, 3, 2, 64, dtype=F16, device="cuda")
    group, shared = ints([0, 3]), ints([50])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.extend(rows, start)
        c.write(0, rows, start, new[0], new[1])
        c.attend(0, q, rows, group, shared, 50, 100, out=out)
    for step in range(20):
        q.normal_(), new.normal_()
        graph.replay()
        verify(dict(cache=c, q=q, rows=rows, lens=[51 + step] * 3), out)


def test_two_graphs_at_once():
    """Each captured call has scratch of its own: two graphs may replay side by side."""
    sets = [make([60], [400], [401 + i for i in range(60)], heads=4, kv=4, seed=i) for i in (1, 2)]
    want = [attend(s) for s in sets]
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attend(s))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_argument_checks():
    s = make([2], [20], [30, 31])
    c, q = s["cache"], s["q"]
    for kw in (dict(q=q.float()), dict(q=q[0]), dict(q=q[..., :32]), dict(rows=s["rows"][:1]), dict(start=ints([0])),
               dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)[:, :, ::2]), dict(max_shared=-1),
               dict(max_own=1 << 20), dict(rows=s["rows"].long())):
        with pytest.raises(ValueError):
            attend({**s, **kw})
    with pytest.raises(ValueError):
        attend(s, scale=0.0)
    with pytest.raises(ValueError):
        attend(s, scale=float("nan"))
    with pytest.raises(ValueError):
        attend(s, layer=1)
    with pytest.raises(ValueError):
        attend(s, out=torch.empty_like(q).float())
    assert attend({**s, "q": q[:0]}).shape == (0, 1, 4, 64)
    verify(s, attend(s))
