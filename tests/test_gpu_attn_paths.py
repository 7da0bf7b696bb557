"""The attention kernels that take calls of many rows: 128-row tiles on the tensor cores, warps for the groups of few rows
and for all own tokens, and the join of their parts.

A few rows that are not very long go another way, in one launch that needs no scratch; every case here asks the library
for its scratch first, so that a case which that launch would take fails instead of testing nothing.  The tensor cores
take shared keys from 24 (head 64) or 16 (head 128) query rows of a group and head on: the groups here have 40 and more
or at most 15.  Values, tolerances and the reference are test_gpu_attn_shared.py's.
"""
import ctypes

import pytest

from whisper4j_b200._lib import IllegalStateError

from .test_gpu_attn_shared import BF16, F16, attend, bad, make, verify

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def by_parts(s):
    """Asserts that the call is not one for the launch without scratch."""
    from whisper4j_b200 import _lib
    c, (n_seq, nq, heads, _) = s["cache"], s["q"].shape
    a = _lib.AttnShared(ctypes.pointer(c._c), 0, heads, nq, n_seq, s["shared"].numel(), s["max_shared"], s["max_own"], 1.0)
    n = ctypes.c_size_t()
    assert _lib.lib().w4j_op_attn_shared_workspace(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value > 0
    return s


# (rows of each group, heads, key/value heads, queries a row): groups on the tensor cores, on warps of 8 and of 16 rows
TC, TC_GROUPED, WARP8, WARP16 = ([80, 75], 1, 1, 1), ([41, 40], 12, 4, 1), ([5] * 32, 1, 1, 1), ([3] * 52, 5, 1, 1)
PATHS = dict(tc=TC, tc_grouped=TC_GROUPED, warp8=WARP8, warp16=WARP16)


def case(path, shared, own, **kw):
    """Every group shares about `shared` tokens; the rows' own numbers of tokens run over `own`."""
    groups, heads, kv, nq = PATHS[path]
    nq = kw.pop("nq", nq)
    per = [max(0, shared - 3 * g % 7) for g in range(len(groups))]
    lens = [per[g] + own[i % len(own)] for g, n in enumerate(groups) for i in range(n)]
    return by_parts(make(groups, per, lens, nq=nq, heads=heads, kv=kv, **kw))


@pytest.mark.parametrize("page", [8, 24, 64, 136, 1024])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("path", PATHS)
def test_page_sizes(path, dim, page):
    s = case(path, 5 * min(page, 150) // 2, [1, 9, 30, 2, 70], page=page, dim=dim, dtype=BF16 if page == 24 else F16)
    verify(s, attend(s))


# shared lengths about the borders of boxes and tiles, none at all, and long ones
@pytest.mark.parametrize("shared", [0, 1, 63, 64, 65, 127, 129, 192, 1100])
@pytest.mark.parametrize("path,dtype", [(p, t) for p in PATHS for t in (F16, BF16)])
def test_shared_lengths(path, dtype, shared):
    s = case(path, shared, [1, 3, 17], page=16, dim=64 if shared % 2 else 128, dtype=dtype)
    verify(s, attend(s))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("path", PATHS)
def test_long_own_parts(path, dim):
    """Own tokens in several pieces, some of which end before they begin."""
    s = case(path, 100, [700, 1, 300, 257, 512], page=24, dim=dim)
    verify(s, attend(s))


@pytest.mark.parametrize("heads,kv,nq", [(10, 2, 7), (5, 1, 20), (1, 1, 33), (16, 16, 17)])
@pytest.mark.parametrize("dim", [64, 128])
def test_several_tiles_of_own_queries(dim, heads, kv, nq):
    groups = [45, 2, 13]
    shared = [80, 0, 21]
    lens = [shared[g] + nq + i % 60 for g, n in enumerate(groups) for i in range(n)]
    s = by_parts(make(groups, shared, lens, nq=nq, heads=heads, kv=kv, dim=dim, page=8))
    verify(s, attend(s))


@pytest.mark.parametrize("heads,kv,dim,dtype", [(6, 6, 64, F16), (8, 2, 64, BF16), (5, 1, 128, F16)])
@pytest.mark.parametrize("nq,shared,lens", [(448, 0, [448, 300, 449, 600]), (130, 200, [329, 330, 331, 700, 513]), (1000, 0, [1000])])
def test_prompts(nq, shared, lens, heads, kv, dim, dtype):
    """A whole prompt's queries at once, one of them longer than its row; all queries of a row against 64 bits together."""
    s = by_parts(make([len(lens)], [shared], lens, nq=nq, heads=heads, kv=kv, dim=dim, dtype=dtype, page=24))
    out, c, rows, table = attend(s), s["cache"], s["rows"].tolist(), s["cache"].table.tolist()
    u, scale = torch.finfo(dtype).eps / 2, dim ** -0.5
    t0 = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for i, n in enumerate(lens):
        pages = table[rows[i]][:-(-n // 24)]
        k, v = (c.pool[w, pages].transpose(0, 1).reshape(kv, -1, dim)[:, :n].double().repeat_interleave(heads // kv, 0) for w in (0, 1))
        x = s["q"][i].double().transpose(0, 1)
        see = n - nq + torch.arange(nq, device="cuda")[:, None] >= torch.arange(n, device="cuda")
        sc = (scale * x @ k.transpose(1, 2)).masked_fill(~see, float("-inf"))
        S = (scale * x.abs() @ k.abs().transpose(1, 2)).amax(2, keepdim=True)
        p = torch.nan_to_num(torch.softmax(sc, 2))
        o, A = p @ v, p @ v.abs()
        e = (dim + 8) * 2 ** -24 * S + 8 * 2 ** -24 * (1 + S)
        tol = A * (u + 2 * e + n * 2 ** -24) + n * t0 / 2 * v.abs().max() + o.abs() * u + t0
        got = out[i].double().transpose(0, 1)
        assert ((got - o).abs() <= tol).all(), i
        assert not got[:, :max(0, nq - n)].any()
    c.check()


@pytest.mark.parametrize("path", PATHS)
def test_rows_that_see_little_or_nothing(path):
    """No token, fewer tokens than queries, and groups that share nothing."""
    groups, heads, kv, _ = PATHS[path]
    n = sum(groups)
    s = by_parts(make(groups, [0] * len(groups), [(0, 1, 2, 9, 0, 40)[i % 6] for i in range(n)], nq=5, heads=heads, kv=kv))
    verify(s, attend(s))


@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("own", [7, 600])
@pytest.mark.parametrize("path", PATHS)
def test_later_tokens_may_be_anything(path, own, what):
    """Tokens that only a row's last two queries see hold NaN or infinities, in a row's one piece or its last of several.
    (Not bit by bit as without them: where a tile holds such a number its 16-key sums start from zero.)"""
    groups, heads, kv, _ = PATHS[path]
    if path.startswith("warp"):
        groups = [1] * 160  # with four queries each as few rows as before
    shared = [50] * len(groups)
    lens = [50 + own + i % 5 for i in range(sum(groups))]
    s = by_parts(make(groups, shared, lens, nq=4, heads=heads, kv=kv))
    c, clean = s["cache"], attend(s)
    verify(s, clean)
    rows, table = s["rows"].tolist(), c.table.tolist()
    for i, n in enumerate(lens):
        p = table[rows[i]][(n - 2) // 16]
        c.pool[:, p, :, (n - 2) % 16] = float(what)
    out = attend(s)
    assert not torch.isfinite(out[:, 2:]).any()
    verify({**s, "q": s["q"][:, :2], "lens": [n - 2 for n in lens]}, out[:, :2])


@pytest.mark.parametrize("hidden", [64, 128, 192, 320])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("path", list(PATHS) + ["direct"])
def test_keys_that_score_minus_infinity(path, dtype, hidden):
    """The first keys score -inf and the others about -200, where no rounding may lose them: their values' mean, for scores
    that are equal.  (Weights are 1 then, and sums of up to 512 numbers of the type's half step each: 2 u |v| at most.)"""
    if path == "direct":
        s = make([2], [400], [410, 403], heads=4, kv=2, dtype=dtype)
    else:
        s = case(path, 400, [3, 10], dtype=dtype)
    c, q = s["cache"], s["q"]
    page, dim = c.page_tokens, c.head_dim
    c.pool.nan_to_num_()
    c.pool[0] = 0
    q.zero_()
    q[..., 0], q[..., 1] = 1, 1
    c.pool[0, ..., 1] = -200  # times scale: -25
    table, rows, start = c.table.tolist(), s["rows"].tolist(), s["start"].tolist()
    for i, n in enumerate(s["lens"]):
        for j in range(hidden // page):
            c.pool[0, table[rows[i]][j], ..., 0] = float("-inf")
    out = attend(s, scale=1.0)
    u = torch.finfo(dtype).eps / 2
    rep = q.shape[2] // c.n_kv_head
    for i, n in enumerate(s["lens"]):
        g = max(x for x in range(len(start) - 1) if start[x] <= i)
        shared = int(s["shared"][g])
        pages = [table[rows[start[g]]][j] if (j + 1) * page <= shared else table[rows[i]][j] for j in range(-(-n // page))]
        v = c.pool[1, pages].transpose(0, 1).reshape(c.n_kv_head, -1, dim)[:, hidden:n].double().repeat_interleave(rep, 0)
        want, a = v.mean(1), v.abs().mean(1)
        tol = a * (2 * u + 2 ** -13) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert ((out[i, 0].double() - want).abs() <= tol).all(), i
    c.check()


@pytest.mark.parametrize("path", PATHS)
def test_nan_in_one_row_stays_there(path):
    s = case(path, 90, [4, 20, 33])
    clean = attend(s)
    s["q"][3] = float("nan")
    out = attend(s)
    assert torch.isnan(out[3]).all()
    keep = [i for i in range(len(s["lens"])) if i != 3]
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("path", PATHS)
def test_bad_sequences_are_marked(path):
    def fresh():
        return case(path, 70, [5, 30, 44])
    clean = attend(fresh())
    n = len(clean)
    s = fresh()
    first = int(s["start"][1])  # sequences of the first group
    others = [i for i in range(n) if i != 2]
    s["rows"][2] = n + 4
    assert torch.equal(bad(s, "out of range", [2])[others], clean[others])
    s = fresh()
    s["cache"].table[int(s["rows"][2]), (s["lens"][2] - 1) // 16] = 1 << 20
    assert torch.equal(bad(s, "table entry", [2])[others], clean[others])
    s = fresh()
    s["shared"][0] = s["max_shared"] + 1
    assert torch.equal(bad(s, "shared", list(range(first)))[first:], clean[first:])
    s = fresh()
    s["cache"].table[int(s["rows"][0]), 1] = -1  # a shared page: the whole group
    assert torch.equal(bad(s, "table entry", list(range(first)))[first:], clean[first:])


@pytest.mark.parametrize("heads,kv,nq,n", [(4, 2, 1, 6), (8, 2, 3, 6), (4, 2, 1, 60), (8, 2, 3, 60)])  # without and with scratch
def test_groups_that_are_wrong_as_a_whole(heads, kv, nq, n):
    """Sequences that are in no group are NaN in all heads; those whose group is right are as ever."""
    def fresh():
        groups = [n, n // 2, n, n // 3]
        return make(groups, [40, 17, 0, 33], [45 + i % 9 for i in range(sum(groups))], nq=nq, heads=heads, kv=kv)

    def wrong(change, lost, same):
        s = fresh()
        change(s["start"])
        out = attend(s)
        with pytest.raises(IllegalStateError, match="ascend"):
            s["cache"].check()
        assert torch.isnan(out[lost]).all() and torch.equal(out[same], clean[same])

    clean = attend(fresh())
    total, g1, g2, g3 = len(clean), n, n + n // 2, 2 * n + n // 2
    if n == 60:
        by_parts(fresh())

    def last_early(start):
        start[4] -= 1
    wrong(last_early, [total - 1], list(range(total - 1)))

    def first_late(start):
        start[0] = 1
    wrong(first_late, [0], list(range(g1, total)))

    def descends(start):  # the third group starts behind the fourth
        start[2] = g3 + 1
    wrong(descends, [], list(range(g2)) + list(range(g3, total)))

    def outside(start):  # the third group ends, and the fourth begins, behind the last sequence
        start[3] = total + 5
    wrong(outside, list(range(g2, total)), list(range(g2)))


@pytest.mark.parametrize("path", PATHS)
def test_in_place_and_repeated(path):
    s = case(path, 200, [4, 300, 33])
    first = attend(s)
    for _ in range(3):
        assert torch.equal(attend(s), first)
    assert torch.equal(attend(s, out=s["q"]), first)  # over the queries


@pytest.mark.parametrize("path", ["direct", "cluster", "tc", "warp8", "warp16"])
def test_waits_that_run_out_are_reported(path):
    """The hook makes every wait for keys count on more bytes than come; nothing faults, and the next call is as ever."""
    from whisper4j_b200._lib import check, lib
    if path == "direct":
        s = make([2], [20], [30, 41])
    elif path == "cluster":
        s = make([1], [0], [3000])
    else:
        s = case(path, 70, [5, 30, 44])
    clean = attend(s)
    check(lib().w4j_test_attn_shared_waits_run_out(1))
    try:
        out = attend(s)
        with pytest.raises(IllegalStateError, match="ran out"):
            s["cache"].check()
    finally:
        check(lib().w4j_test_attn_shared_waits_run_out(0))
    assert torch.isnan(out).all()
    assert torch.equal(attend(s), clean)
    s["cache"].check()


def test_a_pool_beyond_32_bits():
    """Planes of 4 GiB: new pages, copies, reads and moves at the far end of the last ones."""
    from whisper4j_b200 import ops
    n_pages, page = 1 << 17, 16
    c = ops.PagedCache(2, 8, 128, n_pages, page, 4, 512, dtype=BF16)
    c.ref.fill_(1)
    c.ref[-40:] = 0  # the others are somebody else's
    rows, start = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([0, 300, 323], dtype=torch.int32, device="cuda")
    kv = torch.randn(2, 323, 8, 128, device="cuda").to(BF16)
    c.extend(rows, start)
    c.write(1, rows, start, kv[0], kv[1])
    c.fork(torch.tensor([2], dtype=torch.int32, device="cuda"), rows[:1])
    c.check()
    assert c.table[:3, 0].tolist() == [n_pages - 40, n_pages - 21, n_pages - 40] and int(c.table[2, 18]) == n_pages - 19
    for n in (3, 160):  # without and with scratch
        order = [i % 3 for i in range(n)]
        lens = [(300, 23, 300)[i] for i in order]
        q = torch.randn(n, 1, 8, 128, device="cuda").to(BF16)
        s = dict(cache=c, q=q, rows=torch.tensor(order, dtype=torch.int32, device="cuda"), lens=lens, max_shared=0, max_own=300,
                 start=torch.arange(n + 1, dtype=torch.int32, device="cuda"), shared=torch.zeros(n, dtype=torch.int32, device="cuda"))
        out = attend(s, layer=1)
        verify(s, out, layer=1)
    c.ref[5:9] = 0  # holes, far from the pages that close them
    assert int(c.compact()) == n_pages - 40 + 22 - 4
    assert sorted(set(c.table[:3].flatten().tolist()) & {5, 6, 7, 8}) == [5, 6, 7, 8]
    assert torch.equal(attend(s, layer=1), out)
    c.check()
