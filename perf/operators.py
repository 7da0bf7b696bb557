"""Measured cases of the op-level operators for hosts that drive their own decode loop.

Three families, each with its plain form in elementary torch operations beside the library's calls:

* ``attend``: softmax attention of a batch over a paged key/value cache in which the sequences of a group share
  their first tokens, computed once for the whole group;
* ``fork`` / ``turnover``: the pages themselves (a beam reorder; finished rows leaving, the pool closing up and new
  rows coming in);
* ``linear``: a Linear layer in 8-bit integers, activations quantised row by row, weights by output channel.

``run`` takes what ``prepare`` gives, computes one pass and returns its outputs.  Where ``own`` is true it calls
whisper4j_b200.ops, else the plain form.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one stream of base.en under beam search: five beams behind the previous-text prompt, one token each
        dict(name="attend-base-beam5", kind="attend", groups=1, seqs=5, query=1, heads=8, kv_heads=8, dim=64, page=16,
             shared=227, own_lo=57, own_hi=57, type="f16"),
        # 64 streams of large-v3-turbo, five beams each, every stream at its own position of the 448-token context
        dict(name="attend-turbo-64x5", kind="attend", groups=64, seqs=5, query=1, heads=20, kv_heads=20, dim=64, page=16,
             shared=227, own_lo=1, own_hi=221, type="f16"),
        # 256 sequences behind one long common text, ragged tails
        dict(name="attend-256x8192", kind="attend", groups=1, seqs=256, query=1, heads=20, kv_heads=20, dim=64, page=64,
             shared=8192, own_lo=1, own_hi=512, type="f16"),
        # grouped heads, four drafted tokens checked per sequence, four long documents of 16 sequences
        dict(name="attend-grouped-16381", kind="attend", groups=4, seqs=16, query=4, heads=32, kv_heads=8, dim=128,
             page=32, shared=16381, own_lo=4, own_hi=1024, type="bf16"),
        # the beam reorder after one step: one stream of base.en, then 64 streams of large-v3-turbo
        dict(name="fork-base-beam5", kind="fork", groups=1, beams=5, layers=6, kv_heads=8, dim=64, page=16, lo=100,
             hi=100, type="f16"),
        dict(name="fork-turbo-64x5", kind="fork", groups=64, beams=5, layers=4, kv_heads=20, dim=64, page=16, lo=65,
             hi=448, type="f16"),
        # finished rows leave, the pool closes up, new rows enter with their prompts: a few short rows, then 64 long ones
        dict(name="turnover-base-4", kind="turnover", rows=4, layers=6, kv_heads=8, dim=64, page=16, lo=5, hi=90,
             type="f16"),
        dict(name="turnover-turbo-64", kind="turnover", rows=64, layers=4, kv_heads=20, dim=64, page=16, lo=1, hi=448,
             type="f16"),
        # large-v3-turbo's Q/K/V projection of one token
        dict(name="linear-1x1280x3840", kind="linear", m=1, k=1280, n=3840, x="f32", y="f32", ln=False, act="store"),
        # the MLP's second projection for 64 streams of five beams, added to the residual stream
        dict(name="linear-320x5120x1280", kind="linear", m=320, k=5120, n=1280, x="f32", y="f32", ln=False,
             act="residual"),
        # the encoder's LayerNorm, first MLP projection and GELU over eight 30 s windows
        dict(name="linear-12000x1280x5120", kind="linear", m=12000, k=1280, n=5120, x="f32", y="f16", ln=True,
             act="gelu"),
        # sizes that divide by nothing
        dict(name="linear-77x1000x701", kind="linear", m=77, k=1000, n=701, x="bf16", y="bf16", ln=False, act="store"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["attend", "attend", "fork", "turnover", "linear", "linear"])
    if kind == "attend":
        kv_heads = rng.choice([1, 2, 4, 6, 8, 12, 20])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 5])
        query = rng.choice([1, 1, 1, 2, 4, 7])
        own_hi = _log(rng, query, 1100)
        return dict(kind=kind, groups=_log(rng, 1, 64), seqs=_log(rng, 1, 256), query=query, heads=heads,
                    kv_heads=kv_heads, dim=rng.choice([64, 128]), page=rng.choice([8, 16, 24, 32, 64, 128]),
                    shared=_log(rng, 1, 20000) - 1, own_lo=rng.randint(query, max(query, own_hi)),
                    own_hi=max(query, own_hi), type=rng.choice(["f16", "bf16"]))
    if kind == "fork":
        hi = _log(rng, 1, 448)
        return dict(kind=kind, groups=_log(rng, 1, 64), beams=rng.randint(2, 8), layers=rng.choice([1, 4, 6]),
                    kv_heads=rng.choice([2, 6, 8, 20]), dim=rng.choice([64, 128]), page=rng.choice([8, 16, 24, 64]),
                    lo=rng.randint(1, hi), hi=hi, type=rng.choice(["f16", "bf16"]))
    if kind == "turnover":
        hi = _log(rng, 1, 448)
        return dict(kind=kind, rows=_log(rng, 1, 64), layers=rng.choice([1, 4, 6]), kv_heads=rng.choice([2, 6, 8, 20]),
                    dim=rng.choice([64, 128]), page=rng.choice([8, 16, 24, 64]), lo=rng.randint(1, hi), hi=hi,
                    type=rng.choice(["f16", "bf16"]))
    x = rng.choice(["f32", "f16", "bf16"])
    ln = rng.random() < 0.3
    # behind a LayerNorm the integers depend on the last bit of its sums, which a 32-bit output would show
    y = rng.choice(["f16", "bf16"] if ln else ["f32", "f16", "bf16"])
    return dict(kind=kind, m=_log(rng, 1, 12000), k=_log(rng, 16, 5120), n=_log(rng, 1, 5120), x=x, y=y, ln=ln,
                act=rng.choice(["store", "gelu", "residual"]))


def _cost(case):
    """What a drawn case may not have more of than the listed ones of its kind: work, and memory of its cache."""
    rows = case["groups"] * case["beams"] if case["kind"] == "fork" else 0
    tokens = sum(-(-n // case["page"]) * case["page"] for n in _spread(case["lo"], case["hi"], rows)) if rows else 0
    return [*work(case).values(), tokens * 2 * case.get("layers", 0) * case.get("kv_heads", 0) * case.get("dim", 0) * 2]


def draw(rng):
    while True:
        c = _draw(rng)
        if all(v <= max(m) for v, m in zip(_cost(c), zip(*(_cost(p) for p in listed() if p["kind"] == c["kind"])))):
            return c


def _spread(lo, hi, n):
    """n lengths spread evenly over lo .. hi."""
    return [lo + (2 * i + 1) * (hi - lo + 1) // (2 * n) for i in range(n)]


def _shared(case):
    """The groups' shared lengths: not all alike where there are several groups."""
    return [max(0, case["shared"] - (13 * g) % 61) for g in range(case["groups"])]


def work(case):
    kind = case["kind"]
    if kind == "linear":
        size = {"f32": 4, "f16": 2, "bf16": 2}
        m, k, n = case["m"], case["k"], case["n"]
        y = m * n * size[case["y"]] * (2 if case["act"] == "residual" else 1)
        return {"bytes": m * k * size[case["x"]] + n * k + 4 * n * 2 + y + (8 * k if case["ln"] else 0),
                "flops": 2 * m * n * k}
    if kind == "attend":
        b = case["groups"] * case["seqs"]
        shared, tail = _shared(case), _spread(case["own_lo"], case["own_hi"], b)
        rows = case["query"] * case["heads"]
        keys = sum(shared) + sum(tail)
        pairs = rows * (sum(s * case["seqs"] for s in shared) + sum(tail)) - b * case["heads"] * case["query"] * (
            case["query"] - 1) // 2
        return {"bytes": (keys * case["kv_heads"] * 2 + 2 * b * rows) * case["dim"] * 2, "flops": 4 * pairs * case["dim"]}
    token = 2 * case["layers"] * case["kv_heads"] * case["dim"] * 2  # bytes of one token in every plane
    page = case["page"]
    if kind == "fork":
        lens = _spread(case["lo"], case["hi"], case["groups"])
        copied = sum(case["beams"] // 2 * (n % page) for n in lens)
        entries = sum(case["beams"] * -(-n // page) for n in lens)
        return {"bytes": 2 * copied * token + 8 * entries, "flops": 0}
    lens = _spread(case["lo"], case["hi"], case["rows"])
    pages = sum(-(-n // page) for n in lens)
    return {"bytes": 2 * pages * page * token + 2 * sum(lens) * token + 12 * pages, "flops": 0}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _pages(gen, layers, kv_heads, dim, page, n_pages, lens, own_pages, shared_with, dtype):
    """A cache of rows of `lens` tokens.  Row i holds its pages in the order of `own_pages`, an iterator of page
    numbers; the first shared_with[i][1] of them are those of row shared_with[i][0]."""
    width = max(1, max(-(-n // page) for n in lens))
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    ref = torch.zeros(n_pages, dtype=torch.int32)
    for i, n in enumerate(lens):
        row, first = shared_with[i]
        count = -(-n // page)
        table[i, :first] = table[row, :first]
        table[i, first:count] = torch.tensor([next(own_pages) for _ in range(count - first)], dtype=torch.int32)
        ref += torch.bincount(table[i, :count].long(), minlength=n_pages).int()
    pool = torch.randn(2 * layers, n_pages, kv_heads, page, dim, device="cuda", generator=gen, dtype=dtype)
    return dict(pool=pool, ref=ref.cuda(), table=table.cuda(), len=torch.tensor(lens, dtype=torch.int32).cuda())


def _ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def _mixed(v, order):
    at = torch.randperm(len(v), generator=order).tolist()
    return [v[i] for i in at]


def _handle(s):
    from whisper4j_b200 import ops

    return ops.PagedCache.from_tensors(s["pool"], s["ref"], s["table"], s["len"])


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    order = torch.Generator().manual_seed(seed)
    kind = case["kind"]
    if kind == "linear":
        return _prepare_linear(case, gen)
    dtype = DTYPES[case["type"]]
    page, layers = case["page"], case.get("layers", 1)
    if kind == "attend":
        b = case["groups"] * case["seqs"]
        shared = _mixed(_shared(case), order)
        tail = _mixed(_spread(case["own_lo"], case["own_hi"], b), order)
        lens = [shared[i // case["seqs"]] + tail[i] for i in range(b)]
        # the group's full pages are shared, what follows them is each row's own, as forking leaves them
        parents = [(i - i % case["seqs"], shared[i // case["seqs"]] // page if i % case["seqs"] else 0) for i in range(b)]
        need = sum(-(-n // page) - p[1] for n, p in zip(lens, parents))
        s = _pages(gen, 1, case["kv_heads"], case["dim"], page, need + need // 8 + 1, lens,
                   iter(torch.randperm(need + need // 8 + 1, generator=order).tolist()), parents, dtype)
        # the last shared page, where it is a partial one, holds the same tokens in every row
        for g, n in enumerate(shared):
            if n % page and case["seqs"] > 1:
                at = s["table"][g * case["seqs"]:(g + 1) * case["seqs"], n // page].long()
                s["pool"][:, at[1:], :, :n % page] = s["pool"][:, at[:1], :, :n % page]
        s |= dict(rows=_ints(list(range(b))), group_start=_ints([g * case["seqs"] for g in range(case["groups"] + 1)]),
                  shared=_ints(shared), max_shared=max(shared), max_own=max(tail), tail=_ints(tail),
                  q=torch.randn(b, case["query"], case["heads"], case["dim"], device="cuda", generator=gen, dtype=dtype),
                  scale=case["dim"] ** -0.5)
    elif kind == "fork":
        beams, lens = case["beams"], _mixed(_spread(case["lo"], case["hi"], case["groups"]), order)
        rows = [n for n in lens for _ in range(beams)]
        # half of each stream's tokens are its prompt and common to its beams
        parents = [(i - i % beams, n // 2 // page if i % beams else 0) for i, n in enumerate(rows)]
        need = sum(-(-n // page) - p[1] for n, p in zip(rows, parents))
        total = need + 2 * len(rows) + 1
        s = _pages(gen, layers, case["kv_heads"], case["dim"], page, total, rows,
                   iter(torch.randperm(total, generator=order).tolist()), parents, dtype)
        dst, src = [], []
        for g in range(case["groups"]):  # beam j goes on from beam j // 2, under other numbers in each stream
            name = torch.randperm(beams, generator=order).tolist()
            dst += [g * beams + name[j] for j in range(beams)]
            src += [g * beams + name[j // 2] for j in range(beams)]
        s |= dict(dst=_ints(dst), src=_ints(src))
    else:
        n = case["rows"]
        halves = [_mixed(_spread(case["lo"], case["hi"], n), order) for _ in range(2)]
        pages = sum(-(-t // page) for h in halves for t in h)
        s = _pages(gen, layers, case["kv_heads"], case["dim"], page, pages + pages // 8 + 1, halves[0] + halves[1],
                   iter(range(pages)), [(0, 0)] * (2 * n), dtype)
        s["rows"] = [_ints(list(range(n))), _ints(list(range(n, 2 * n)))]
        s["start"] = [_ints([sum(h[:i]) for i in range(n + 1)]) for h in halves]
        s["kv"] = [torch.randn(2 * layers, sum(h), case["kv_heads"], case["dim"], device="cuda", generator=gen, dtype=dtype)
                   for h in halves]
        s["turn"] = 0
    s["case"] = case
    if own:
        s["cache"] = _handle(s)
    return s


def _prepare_linear(case, gen):
    m, k, n = case["m"], case["k"], case["n"]
    x = torch.randn(m, k, device="cuda", generator=gen)
    x *= 1 + 7 * (torch.rand(k, device="cuda", generator=gen) < 0.02)  # a few channels stand out, as in trained models
    w = torch.randn(n, k, device="cuda", generator=gen) * k ** -0.5
    ws = w.abs().amax(1) / 127
    wq = torch.round(w.double() / ws.double()[:, None]).to(torch.int8)
    s = dict(case=case, x=x.to(DTYPES[case["x"]]), wq=wq, ws=ws, bias=0.1 * torch.randn(n, device="cuda", generator=gen),
             ln=None, y=None)
    if case["ln"]:
        s["ln"] = (1 + 0.1 * torch.randn(k, device="cuda", generator=gen), 0.1 * torch.randn(k, device="cuda", generator=gen))
    if case["act"] == "residual":
        s["y"] = torch.randn(m, n, device="cuda", generator=gen).to(DTYPES[case["y"]])
    if own:
        from whisper4j_b200 import ops

        s["layer"] = ops.Int8Linear(wq, ws, s["bias"])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if kind == "linear":
        if own:
            return s["layer"](s["x"], ln=s["ln"], epilogue=s["case"]["act"], out=s["y"], out_dtype=DTYPES[s["case"]["y"]])
        return _plain_linear(s)
    if kind == "attend":
        if own:
            return s["cache"].attend(0, s["q"], s["rows"], s["group_start"], s["shared"], max_shared=s["max_shared"],
                                     max_own=s["max_own"], scale=s["scale"])
        return _plain_attend(s)
    if kind == "fork":
        if own:
            s["cache"].fork(s["dst"], s["src"])
        else:
            _plain_fork(s, s["dst"].long(), s["src"].long())
        return {k: s[k].view(torch.int16) if k == "pool" else s[k] for k in ("pool", "ref", "table", "len")}
    turn, s["turn"] = s["turn"], 1 - s["turn"]
    rows, start, kv = s["rows"][turn], s["start"][turn], s["kv"][turn]
    layers = s["case"]["layers"]
    if own:
        cache = s["cache"]
        cache.free(rows)
        live = cache.compact()
        cache.extend(rows, start)
        for layer in range(layers):
            cache.write(layer, rows, start, kv[2 * layer], kv[2 * layer + 1])
    else:
        _plain_free(s, rows.long())
        live = _plain_compact(s)
        _plain_extend(s, rows.long(), start.long())
        for layer in range(layers):
            _plain_write(s, layer, rows.long(), start.long(), kv[2 * layer], kv[2 * layer + 1])
    return {"live": live, **{k: s[k].view(torch.int16) if k == "pool" else s[k] for k in ("pool", "ref", "table", "len")}}


def _plain_linear(s):
    case, x = s["case"], s["x"].float()
    if s["ln"] is not None:
        x = x - x.mean(1, keepdim=True)
        x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-5) * s["ln"][0] + s["ln"][1]
    xs = x.abs().amax(1, keepdim=True) / 127
    # a quotient next to a half goes to its own side in 64 bits
    xq = torch.nan_to_num(torch.round(x.double() / xs.double())).float()
    y = (xq @ s["wq"].float().T) * xs * s["ws"] + s["bias"]
    if case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if case["act"] == "residual":
        s["y"].copy_(s["y"].float() + y)
        return s["y"]
    return y.to(DTYPES[case["y"]])


def _gather(s, plane, table, tokens):
    """Keys or values of the first `tokens` tokens of the rows of `table`: (rows, kv_heads, tokens, dim) in 32 bits."""
    page = s["case"]["page"]
    t = torch.arange(tokens, device="cuda")
    at = table[:, (t // page).clamp(max=table.shape[1] - 1)].long()
    return s["pool"][plane, at, :, t % page].float().movedim(2, 1)


def _plain_attend(s):
    case = s["case"]
    g, n, nq, kv, d = (case[k] for k in ("groups", "seqs", "query", "kv_heads", "dim"))
    rep, page, most = case["heads"] // kv, case["page"], s["max_shared"]
    # the shared tokens, once for all rows of the group
    q = s["q"].float().view(g, n, nq, kv, rep, d) * s["scale"]
    head = s["table"].view(g, n, -1)[:, 0]
    qs = q.movedim(3, 1).reshape(g, kv, n * nq * rep, d)
    common = qs @ _gather(s, 0, head, most).transpose(2, 3)
    common.masked_fill_(torch.arange(most, device="cuda") >= s["shared"][:, None, None, None], float("-inf"))
    # each row's own tokens
    shared = s["shared"].repeat_interleave(n).long()
    t = shared[:, None] + torch.arange(s["max_own"], device="cuda")
    at = s["table"].long().gather(1, (t // page).clamp(max=s["table"].shape[1] - 1))
    k, v = (s["pool"][plane, at, :, t % page].float().movedim(2, 1) for plane in (0, 1))
    qo = q.view(g * n, nq, kv, rep, d).movedim(2, 1).reshape(g * n, kv, nq * rep, d)
    alone = (qo @ k.transpose(2, 3)).view(g * n, kv, nq, rep, -1)
    seen = s["len"].long()[:, None] - nq + torch.arange(nq, device="cuda")  # the last token each query sees
    alone.masked_fill_(t[:, None, None, None] > seen[:, None, :, None, None], float("-inf"))
    common = common.view(g, kv, n, nq, rep, most).movedim(2, 1).reshape(g * n, kv, nq, rep, most)
    top = alone.amax(4, keepdim=True)
    top = torch.maximum(top, common.amax(4, keepdim=True)) if most else top
    alone, common = torch.exp(alone - top), torch.exp(common - top)
    total = alone.sum(4, keepdim=True) + common.sum(4, keepdim=True)
    o = (alone.view(g * n, kv, nq * rep, -1) @ v).view(g * n, kv, nq, rep, d)
    common = common.view(g, n, kv, nq, rep, most).movedim(1, 2).reshape(g, kv, n * nq * rep, most)
    o += (common @ _gather(s, 1, head, most)).view(g, kv, n, nq, rep, d).movedim(2, 1).reshape(g * n, kv, nq, rep, d)
    return (o / total).movedim(1, 2).reshape(g * n, nq, case["heads"], d).to(s["q"].dtype)


def _free_pages(s):
    """Page numbers, the free ones first, each kind in ascending order."""
    return torch.sort((s["ref"] > 0).int(), stable=True)[1]


def _count(s, table, pages, by):
    """Adds `by` to the count of every page of the rows of `table` that hold `pages` pages each."""
    live = torch.arange(table.shape[1], device="cuda") < pages[:, None]
    s["ref"].scatter_add_(0, torch.where(live, table, 0).view(-1).long(), (live.view(-1) * by).int())


def _plain_fork(s, dst, src):
    page = s["case"]["page"]
    n, at = len(dst), torch.arange(len(dst), device="cuda")
    was, held = s["table"][dst], -(-s["len"][dst] // page)
    new, length = s["table"][src], s["len"][src]
    count = -(-length // page)
    # who keeps a partial last page: the source row, if it goes on, else the first that takes it over
    stays = torch.ones_like(s["len"], dtype=torch.bool).scatter_(0, dst, dst == src)
    first = torch.full_like(s["len"], n, dtype=torch.int64).scatter_reduce_(0, src, at, "amin")
    copies = (length % page > 0) & (dst != src) & (stays[src] | (first[src] != at))
    c = copies.nonzero()[:, 0]
    got = _free_pages(s)[:len(c)]
    last = (count[c] - 1).long()
    old = new[c, last].long()
    new[c, last] = got.int()
    _count(s, was, held, -1)
    _count(s, new, count, 1)
    keep = torch.arange(page, device="cuda") < (length[c] % page)[:, None]
    s["pool"][:, got] = torch.where(keep[None, :, None, :, None], s["pool"][:, old], s["pool"][:, got])
    live = torch.arange(new.shape[1], device="cuda") < count[:, None]
    s["table"][dst] = torch.where(live, new, was)
    s["len"][dst] = length


def _plain_free(s, rows):
    _count(s, s["table"][rows], -(-s["len"][rows] // s["case"]["page"]), -1)
    s["len"][rows] = 0


def _plain_compact(s):
    live = (s["ref"] > 0)
    count = live.sum()
    at = torch.arange(len(live), device="cuda")
    holes, high = (~live & (at < count)).nonzero()[:, 0], (live & (at >= count)).nonzero()[:, 0]
    to = at.clone()
    to[high] = holes
    s["pool"][:, holes] = s["pool"][:, high]
    s["ref"][holes] = s["ref"][high]
    s["ref"][high] = 0
    held = torch.arange(s["table"].shape[1], device="cuda") < (-(-s["len"] // s["case"]["page"]))[:, None]
    s["table"].copy_(torch.where(held, to[torch.where(held, s["table"], 0).long()].int(), s["table"]))
    return count.int().view(1)


def _plain_extend(s, rows, start):
    page = s["case"]["page"]
    before, length = s["len"][rows], s["len"][rows] + (start[1:] - start[:-1]).int()
    had, have = -(-before // page), -(-length // page)
    at = torch.arange(s["table"].shape[1], device="cuda")
    new = (at >= had[:, None]) & (at < have[:, None])
    rank = (new.view(-1).long().cumsum(0) - 1).view(new.shape)
    got = _free_pages(s)
    table = torch.where(new, got[rank.clamp(0, len(got) - 1)].int(), s["table"][rows])
    s["table"][rows] = table
    s["ref"].scatter_add_(0, torch.where(new, table, 0).view(-1).long(), new.view(-1).int())
    s["len"][rows] = length


def _plain_write(s, layer, rows, start, k, v):
    page = s["case"]["page"]
    t = torch.arange(len(k), device="cuda")
    i = torch.searchsorted(start, t, right=True) - 1
    at = s["len"][rows[i]].long() - start[i + 1] + t  # the place in its row of each new token
    p = s["table"][rows[i], at // page].long()
    s["pool"][2 * layer, p, :, at % page] = k
    s["pool"][2 * layer + 1, p, :, at % page] = v


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] in ("fork", "turnover"):
        return None  # nothing is computed: whole numbers and moved values
    s = prepare(case, seed)
    if case["kind"] == "linear":
        x = s["x"].double()
        if case["ln"]:
            mean = x.mean(1, keepdim=True)
            var = ((x - mean) ** 2).mean(1, keepdim=True)
            x = (x - mean) / torch.sqrt(var + 1e-5) * s["ln"][0].double() + s["ln"][1].double()
        step = (x.abs().amax(1) / 127).float().double()  # a scale is a 32-bit number
        level = torch.where(step[:, None] > 0, x / step[:, None], 0).round()
        y = torch.einsum("mk,nk->mn", level, s["wq"].double()) * torch.outer(step, s["ws"].double()) + s["bias"].double()
        if case["act"] == "gelu":
            y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
        return y + s["y"].double() if case["act"] == "residual" else y
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    rep, page, lens, nq = case["heads"] // case["kv_heads"], case["page"], s["len"].tolist(), case["query"]
    for b, n in enumerate(lens):  # row by row over all of its tokens
        pages = s["table"][b, :-(-n // page)].long()
        k, v = (s["pool"][i, pages].transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :n].double() for i in (0, 1))
        for t in range(nq):
            m = n - nq + t + 1
            q = s["q"][b, t].double().view(case["kv_heads"], rep, case["dim"])
            p = torch.softmax(s["scale"] * torch.einsum("hrd,hkd->hrk", q, k[:, :m]), 2)
            out[b, t] = torch.einsum("hrk,hkd->hrd", p, v[:, :m]).reshape(case["heads"], case["dim"])
    return out
