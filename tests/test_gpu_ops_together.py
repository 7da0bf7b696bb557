"""The operators together, as a host's own loop uses them: two layers of a decoder step over a paged cache, a prompt that
the beams of a stream share, a beam reorder after every step, rows that leave and a pool that closes up; against the same
steps in 64 bits on the numbers that the quantised weights stand for, with a cache per beam that nobody shares.

Each step's outputs carry the 16-bit roundings of the projections (u = eps / 2 of float16 each) and of the quantised
activations (half of 1 / 127 of a row's largest) through attention, so outputs are compared in the 2-norm: a layer adds
to a residual stream of norm |x| a change of norm |d|, off by at most (1 / 127 + 8 u) |d| for each of its four
quantisations (an error of half a step of the largest element, uniformly in a row, is below 1 / 127 of the row's norm).
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

HEADS, DIM, LAYERS = 6, 64, 2
D = HEADS * DIM


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Layer:
    def __init__(self, g):
        from whisper4j_b200 import ops
        w = [torch.randn(n, k, device="cuda", generator=g) * k ** -0.5 for n, k in ((3 * D, D), (D, D), (4 * D, D), (D, 4 * D))]
        b = [0.1 * torch.randn(t.shape[0], device="cuda", generator=g) for t in w]
        self.ln = [(1 + 0.1 * torch.randn(D, device="cuda", generator=g), 0.1 * torch.randn(D, device="cuda", generator=g))
                   for _ in range(2)]
        self.qkv, self.out, self.up, self.down = (ops.Int8Linear.from_float(t, c) for t, c in zip(w, b))
        # the numbers that the integers stand for
        self.exact = [(m.weight[:, :m.k].double() * m.scale.double()[:, None], m.bias.double())
                      for m in (self.qkv, self.out, self.up, self.down)]


def norm(x, ln):
    x = x - x.mean(-1, keepdim=True)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * ln[0].double() + ln[1].double()


def exact_step(layers, x, caches, n_new):
    """x: (rows, n_new, D) in 64 bits; caches[row][layer]: (k, v) lists of tokens, extended here."""
    for li, layer in enumerate(layers):
        (wq, bq), (wo, bo), (wu, bu), (wd, bd) = layer.exact
        qkv = norm(x, layer.ln[0]) @ wq.T + bq
        q, k, v = (t.unflatten(2, (HEADS, DIM)) for t in qkv.split(D, 2))
        att = torch.empty_like(q)
        for r in range(x.shape[0]):
            ks, vs = (torch.cat([old, new], 0) for old, new in zip(caches[r][li], (k[r], v[r])))
            caches[r][li] = (ks, vs)
            for t in range(n_new):
                n = ks.shape[0] - n_new + t + 1
                p = torch.softmax(torch.einsum("hd,khd->hk", q[r, t], ks[:n]) * DIM ** -0.5, 1)
                att[r, t] = torch.einsum("hk,khd->hd", p, vs[:n])
        x = x + att.flatten(2) @ wo.T + bo
        h = norm(x, layer.ln[1]) @ wu.T + bu
        h = h / (1 + torch.exp(-2 * 0.7978845608028654 * (h + 0.044715 * h ** 3)))
        x = x + h @ wd.T + bd
    return x


def step(layers, x, cache, rows, start, group, shared, max_shared, max_own):
    """The same by the operators: x (rows, n_new, D) float32, changed in place."""
    n, n_new, _ = x.shape
    flat = x.view(n * n_new, D)
    cache.extend(rows, start)
    for li, layer in enumerate(layers):
        qkv = layer.qkv(flat, ln=layer.ln[0], out_dtype=torch.float16).view(n * n_new, 3, HEADS, DIM)
        cache.write(li, rows, start, qkv[:, 1], qkv[:, 2])
        q = qkv[:, 0].unflatten(0, (n, n_new))
        att = cache.attend(li, q, rows, group, shared, max_shared, max_own)
        layer.out(att.view(n * n_new, D), epilogue="residual", out=flat)
        h = layer.up(flat, ln=layer.ln[1], epilogue="gelu", out_dtype=torch.float16)
        layer.down(h, epilogue="residual", out=flat)
    return x


def near(got, want, x0):
    """Off by at most (1 / 127 + 8 u) of each layer's changes, four times over."""
    change = (want - x0.double()).norm(dim=-1)
    bound = 4 * LAYERS * (1 / 127 + 8 * 2.0 ** -11) * (change + x0.double().norm(dim=-1))
    assert ((got.double() - want).norm(dim=-1) <= bound).all()
    return float(((got.double() - want).norm(dim=-1) / want.norm(dim=-1)).max())


@pytest.mark.parametrize("streams,beams,prompt", [(1, 5, 37), (3, 4, 16), (20, 5, 50)])
def test_beam_search_of_a_small_decoder(streams, beams, prompt):
    from whisper4j_b200 import ops
    g = torch.Generator("cuda").manual_seed(streams)
    layers = [Layer(g) for _ in range(LAYERS)]
    n = streams * beams
    cache = ops.PagedCache(LAYERS, HEADS, DIM, n_pages=40 * n, page_tokens=16, n_rows=n + 3, max_tokens=prompt + 20)
    heads = [s * beams for s in range(streams)]  # the row of each stream's first beam
    one = [[(torch.empty(0, HEADS, DIM, dtype=torch.float64, device="cuda"),) * 2 for _ in range(LAYERS)] for _ in heads]
    # the prompt, once for each stream: every token sees those before it
    x = torch.randn(streams, prompt, D, device="cuda", generator=g)
    x0, want = x.clone(), exact_step(layers, x.double(), one, prompt)
    step(layers, x, cache, ints(heads), ints([prompt * i for i in range(streams + 1)]), ints(list(range(streams + 1))),
         ints([0] * streams), 0, prompt)
    worst = near(x, want, x0)
    # the other beams go on from there
    cache.fork(ints([s * beams + b for s in range(streams) for b in range(1, beams)]), ints([h for h in heads for _ in range(1, beams)]))
    caches = [[kv for kv in one[r // beams]] for r in range(n)]
    rows, start = ints(list(range(n))), ints(list(range(n + 1)))
    group, shared = ints([s * beams for s in range(streams + 1)]), ints([prompt] * streams)
    order = torch.Generator().manual_seed(5)
    for t in range(6):
        x = torch.randn(n, 1, D, device="cuda", generator=g)
        x0, want = x.clone(), exact_step(layers, x.double(), caches, 1)
        step(layers, x, cache, rows, start, group, shared, prompt, 20)
        worst = max(worst, near(x, want, x0))
        src = [s * beams + int(b) for s in range(streams) for b in torch.randint(0, beams, (beams,), generator=order)]
        cache.fork(rows, ints(src))
        caches = [[kv for kv in caches[r]] for r in src]
        if t == 3:
            assert int(cache.compact()) == int((cache.ref > 0).sum())
    assert worst < 0.05  # far inside the bound: roundings do not conspire
    assert cache.len[:n].tolist() == [prompt + 6] * n
    cache.free(rows)
    cache.check()
    assert not cache.ref.any()


def test_a_step_in_a_graph_gives_what_it_gives_outside():
    from whisper4j_b200 import ops
    g = torch.Generator("cuda").manual_seed(3)
    layers = [Layer(g) for _ in range(LAYERS)]
    caches = [ops.PagedCache(LAYERS, HEADS, DIM, 200, 16, 10, 100) for _ in range(2)]
    rows, start, group, shared = ints(list(range(10))), ints(list(range(11))), ints([0, 5, 10]), ints([20, 20])
    first = torch.randn(2, 20, D, device="cuda", generator=g)
    for c in caches:
        step(layers, first.clone(), c, ints([0, 5]), ints([0, 20, 40]), ints([0, 1, 2]), ints([0, 0]), 0, 20)
        c.fork(ints([1, 2, 3, 4, 6, 7, 8, 9]), ints([0] * 4 + [5] * 4))
    x = torch.zeros(10, 1, D, device="cuda")
    step(layers, x.clone(), ops.PagedCache(LAYERS, HEADS, DIM, 200, 16, 10, 100), rows, start, group, ints([0, 0]), 20, 80)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(layers, x, caches[0], rows, start, group, shared, 20, 80)
        caches[0].fork(rows, rows.flip(0).contiguous())
    for _ in range(5):
        new = torch.randn(10, 1, D, device="cuda", generator=g)
        x.copy_(new)
        graph.replay()
        step(layers, new, caches[1], rows, start, group, shared, 20, 80)
        caches[1].fork(rows, rows.flip(0).contiguous())
        assert torch.equal(x, new)
    for a, b in zip(caches[0].pool.flatten(0, 1), caches[1].pool.flatten(0, 1)):
        assert torch.equal(a, b)
    for c in caches:
        c.check()


def test_gradients_are_refused_and_changes_are_counted():
    """While autograd records, tensors that require a gradient are refused (the outputs would have none in silence), and a
    tensor that was kept for a backward pass and then written over makes that pass fail."""
    from whisper4j_b200 import ops

    c = ops.PagedCache(1, 2, 64, 8, 16, 2, 64)
    rows, start, group, shared = ints([0]), ints([0, 3]), ints([0, 1]), ints([0])
    kv = torch.randn(2, 3, 2, 64, device="cuda").half()
    c.extend(rows, start)
    c.write(0, rows, start, kv[0], kv[1])
    q = torch.randn(1, 1, 2, 64, device="cuda").half()
    x, w = torch.randn(3, 32, device="cuda"), torch.nn.Parameter(torch.randn(16, 32, device="cuda"))
    bias = torch.nn.Parameter(torch.randn(16, device="cuda"))
    layer = ops.Int8Linear.from_float(w, bias)
    norm = (torch.ones(32, device="cuda"), torch.zeros(32, device="cuda"))

    def grad(t):
        return t.detach().clone().requires_grad_()

    y = torch.zeros(3, 16, device="cuda")
    calls = (lambda: c.write(0, rows, start, grad(kv[0]), kv[1]), lambda: c.attend(0, grad(q), rows, group, shared, 0, 3),
             lambda: c.attend(0, q, rows, group, shared, 0, 3, out=grad(q)), lambda: ops.quantize_rows(grad(x)),
             lambda: layer(grad(x)), lambda: layer(x, ln=(grad(norm[0]), norm[1])), lambda: layer(x, out=grad(y)),
             lambda: layer(x, epilogue="residual", out=grad(y)))
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    with pytest.raises(ValueError, match="gradient"):
        ops.PagedCache.from_tensors(grad(c.pool), c.ref, c.table, c.len)
    layer(x), layer(x, ln=norm)  # the layer's own numbers are none
    a = torch.ones(3, 16, device="cuda", requires_grad=True)
    for over in (lambda t: layer(x, out=t), lambda t: layer(x, epilogue="residual", out=t)):
        kept = torch.zeros(3, 16, device="cuda")
        product = (a * kept).sum()
        over(kept)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()
    kept = q.clone()
    product = (kept * torch.ones_like(q).requires_grad_()).sum()
    c.attend(0, q, rows, group, shared, 0, 3, out=kept)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    for call in (lambda: c.write(0, rows, start, kv[0], kv[1]), lambda: c.fork(ints([1]), ints([0])), lambda: c.compact()):
        product = (c.pool[0] * torch.ones_like(c.pool[0]).requires_grad_()).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()
    with torch.inference_mode():
        layer(x, out=torch.empty(3, 16, device="cuda"))
