"""The 8-bit integer Linear against its definition in 64 bits.

The quantised numbers of a row without a LayerNorm are exactly defined and have to be equal.  A product's integer sum is
exact; after it come the conversion (2^-24), two products (2^-24 each) and the bias (2^-24) in 32 bits, and the
rounding to y's type (u = eps / 2, nothing for 32 bits), so |error| <= 4 2^-24 (|product| + |y|) + u |y|; a residual adds
one more sum of 32 bits.  GELU has slope below 1.13, and its own arithmetic v / (1 + exp(-2 u)) an exponential of
2 + 1.2 |2 u| units in the last place with an argument that is off by 4 2^-24 |2 u|: (8 + 8 |u|) 2^-23 relative.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = [torch.float32, torch.float16, torch.bfloat16]
E = 2.0 ** -24


def quantised(x):
    """(q, scale) of float32-valued rows, in 64 bits."""
    x = x.double()
    s = torch.from_numpy(x.abs().amax(1).float().cpu().numpy() * np.float32(1 / 127)).to(x.device)
    q = torch.where(s[:, None] > 0, x / s.double()[:, None], 0).round().clamp(-127, 127)
    return q.to(torch.int8), s


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 1280), (3, 7), (5, 8), (2, 9), (4, 16), (7, 100), (33, 1000), (300, 1280), (64, 2049),
                                 (10, 5120), (3, 8200), (2, 20001), (1300, 1280), (1500, 130), (1201, 2048), (1200, 4096)])
def test_quantize_is_exact(m, k, dtype):
    from whisper4j_b200 import ops
    g = torch.Generator("cuda").manual_seed(m + k)
    x = (torch.randn(m, k, device="cuda", generator=g) * torch.rand(m, 1, device="cuda", generator=g) * 50).to(dtype)
    q, s = ops.quantize_rows(x)
    qw, sw = quantised(x.float())
    assert q.shape == (m, (k + 15) // 16 * 16)
    assert torch.equal(s, sw)
    assert torch.equal(q[:, :k], qw)
    assert not q[:, k:].any()


def test_quantize_ties_borders_and_extremes():
    from whisper4j_b200 import ops
    rows = [[127.0, 0.5, 1.5, -0.5, -2.5, 126.5, 3.5 + 2 ** -20, 3.5 - 2 ** -20],
            [3.0, 0.0, -3.0, 1.0, 2.0, 1e-30, -1e-30, 0.1],
            [0.0] * 8, [-0.0] * 8, [1e-40] * 8, [1e-45, 0, 0, 0, 0, 0, 0, 0], [3e-38, 1e-38, -2e-38, 1e-39, 5e-39, 0, 0, 0],
            [3.4e38, -3.4e38, 1e38, 1.0, 1e30, 2e38, 0, -1e38], [1e-31 * i for i in range(8)],
            [1e-44, 2e-44, 3e-44, 7e-44, 1e-43, 9e-44, 0, 0]]
    x = torch.tensor(rows, dtype=torch.float32, device="cuda")
    rnd = torch.randn(20000, 8, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    # quotients next to halves: x = (n + 1/2) s, one step to either side
    s = (rnd[:, :1].abs() + 0.1) * 127 / 127
    n = torch.randint(-126, 126, (20000, 8), device="cuda", generator=torch.Generator("cuda").manual_seed(2)) + 0.5
    near = (n * s).float()
    near[:, 0] = (s * 127)[:, 0]
    near[:, 3] = torch.nextafter(near[:, 3], torch.tensor(9e9, device="cuda"))
    near[:, 4] = torch.nextafter(near[:, 4], torch.tensor(-9e9, device="cuda"))
    for t in (x, near):
        q, sc = ops.quantize_rows(t)
        qw, sw = quantised(t)
        assert torch.equal(sc, sw)
        assert torch.equal(q[:, :8], qw)


def test_rows_that_are_not_finite():
    from whisper4j_b200 import ops
    x = torch.randn(6, 40, device="cuda")
    x[1, 3], x[2, 39], x[4, 0] = float("nan"), float("inf"), float("-inf")
    q, s = ops.quantize_rows(x)
    assert torch.isnan(s).tolist() == [False, True, True, False, True, False]
    assert not q[[1, 2, 4]].any()
    y = ops.Int8Linear.from_float(torch.randn(9, 40, device="cuda"))(x)
    assert torch.isnan(y).all(1).tolist() == [False, True, True, False, True, False]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 16), (4, 1280), (33, 777), (2, 5120), (2, 9001), (1500, 1280), (1200, 2048)])
def test_quantize_behind_a_layer_norm(m, k, dtype):
    """The normalised row is off by 32-bit sums of depth d, a thread's run of 8 ceil(K / 2048) elements (ceil(K / 32) where
    rows are many) and 20 for the warp and the block: the mean by d E mean|x|, the deviation's factor by (d + 8) E; a
    quantised number by half a step more."""
    from whisper4j_b200 import ops
    g = torch.Generator("cuda").manual_seed(k)
    x = (torch.randn(m, k, device="cuda", generator=g) * 3 + 1).to(dtype)
    gamma = 1 + 0.1 * torch.randn(k, device="cuda", generator=g)
    beta = 0.1 * torch.randn(k, device="cuda", generator=g)
    q, s = ops.quantize_rows(x, ln=(gamma, beta))
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    y = (x - mean) * rstd * gamma.double() + beta.double()
    d = (8 * math.ceil(k / 2048) if m < 1000 else math.ceil(k / 32)) + 20
    off = gamma.double().abs() * rstd * d * E * x.abs().mean(1, keepdim=True) + (y - beta.double()).abs() * (d + 8) * E + y.abs() * 2 * E
    want = y.abs().amax(1) / 127
    assert ((s.double() - want).abs() <= off.amax(1) / 127 + 2 * E * want).all()
    back = q[:, :k].double() * s.double()[:, None]
    assert ((back - y).abs() <= 0.5 * s.double()[:, None] * (1 + 1e-6) + off).all()


def product_case(m, k, n, ytype, epilogue, bias, seed=0, big=False, ldy=None):
    from whisper4j_b200 import _lib
    from whisper4j_b200._lib import check, lib
    g = torch.Generator("cuda").manual_seed(seed + m + 3 * k + 7 * n)
    k16, ldy = (k + 15) // 16 * 16, ldy or n + 3
    xq = torch.zeros(m, k16 + 32, dtype=torch.int8, device="cuda")
    wq = torch.zeros(n, k16 + 16, dtype=torch.int8, device="cuda")
    if big:  # the largest sums there are
        xq[:, :k], wq[:, :k] = 127, 127
        xq[1::2, :k] = -128
    else:
        xq[:, :k] = torch.randint(-128, 128, (m, k), device="cuda", generator=g)
        wq[:, :k] = torch.randint(-128, 128, (n, k), device="cuda", generator=g)
    xq[:, k16:], wq[:, k16:] = 99, 99  # behind the padding there may be anything
    scale = 4.0 / (74 * 74 * math.sqrt(k))
    xs = torch.rand(m, device="cuda", generator=g) + 0.5
    ws = (torch.rand(n, device="cuda", generator=g) + 0.5) * scale
    b = torch.randn(n, device="cuda", generator=g) if bias else None
    y = torch.randn(m, ldy, device="cuda", generator=g).to(ytype)
    before = y.clone()
    code = {torch.float32: _lib.GGML_F32, torch.float16: _lib.GGML_F16, torch.bfloat16: _lib.GGML_BF16}[ytype]
    check(lib().w4j_op_linear_i8(0, xq.data_ptr(), k16 + 32, xs.data_ptr(), m, k, wq.data_ptr(), k16 + 16, ws.data_ptr(), n,
                                 b.data_ptr() if bias else None, epilogue, y.data_ptr(), code, ldy,
                                 torch.cuda.current_stream().cuda_stream))
    assert torch.equal(y[:, n:], before[:, n:])  # nothing behind the last channel
    prod = (xq[:, :k].double() @ wq[:, :k].double().T) * xs.double()[:, None] * ws.double()
    v = prod + (b.double() if bias else 0)
    tol = 4 * E * (prod.abs() + v.abs())
    if epilogue == 1:
        u = math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
        v = v / (1 + torch.exp(-2 * u))
        tol = 1.13 * tol + v.abs() * (8 + 8 * u.abs()) * 2 * E + 1e-36
    elif epilogue == 2:
        v = v + before[:, :n].double()
        tol = tol + E * v.abs()
    half = 0 if ytype == torch.float32 else torch.finfo(ytype).eps / 2
    tol = tol * (1 + half) + half * v.abs() + (torch.finfo(ytype).smallest_normal * torch.finfo(ytype).eps)
    bad = (y[:, :n].double() - v).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("ytype", TYPES)
@pytest.mark.parametrize("epilogue", [0, 1, 2])
@pytest.mark.parametrize("m,k,n", [(1, 16, 1), (1, 1280, 3840), (2, 384, 51), (5, 100, 700), (8, 5120, 1280), (9, 1280, 129),
                                   (16, 2048, 512), (17, 512, 1000), (40, 1280, 1280), (77, 1000, 701), (128, 5120, 1280),
                                   (130, 384, 384), (320, 5120, 1280), (700, 1280, 640)])
def test_product(m, k, n, epilogue, ytype):
    product_case(m, k, n, ytype, epilogue, bias=(m + n) % 2 == 0 or epilogue == 1)


@pytest.mark.parametrize("m,k,n", [(3000, 1280, 5120), (1500, 384, 1536), (2049, 1008, 2050), (257, 5120, 1300)])
@pytest.mark.parametrize("epilogue,ytype", [(0, torch.float32), (1, torch.float16), (2, torch.bfloat16)])
def test_large_products(m, k, n, epilogue, ytype):
    product_case(m, k, n, ytype, epilogue, True)


@pytest.mark.parametrize("m,k,n", [(3000, 1280, 5120), (2049, 1008, 2050), (1537, 200, 2000), (12000, 48, 264)])
@pytest.mark.parametrize("epilogue", [0, 1, 2])
@pytest.mark.parametrize("ytype", TYPES)
def test_large_products_with_aligned_rows(m, k, n, epilogue, ytype):
    """Rows of y a multiple of 16 bytes apart: outputs may leave in boxes."""
    product_case(m, k, n, ytype, epilogue, epilogue == 1, ldy=(n + 23) // 8 * 8)


@pytest.mark.parametrize("m", [1, 4, 60, 300])
def test_sums_at_the_limit_of_32_bits(m):
    product_case(m, 131056, 130, torch.float32, 0, False, big=True)


@pytest.mark.parametrize("xtype,ytype", [(torch.float32, torch.float32), (torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16)])
def test_layer(xtype, ytype):
    """The whole layer against a Linear on the numbers that its integers stand for."""
    from whisper4j_b200 import ops
    g = torch.Generator("cuda").manual_seed(9)
    w, b = torch.randn(700, 1000, device="cuda", generator=g) * 0.03, torch.randn(700, device="cuda", generator=g)
    x = torch.randn(50, 1100, device="cuda", generator=g).to(xtype)[:, 60:1060]
    layer = ops.Int8Linear.from_float(w, b)
    wq, ws = quantised(w)
    assert torch.equal(layer.weight[:, :1000], wq) and torch.equal(layer.scale, ws)
    xq, xs = quantised(x.float())
    v = (xq.double() @ wq.double().T) * xs.double()[:, None] * ws.double() + b.double()
    half = 0 if ytype == torch.float32 else torch.finfo(ytype).eps / 2
    y = layer(x, out_dtype=ytype)
    assert y.dtype == ytype
    assert ((y.double() - v).abs() <= (8 * E + half) * (v.abs() + b.double().abs())).all()
    wide = torch.zeros(50, 1500, dtype=ytype, device="cuda")
    layer(x, out=wide[:, 3:703])
    assert torch.equal(wide[:, 3:703], y) and not wide[:, :3].any() and not wide[:, 703:].any()
    again = layer(x, epilogue="residual", out=y.clone())
    assert ((again.double() - 2 * v).abs() <= (16 * E + 3 * half) * (2 * v.abs() + b.double().abs())).all()
    assert layer(x[:0]).shape == (0, 700)


@pytest.mark.parametrize("ln", [False, True])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("k,n,xtype", [(1, 3, torch.float32), (384, 1152, torch.float16), (1000, 50, torch.bfloat16),
                                       (1530, 4737, torch.float16), (768, 129, torch.float16), (511, 40, torch.float16), (380, 9475, torch.bfloat16),
                                       (5120, 129, torch.float32), (6200, 40, torch.float32), (20000, 10, torch.float32)])
def test_layer_of_a_few_rows(m, k, n, xtype, ln):
    """One launch where the rows are few and short, two where not; behind a LayerNorm against its exact value: a
    quantised number may be half a step off, and more by the LayerNorm's own sums (a run of ceil(K / 32) + 20 at most)."""
    from whisper4j_b200 import ops
    g = torch.Generator("cuda").manual_seed(m + k)
    w, b = torch.randn(n, k, device="cuda", generator=g) * k ** -0.5, torch.randn(n, device="cuda", generator=g)
    x = (torch.randn(m, k + 3, device="cuda", generator=g) * 2 + 0.5).to(xtype)[:, 1:k + 1]
    norm = (1 + 0.1 * torch.randn(k, device="cuda", generator=g), 0.1 * torch.randn(k, device="cuda", generator=g)) if ln else None
    layer = ops.Int8Linear.from_float(w, b)
    y = layer(x, ln=norm, out_dtype=torch.float32)
    wq, ws = quantised(w)
    v = x.double()
    if not ln:
        q, s = quantised(x.float())
        want = (q.double() @ wq.double().T) * s.double()[:, None] * ws.double() + b.double()
        assert ((y.double() - want).abs() <= 8 * E * (want.abs() + b.double().abs())).all()
        return
    mean = v.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    z = (v - mean) * rstd * norm[0].double() + norm[1].double()
    d = math.ceil(k / 32) + 20
    off = norm[0].double().abs() * rstd * d * E * v.abs().mean(1, keepdim=True) + (z - norm[1].double()).abs() * (d + 8) * E + z.abs() * 2 * E
    step = z.abs().amax(1, keepdim=True) / 127
    wide = wq.double().abs() * ws.double()[:, None]
    want = z @ (wq.double() * ws.double()[:, None]).T + b.double()
    tol = (0.5 * step * (1 + 1e-5) + off).expand_as(z) @ wide.T
    assert ((y.double() - want).abs() <= tol + 8 * E * (want.abs() + b.double().abs())).all()


def test_a_few_rows_that_are_not_finite():
    from whisper4j_b200 import ops
    layer = ops.Int8Linear.from_float(torch.randn(20, 70, device="cuda"))
    x = torch.randn(5, 70, device="cuda")
    x[1, 69], x[2], x[3, 0], x[4] = float("nan"), 0, float("-inf"), 1e-42
    y = layer(x)
    assert torch.isnan(y).all(1).tolist() == [False, True, False, True, False]
    assert not y[2].any()


def test_captured_on_a_side_stream():
    from whisper4j_b200 import ops
    layer = ops.Int8Linear.from_float(torch.randn(640, 320, device="cuda"))
    x = torch.zeros(70, 320, device="cuda")
    out = torch.empty(70, 640, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x, out=out)
    for i in range(5):
        x.normal_()
        graph.replay()
        assert torch.equal(out, layer(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = layer(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, out)


def test_refusals():
    from whisper4j_b200 import ops
    w = torch.randn(30, 40, device="cuda")
    layer = ops.Int8Linear.from_float(w)
    x = torch.randn(3, 40, device="cuda")
    for bad in (lambda: layer(x[:, :39]), lambda: layer(x.double()), lambda: layer(x.cpu()), lambda: layer(x, epilogue="relu"),
                lambda: layer(x, epilogue="residual"), lambda: layer(x, out=torch.empty(3, 31, device="cuda")),
                lambda: layer(x, out=torch.empty(3, 30, device="cuda"), out_dtype=torch.float16), lambda: layer(x.t()),
                lambda: layer(x, ln=(x[0], x[0, :39])), lambda: ops.Int8Linear(w, w[:, 0]),
                lambda: ops.Int8Linear(layer.weight, layer.scale[:5]), lambda: layer(x.T.contiguous().T)):
        with pytest.raises(ValueError):
            bad()


def gelu_of(v, m, ytype, quantised=True):
    """GELU of the biases v as each of m rows has them, by a product whose sums are 0."""
    from whisper4j_b200 import _lib, ops
    from whisper4j_b200._lib import check, lib
    n = len(v)
    b = torch.tensor(v, dtype=torch.float32, device="cuda")
    w, ws = torch.ones(n, 16, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda")
    y = torch.full((m, n), 5.0, dtype=ytype, device="cuda")
    if not quantised:
        return ops.Int8Linear(w, ws, b)(torch.zeros(m, 16, device="cuda"), epilogue="gelu", out=y)
    x, xs = torch.zeros(m, 16, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda")
    code = {torch.float32: _lib.GGML_F32, torch.float16: _lib.GGML_F16, torch.bfloat16: _lib.GGML_BF16}[ytype]
    check(lib().w4j_op_linear_i8(0, x.data_ptr(), 16, xs.data_ptr(), m, 16, w.data_ptr(), 16, ws.data_ptr(), n, b.data_ptr(), 1,
                                 y.data_ptr(), code, n, torch.cuda.current_stream().cuda_stream))
    return y


GELU_ROWS = [(1, False), (3, False), (1, True), (4, True), (8, True), (40, True), (130, True), (1500, True)]  # the kernels


@pytest.mark.parametrize("ytype", TYPES)
@pytest.mark.parametrize("m,quantised", GELU_ROWS)
def test_gelu_far_from_zero(m, quantised, ytype):
    """Beyond |v| = 8 GELU is v or, to 1e-18, 0, whatever the number beside it that an epilogue may take along."""
    far = [-7.6, -7.7, -8.0, -30.0, -100.0, -1e4, -1e19, -1e20, -1e38, 1e-30, 8.0, 100.0, 6e4, 0.0, -0.5, 1.0]
    v = [far[i % 16] for i in range(480)] + [far[i // 16 % 16] for i in range(480)] + [far[i * 5 % 16] for i in range(480)]
    y = gelu_of(v, m, ytype, quantised).double()
    x = torch.tensor(v, dtype=torch.float64, device="cuda").float().double()
    u = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    want = torch.where(x < -8, 0, x / (1 + torch.exp(-2 * u)))
    half = 0 if ytype == torch.float32 else torch.finfo(ytype).eps / 2
    tol = want.abs() * ((8 + 8 * u.abs().clamp(max=50)) * 2 * E + half) + 1e-18 * (x < -7) + torch.finfo(ytype).smallest_normal * torch.finfo(ytype).eps
    assert ((y - want).abs() <= tol).all()
    odd = gelu_of([float("nan"), float("inf"), float("-inf"), 2.0] * 400, m, torch.float32, quantised)[:, :4]
    assert torch.isnan(odd[:, [0, 2]]).all() and (odd[:, 1] == float("inf")).all()  # the formula's -inf x 0 is none
    assert ((odd[:, 3] - 1.9545976).abs() <= 1e-5).all()


@pytest.mark.parametrize("epilogue", ["store", "gelu", "residual"])
@pytest.mark.parametrize("ln", [False, True])
@pytest.mark.parametrize("m,k", [(1, 1280), (2, 512), (4, 384), (5, 512), (300, 512), (2100, 256)])
def test_outputs_over_the_inputs(m, k, ln, epilogue):
    """h = h + W LayerNorm(h) in place, and outputs that lie across their inputs."""
    from whisper4j_b200 import _lib, ops
    g = torch.Generator("cuda").manual_seed(m)
    layer = ops.Int8Linear.from_float(torch.randn(k, k, device="cuda", generator=g) * k ** -0.5, torch.randn(k, device="cuda", generator=g))
    norm = (1 + 0.1 * torch.randn(k, device="cuda", generator=g), 0.1 * torch.randn(k, device="cuda", generator=g)) if ln else None
    x = torch.randn(m, k, device="cuda", generator=g)
    # the rows quantised first, then the product: whole numbers behind a LayerNorm are these
    q, s = ops.quantize_rows(x, norm)
    want = x.clone()
    _lib.check(_lib.lib().w4j_op_linear_i8(0, q.data_ptr(), k, s.data_ptr(), m, k, layer.weight.data_ptr(), k, layer.scale.data_ptr(), k,
                                           layer.bias.data_ptr(), ops.Int8Linear.EPILOGUES[epilogue], want.data_ptr(), 0, k,
                                           torch.cuda.current_stream().cuda_stream))
    for _ in range(5):
        h = x.clone()
        assert torch.equal(layer(h, ln=norm, epilogue=epilogue, out=h), want)
        wide = torch.zeros(m, 2 * k, device="cuda")
        wide[:, :k] = x
        if epilogue == "residual":
            base = wide[:, k // 2:k // 2 + k].clone()
            out = layer(wide[:, :k], ln=norm, epilogue=epilogue, out=wide[:, k // 2:k // 2 + k])
            assert ((out - base - (want - x)).abs() <= 4 * E * (out.abs() + want.abs() + x.abs() + base.abs())).all()  # four sums
        else:
            assert torch.equal(layer(wide[:, :k], ln=norm, epilogue=epilogue, out=wide[:, k // 2:k // 2 + k]), want)


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.float8_e4m3fn])
def test_types_of_outputs_are_refused_as_arguments(dtype):
    from whisper4j_b200 import ops
    layer = ops.Int8Linear.from_float(torch.randn(30, 40, device="cuda"))
    for m in (1, 40):
        with pytest.raises(ValueError, match="out"):
            layer(torch.randn(m, 40, device="cuda"), out_dtype=dtype)
        with pytest.raises(ValueError, match="out"):
            layer(torch.randn(m, 40, device="cuda"), out=torch.empty(m, 30, device="cuda").to(dtype))


@pytest.mark.parametrize("ldy", [(1 << 15) + 8, (1 << 15) + 9])  # whole boxes of outputs, and single ones
def test_outputs_and_rows_beyond_32_bits(ldy):
    from whisper4j_b200 import ops
    m, n, k = (1 << 17) + 3, (1 << 15) + 8, 48
    layer = ops.Int8Linear.from_float(torch.randn(n, k, device="cuda"), torch.randn(n, device="cuda"))
    x = torch.randn(m, k, device="cuda")
    y = torch.empty(m, ldy, device="cuda", dtype=torch.float16)[:, :n]
    layer(x, out=y)
    for a in (0, (1 << 16) - 40, m - 80):
        part = layer(x[a:a + 80], out_dtype=torch.float16).double()
        assert ((y[a:a + 80].double() - part).abs() <= 2 * torch.finfo(torch.float16).eps * part.abs() + 2 ** -24).all()
    del y
    wide = torch.randn(80, 1040, device="cuda", dtype=torch.float16).repeat(1 << 15, 1)
    q, s = ops.quantize_rows(wide)
    want = ops.quantize_rows(wide[:80].clone())
    assert torch.equal(q[-80:], want[0]) and torch.equal(s[-80:], want[1]) and torch.equal(q[80 << 14:][:80], want[0])
