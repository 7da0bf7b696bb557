"""Refusals of the op-level operators: every argument check that needs no device (dummy pointers, no launch)."""
import ctypes

import pytest

from whisper4j_b200 import _lib
from whisper4j_b200._lib import GGML_BF16, GGML_F16, GGML_F32, W4J_ERR_ARG, W4J_ERR_CUDA, W4J_OK, Pages, lib

P = 4096  # an aligned dummy address; refused calls never reach it


def cache(**kw):
    f = dict(device=0, type=GGML_F16, n_layer=2, n_kv_head=3, head_dim=64, page_tokens=16, n_pages=10, n_rows=4,
             table_width=5, pool=P, ref=P, table=P, len=P, status=P, work=P, work_bytes=1 << 30)
    f.update(kw)
    return Pages(**f)


def refused(rc, text):
    assert rc == W4J_ERR_ARG, lib().w4j_last_error()
    assert text in lib().w4j_last_error().decode()


def workspace(fn, *args):
    n = ctypes.c_size_t(77)
    rc = fn(*args, ctypes.byref(n))
    assert rc == W4J_OK or n.value == 0
    return rc, n.value


BAD_CACHES = [(dict(type=GGML_F32), "type"), (dict(head_dim=96), "head_dim"), (dict(page_tokens=0), "page_tokens"),
              (dict(page_tokens=12), "page_tokens"), (dict(page_tokens=1032), "page_tokens"), (dict(n_layer=0), "n_layer"),
              (dict(n_kv_head=-1), "n_kv_head"), (dict(n_pages=0), "n_pages"), (dict(n_pages=(1 << 21) + 1), "n_pages"),
              (dict(n_rows=0), "n_rows"), (dict(table_width=0), "table_width"),
              (dict(table_width=1 << 27), "table_width"),
              (dict(n_pages=1 << 21, n_kv_head=64, page_tokens=16), "2^31")]
BAD_POINTERS = [(dict(pool=None), "null"), (dict(ref=None), "null"), (dict(table=None), "null"), (dict(len=None), "null"),
                (dict(status=None), "null"), (dict(work=None), "null"), (dict(pool=P + 8), "aligned"),
                (dict(work=P + 4), "aligned"), (dict(work_bytes=100), "work")]


@pytest.mark.parametrize("kw,text", BAD_CACHES)
def test_workspace_refuses_sizes(kw, text):
    refused(workspace(lib().w4j_op_pages_workspace, ctypes.byref(cache(**kw)))[0], text)


def test_workspace_grows_with_the_cache():
    w = lib().w4j_op_pages_workspace
    small = workspace(w, ctypes.byref(cache(pool=None, work=None)))[1]
    assert 0 < small < workspace(w, ctypes.byref(cache(n_rows=8)))[1] < 1 << 16
    refused(workspace(w, None)[0], "null")
    refused(w(ctypes.byref(cache()), None), "null")


@pytest.mark.parametrize("kw,text", BAD_CACHES + BAD_POINTERS)
def test_every_call_refuses_a_bad_cache(kw, text):
    c, L = ctypes.byref(cache(**kw)), lib()
    refused(L.w4j_op_pages_extend(c, P, P, 1, None), text)
    refused(L.w4j_op_pages_write(c, 0, P, P, 1, P, 192, P, 192, 1, None), text)
    refused(L.w4j_op_pages_fork(c, P, P, 1, None), text)
    refused(L.w4j_op_pages_free(c, P, 1, None), text)
    refused(L.w4j_op_pages_compact(c, None, None), text)


def test_row_lists():
    c, L = ctypes.byref(cache()), lib()
    for n in (-1, 5):
        refused(L.w4j_op_pages_extend(c, P, P, n, None), "rows")
        refused(L.w4j_op_pages_write(c, 0, P, P, n, P, 192, P, 192, 1, None), "rows")
        refused(L.w4j_op_pages_fork(c, P, P, n, None), "rows")
        refused(L.w4j_op_pages_free(c, P, n, None), "rows")
    refused(L.w4j_op_pages_extend(c, P, None, 1, None), "null")
    refused(L.w4j_op_pages_fork(c, None, P, 1, None), "null")
    refused(L.w4j_op_pages_free(c, None, 1, None), "null")
    refused(L.w4j_op_pages_extend(None, P, P, 1, None), "null")
    # nothing to do is no error, and needs no device
    assert L.w4j_op_pages_extend(c, None, None, 0, None) == W4J_OK
    assert L.w4j_op_pages_fork(c, None, None, 0, None) == W4J_OK
    assert L.w4j_op_pages_free(c, None, 0, None) == W4J_OK
    assert L.w4j_op_pages_write(c, 0, P, P, 1, None, 0, None, 0, 0, None) == W4J_OK


@pytest.mark.parametrize("layer,k,ks,v,vs,tokens,text", [
    (-1, P, 192, P, 192, 1, "layer"), (2, P, 192, P, 192, 1, "layer"), (0, P, 192, P, 192, -1, "n_tokens"),
    (0, None, 192, P, 192, 1, "null"), (0, P, 192, None, 192, 1, "null"), (0, P, 184, P, 192, 1, "strides"),
    (0, P, 192, P, 196, 1, "strides"), (0, P, -192, P, 192, 2, "strides"), (0, P + 2, 192, P, 192, 1, "aligned"),
    (0, P, 192, P + 8, 192, 1, "aligned")])
def test_write_refusals(layer, k, ks, v, vs, tokens, text):
    refused(lib().w4j_op_pages_write(ctypes.byref(cache()), layer, P, P, 1, k, ks, v, vs, tokens, None), text)


def test_bf16_is_a_cache_type():
    assert workspace(lib().w4j_op_pages_workspace, ctypes.byref(cache(type=GGML_BF16, head_dim=128)))[1] > 0


def test_a_device_that_is_not_there():
    if _has_gpu():
        refused(lib().w4j_op_pages_free(ctypes.byref(cache(device=99)), P, 1, None), "device 99")
        refused(lib().w4j_op_pages_free(ctypes.byref(cache(device=-1)), P, 1, None), "device -1")
    else:
        assert lib().w4j_op_pages_free(ctypes.byref(cache()), P, 1, None) == W4J_ERR_CUDA


def _has_gpu():
    torch = pytest.importorskip("torch")
    return torch.cuda.is_available()


def test_python_cache_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from whisper4j_b200 import ops
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.PagedCache.from_tensors(torch.zeros(2, 4, 2, 16, 64, dtype=torch.float16), i, i.view(4, 1), i)
    with pytest.raises(ValueError, match="pool"):
        ops.PagedCache.from_tensors(torch.zeros(2, 4, 2, 16, 64), i, i.view(4, 1), i)
    with pytest.raises(ValueError, match="positive"):
        ops.PagedCache(1, 2, 64, 0, 16, 4, 64, device="cpu")


def attn(c, **kw):
    f = dict(cache=ctypes.pointer(c) if c is not None else None, layer=0, n_head=6, n_query=1, n_seq=2, n_group=1,
             max_shared=20, max_own=30, scale=0.125, q=P, out=P, q_stride=384, out_stride=384, rows=P, group_start=P, shared=P,
             work=P, work_bytes=1 << 40)
    f.update(kw)
    return _lib.AttnShared(**f)


@pytest.mark.parametrize("kw,text", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(n_head=4), "n_head"), (dict(n_head=0), "n_head"),
    (dict(n_query=0), "n_query"), (dict(n_query=4097), "n_query"), (dict(n_seq=0), "n_seq"), (dict(n_seq=65537), "n_seq"),
    (dict(n_group=0), "n_group"), (dict(n_seq=65536, n_query=4096), "2^24"), (dict(max_shared=-1), "max_shared"),
    (dict(max_shared=81), "max_shared"), (dict(max_own=81), "max_own")])
def test_attention_refuses_sizes(kw, text):
    a = ctypes.byref(attn(cache(), **kw))
    refused(workspace(lib().w4j_op_attn_shared_workspace, a)[0], text)
    refused(lib().w4j_op_attn_shared(a, None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(rows=None), "null"), (dict(group_start=None), "null"),
    (dict(shared=None), "null"), (dict(work=None, n_seq=100), "work"), (dict(q_stride=376), "strides"), (dict(out_stride=388), "strides"),
    (dict(q=P + 8), "aligned"), (dict(out=P + 2), "aligned"), (dict(work=P + 8, n_seq=100), "work"),
    (dict(work_bytes=64, n_seq=100), "work"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale")])
def test_attention_refuses_arguments(kw, text):
    refused(lib().w4j_op_attn_shared(ctypes.byref(attn(cache(), **kw)), None), text)


def test_attention_refuses_a_bad_cache():
    for kw, text in BAD_CACHES + BAD_POINTERS:
        refused(lib().w4j_op_attn_shared(ctypes.byref(attn(cache(**kw))), None), text)
    refused(lib().w4j_op_attn_shared(ctypes.byref(attn(None)), None), "null")
    refused(lib().w4j_op_attn_shared(None, None), "null")


def quantize(device=0, x=P, x_type=GGML_F32, m=2, k=100, ldx=100, g=None, b=None, q=P, ldq=112, scale=P):
    return lib().w4j_op_quantize_rows(device, x, x_type, m, k, ldx, g, b, q, ldq, scale, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"), (dict(x_type=8), "x_type"), (dict(m=0), "shape"),
    (dict(k=0, ldq=16), "shape"), (dict(k=-3), "shape"), (dict(ldx=99), "ldx"), (dict(ldq=96), "ldq"), (dict(ldq=104), "ldq"),
    (dict(q=P + 8), "ldq"), (dict(x=P + 2), "aligned"), (dict(x=P + 1, x_type=GGML_F16), "aligned"), (dict(scale=P + 2), "aligned"),
    (dict(g=P), "gamma"), (dict(b=P), "gamma")])
def test_quantize_refusals(kw, text):
    refused(quantize(**kw), text)


def linear(device=0, x=P, ldx=112, xs=P, m=2, k=100, w=P, ldw=112, ws=P, n=30, bias=None, epilogue=0, y=P, y_type=GGML_F32, ldy=30):
    return lib().w4j_op_linear_i8(device, x, ldx, xs, m, k, w, ldw, ws, n, bias, epilogue, y, y_type, ldy, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(xs=None), "null"), (dict(w=None), "null"), (dict(ws=None), "null"), (dict(y=None), "null"),
    (dict(y_type=8), "y_type"), (dict(m=0), "shape"), (dict(n=0, ldy=0), "shape"), (dict(k=0), "shape"), (dict(m=(1 << 24) + 1), "shape"),
    (dict(m=1 << 20, n=1 << 20, ldy=1 << 20), "2^38"), (dict(k=131057, ldx=131072, ldw=131072), "131056"), (dict(ldx=96), "rows"), (dict(ldw=104), "rows"), (dict(x=P + 8), "aligned"),
    (dict(w=P + 4), "aligned"), (dict(ldy=29), "ldy"), (dict(y=P + 2), "aligned"), (dict(epilogue=3), "epilogue"),
    (dict(epilogue=-1), "epilogue")])
def test_linear_refusals(kw, text):
    refused(linear(**kw), text)


def layer(device=0, x=P, x_type=GGML_F32, ldx=100, g=None, b=None, m=9, k=100, w=P, ldw=112, ws=P, n=30, bias=None, epilogue=0, y=P,
          y_type=GGML_F32, ldy=30, work=P, work_bytes=9 * 116):
    return lib().w4j_op_linear_i8_layer(device, x, x_type, ldx, g, b, m, k, w, ldw, ws, n, bias, epilogue, y, y_type, ldy, work,
                                        work_bytes, None)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(ws=None), "null"), (dict(y=None), "null"), (dict(x_type=8), "x_type"),
    (dict(y_type=2), "y_type"), (dict(m=0), "shape"), (dict(n=0), "shape"), (dict(k=0), "shape"), (dict(ldx=99), "ldx"),
    (dict(g=P), "gamma"), (dict(k=131057, ldx=131057, ldw=131072, work_bytes=1 << 30), "131056"), (dict(ldw=104), "rows"),
    (dict(w=P + 8), "aligned"), (dict(ldy=29), "ldy"), (dict(y=P + 2), "aligned"), (dict(x=P + 2), "aligned"),
    (dict(epilogue=3), "epilogue"), (dict(work=None), "work"), (dict(work=P + 4), "work"), (dict(work_bytes=9 * 116 - 1), "work")])
def test_layer_refusals(kw, text):
    refused(layer(**kw), text)


def test_layer_workspace():
    w = lib().w4j_op_linear_i8_layer_workspace
    for m, k, n in ((9, 100, 9 * (112 + 4)), (1, 1280, 0), (4, 380, 0), (2, 1280, 2 * 1284), (1, 40000, 40004), (5, 100, 5 * (112 + 4)), (8, 7000, 8 * (7008 + 4))):
        assert workspace(w, m, k) == (W4J_OK, n)
    for m, k in ((0, 1), (1, 0), (1, 131057), ((1 << 24) + 1, 1)):
        refused(workspace(w, m, k)[0], "shape")
    refused(w(1, 1, None), "null")


def test_a_few_short_rows_need_no_scratch():
    w = lib().w4j_op_attn_shared_workspace
    assert workspace(w, ctypes.byref(attn(cache()))) == (W4J_OK, 0)
    assert workspace(w, ctypes.byref(attn(cache(), n_seq=100)))[1] > 0
    # rows may outgrow max_own, 0 included: parts need their scratch all the same
    assert workspace(w, ctypes.byref(attn(cache(), n_seq=200, max_shared=0, max_own=0)))[1] > 0


def test_scratch_stays_in_proportion():
    """However long the rows may be, their pieces are not many times more than the device takes at once."""
    w = lib().w4j_op_attn_shared_workspace
    c = cache(page_tokens=1024, table_width=1 << 20, n_pages=1000)
    one = workspace(w, ctypes.byref(attn(c, n_seq=1, max_shared=0, max_own=1 << 30)))[1]
    many = workspace(w, ctypes.byref(attn(c, n_seq=60000, max_shared=0, max_own=1 << 30)))[1]
    assert 0 < one < 64 << 20
    assert 0 < many <= 60000 * 6 * 66 * 4
    both = workspace(w, ctypes.byref(attn(c, n_seq=2, max_shared=1 << 30, max_own=1 << 30)))[1]
    assert 0 < both < 256 << 20


def test_the_hook_for_waits_refuses_negative_counts():
    refused(lib().w4j_test_attn_shared_waits_run_out(-1), "n_calls")
    assert lib().w4j_test_attn_shared_waits_run_out(0) == W4J_OK


@pytest.mark.parametrize("off", [1, 2, 3])
def test_arrays_of_32_bit_numbers_are_aligned(off):
    """The kernels read them as such; an address between two numbers would be a fault of the device."""
    L, bad, c = lib(), P + off, ctypes.byref(cache())
    for name in ("ref", "table", "len", "status"):
        other = cache(**{name: bad})
        refused(L.w4j_op_pages_free(ctypes.byref(other), P, 1, None), "aligned")
        refused(L.w4j_op_pages_compact(ctypes.byref(other), None, None), "aligned")
        refused(L.w4j_op_attn_shared(ctypes.byref(attn(other)), None), "aligned")
    for a, b in ((bad, P), (P, bad)):
        refused(L.w4j_op_pages_extend(c, a, b, 1, None), "aligned")
        refused(L.w4j_op_pages_write(c, 0, a, b, 1, P, 192, P, 192, 1, None), "aligned")
        refused(L.w4j_op_pages_fork(c, a, b, 1, None), "aligned")
    refused(L.w4j_op_pages_free(c, bad, 1, None), "aligned")
    refused(L.w4j_op_pages_compact(c, bad, None), "aligned")
    for name in ("rows", "group_start", "shared"):
        refused(L.w4j_op_attn_shared(ctypes.byref(attn(cache(), **{name: bad})), None), "aligned")
    for kw in (dict(g=bad, b=P), dict(g=P, b=bad)):
        refused(quantize(**kw), "aligned")
        refused(layer(**kw), "aligned")
    for kw in (dict(ws=bad), dict(bias=bad)):
        refused(linear(**kw), "aligned")
        refused(layer(**kw), "aligned")
    refused(linear(xs=bad), "aligned")
