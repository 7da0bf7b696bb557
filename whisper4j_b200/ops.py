"""Op-level operators over torch tensors, for hosts that drive their own decode loop.

Thin bindings of the ``w4j_op_*`` entry points in include/whisper4j_cuda.h: they check what a tensor knows
(type, device, layout, shape), hand over the current stream of the tensors' device and allocate outputs and
scratch with torch's allocator, so calls can be captured into CUDA graphs.  Nothing is synchronised.  There are no
gradients: while they are recorded, a tensor that requires one is refused.  A refused
argument is a ValueError; what only the device can see (a row named twice, no free page) raises a bit of the
cache's ``status``, which ``PagedCache.check`` reads.

    PagedCache     a key/value cache of pages that rows (beams, re-decodes of a window) share
    quantize_rows  rows to 8-bit integers, a scale for each
    Int8Linear     a Linear layer in 8-bit integers

A decode step lasts tens of microseconds, so the checks are written to cost little: messages are put together
only where a check fails.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import GGML_BF16, GGML_F16, GGML_F32, AttnShared, IllegalStateError, Pages, check

_TYPES = {torch.float32: GGML_F32, torch.float16: GGML_F16, torch.bfloat16: GGML_BF16}
_INT32 = torch.int32
_STATUS = {_lib.PAGES_BAD_ROW: "a row is out of range or named twice", _lib.PAGES_FULL: "too few free pages",
           _lib.PAGES_TOO_LONG: "a row would outgrow its table",
           _lib.PAGES_BAD_START: "start does not ascend from 0 or does not fit the rows",
           _lib.PAGES_BAD_PAGE: "a table entry names no held page",
           _lib.PAGES_BAD_SHARED: "a shared length is over max_shared or over what a row's queries see",
           _lib.PAGES_TIMEOUT: "a wait inside a kernel ran out"}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _no_gradient(name):
    """Of a tensor that requires a gradient."""
    if torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and this operator has none: call it under torch.no_grad()")


# autograd has to hear of tensors that a call changes through their addresses
_changed = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version


def _shape(t):
    return f"{t.dtype} {tuple(t.shape)} strides {tuple(t.stride())} on {t.device}"


class PagedCache:
    """Keys and values of ``n_rows`` sequences on pages of ``page_tokens`` tokens, ``n_layer`` layers deep.

    pool (2 n_layer, n_pages, n_kv_head, page_tokens, head_dim) float16 or bfloat16; ref (n_pages,), table
    (n_rows, width), len (n_rows,) and status (1,) int32: the tensors are the cache's state and may be read at any
    time.  Row and token counts come as int32 tensors on the cache's device: ``rows`` names distinct rows and
    ``start`` (one longer, from 0, ascending) deals tokens to them, token start[i] .. start[i + 1] - 1 to rows[i].
    """

    def __init__(self, n_layer, n_kv_head, head_dim, n_pages, page_tokens, n_rows, max_tokens, dtype=torch.float16,
                 device="cuda"):
        _need(min(n_layer, n_kv_head, head_dim, n_pages, page_tokens, n_rows, max_tokens) > 0, "sizes must be positive")
        width = -(-max_tokens // page_tokens)
        z = dict(dtype=torch.int32, device=device)
        self._adopt(torch.zeros(2 * n_layer, n_pages, n_kv_head, page_tokens, head_dim, dtype=dtype, device=device),
                    torch.zeros(n_pages, **z), torch.zeros(n_rows, width, **z), torch.zeros(n_rows, **z))

    @classmethod
    def from_tensors(cls, pool, ref, table, len):
        """A cache over state that exists already (ref, table and len consistent with one another)."""
        cache = cls.__new__(cls)
        cache._adopt(pool, ref, table, len)
        return cache

    def _adopt(self, pool, ref, table, length):
        _need(pool.dim() == 5 and pool.shape[0] % 2 == 0 and pool.is_contiguous() and pool.dtype in
              (torch.float16, torch.bfloat16),
              "pool must be a contiguous (2 n_layer, n_pages, n_kv_head, page_tokens, head_dim) float16 or bfloat16 tensor")
        _need(pool.is_cuda, "a paged cache lives on a CUDA device")
        _need(not pool.requires_grad, "a paged cache holds no gradients")
        self.pool, self.ref, self.table, self.len, self.device = pool, ref, table, length, pool.device
        self.dtype, self._index = pool.dtype, pool.device.index
        self.n_layer, self.n_rows = pool.shape[0] // 2, length.numel()
        self.n_kv_head, self.page_tokens, self.head_dim = pool.shape[2:]
        self._head_strides, self._pools = (self.head_dim, 1), (pool,)
        for t, shape, name in ((ref, (pool.shape[1],), "ref"), (length, (self.n_rows,), "len"),
                               (table, (self.n_rows, table.shape[-1]), "table")):
            _need(t.shape == shape and t.dtype == _INT32 and t.device == self.device and t.is_contiguous(),
                  f"{name} must be a contiguous int32 tensor of shape {shape} on {self.device}")
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._lib = _lib.lib()
        c = self._c = Pages(self._index, _TYPES[pool.dtype], self.n_layer, self.n_kv_head, self.head_dim,
                            self.page_tokens, pool.shape[1], self.n_rows, table.shape[1], pool.data_ptr(), ref.data_ptr(),
                            table.data_ptr(), length.data_ptr(), self.status.data_ptr())
        self._ref, self._ptr = ctypes.byref(c), ctypes.pointer(c)
        n_bytes = ctypes.c_size_t()
        check(self._lib.w4j_op_pages_workspace(self._ref, ctypes.byref(n_bytes)))
        c.work_bytes = n_bytes.value
        self._work = torch.zeros(c.work_bytes, dtype=torch.uint8, device=self.device)
        c.work = self._work.data_ptr()
        self._attend_work = None, 0  # sizes of the last attend and its scratch

    def _ints(self, t, name, n=None):
        """Address and length of a contiguous int32 vector on the cache's device."""
        if t.dtype is not _INT32 or t.dim() != 1 or t.get_device() != self._index or not t.is_contiguous() or (
                n is not None and t.numel() != n):
            raise ValueError(f"{name} must be a contiguous int32 vector{'' if n is None else f' of {n}'} on {self.device}, "
                             f"not {_shape(t)}")
        return t.data_ptr(), t.numel()

    def extend(self, rows, start):
        """Grow row rows[i] by start[i + 1] - start[i] tokens; ``write`` brings their keys and values."""
        r, n = self._ints(rows, "rows")
        s, _ = self._ints(start, "start", n + 1)
        check(self._lib.w4j_op_pages_extend(self._ref, r, s, n, _raw_stream(self._index)))

    def write(self, layer, rows, start, k, v):
        """Keys and values (n_tokens, n_kv_head, head_dim) of the tokens that ``extend(rows, start)`` made room for.  Where
        that was refused, nothing is written to its rows."""
        if k.requires_grad or v.requires_grad:
            _no_gradient("k or v")
        r, n = self._ints(rows, "rows")
        s, _ = self._ints(start, "start", n + 1)
        ks, tokens = self._tokens(k, "k"), k.shape[0]
        vs = self._tokens(v, "v")
        _need(v.shape[0] == tokens, "k and v must have the same tokens")
        check(self._lib.w4j_op_pages_write(self._ref, layer, r, s, n, k.data_ptr(), ks, v.data_ptr(), vs, tokens,
                                           _raw_stream(self._index)))
        _changed(self._pools)

    def _tokens(self, t, name):
        """Elements from one token of k or v to the next."""
        shape, stride = t.shape, t.stride()
        if t.dtype is not self.dtype or t.get_device() != self._index or len(shape) != 3 or shape[1] != self.n_kv_head or (
                shape[2] != self.head_dim) or (stride[1:] != self._head_strides and (self.n_kv_head > 1 or stride[2] != 1)):
            raise ValueError(f"{name} must be (n_tokens, {self.n_kv_head}, {self.head_dim}) {self.dtype} with contiguous heads "
                             f"on {self.device}, not {_shape(t)}")
        return stride[0] if shape[0] > 1 else self.n_kv_head * self.head_dim

    def fork(self, dst, src):
        """Row dst[i] becomes what row src[i] was before the call (-1: empty), for all i at once."""
        d, n = self._ints(dst, "dst")
        s, _ = self._ints(src, "src", n)
        check(self._lib.w4j_op_pages_fork(self._ref, d, s, n, _raw_stream(self._index)))
        _changed(self._pools)

    def free(self, rows):
        """Empty the rows; pages that nobody else holds become free."""
        r, n = self._ints(rows, "rows")
        check(self._lib.w4j_op_pages_free(self._ref, r, n, _raw_stream(self._index)))

    def compact(self):
        """Move the held pages to the front of the pool; returns their number as a (1,) int32 tensor."""
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        check(self._lib.w4j_op_pages_compact(self._ref, live.data_ptr(), _raw_stream(self._index)))
        _changed(self._pools)
        return live

    def attend(self, layer, q, rows, group_start, shared, max_shared, max_own, scale=None, out=None):
        """Attention of one layer: q (n_seq, n_query, n_head, head_dim) -> out of the same shape.

        Sequence i is row rows[i]; its queries are the row's last n_query tokens, already written, and see their own
        token and all before it.  Group g is sequences group_start[g] .. group_start[g + 1] - 1, whose rows hold the same
        first shared[g] tokens: they are read once for the group.  max_shared and max_own are upper bounds, known on
        the host, of shared and of the rows' tokens behind it.  ``scale`` defaults to head_dim ** -0.5.
        """
        if q.dim() != 4 or q.dtype is not self.dtype or q.get_device() != self._index or q.shape[3] != self.head_dim:
            raise ValueError(f"q must be (n_seq, n_query, n_head, {self.head_dim}) {self.dtype} on {self.device}, not {_shape(q)}")
        n_seq, n_query, n_head, _ = q.shape
        given = out is not None
        if q.requires_grad or (given and out.requires_grad):
            _no_gradient("q or out")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != self._index:
            raise ValueError(f"out must be like q, not {_shape(out)}")
        if q.numel() == 0:
            return out
        r, _ = self._ints(rows, "rows", n_seq)
        sh, n = self._ints(shared, "shared")
        g, _ = self._ints(group_start, "group_start", n + 1)
        a = AttnShared(self._ptr, layer, n_head, n_query, n_seq, n, max_shared, max_own,
                       self.head_dim ** -0.5 if scale is None else scale, q.data_ptr(), out.data_ptr(),
                       self._query_stride(q, "q"), self._query_stride(out, "out"), r, g, sh)
        ref, sizes = ctypes.byref(a), (n_head, n_query, n_seq, n, max_shared, max_own)
        last, n_bytes = self._attend_work
        if sizes != last:
            size = ctypes.c_size_t()
            check(self._lib.w4j_op_attn_shared_workspace(ref, size))
            n_bytes = size.value
            self._attend_work = sizes, n_bytes
        if n_bytes:
            work = torch.empty(n_bytes, dtype=torch.uint8, device=self.device)
            a.work, a.work_bytes = work.data_ptr(), n_bytes
        check(self._lib.w4j_op_attn_shared(ref, _raw_stream(self._index)))
        if given:
            _changed((out,))
        return out

    @staticmethod
    def _query_stride(t, name):
        """Elements from one query token to the next; sequences follow one another."""
        n_seq, n_query, n_head, dim = t.shape
        if t.is_contiguous():
            return n_head * dim
        stride = t.stride(1) if n_query > 1 else t.stride(0) if n_seq > 1 else n_head * dim
        _need(t.stride(3) == 1 and (n_head == 1 or t.stride(2) == dim) and (n_seq == 1 or t.stride(0) == n_query * stride),
              f"{name} must have contiguous heads and evenly spaced tokens")
        return stride

    def check(self):
        """Wait for the calls so far; IllegalStateError where one of them could not be done (and clear that)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise IllegalStateError("; ".join(text for bit, text in _STATUS.items() if bits & bit))


def _vector(t, n, index, name):
    if t.dtype is not torch.float32 or t.dim() != 1 or t.numel() != n or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 vector of {n} on cuda:{index}, not {_shape(t)}")
    return t.data_ptr()


def _matrix(t, name):
    """Rows, columns and elements from one row to the next of a float matrix with contiguous rows."""
    if t.dim() != 2 or t.dtype not in _TYPES or not t.is_cuda:
        raise ValueError(f"{name} must be a float32, float16 or bfloat16 matrix on a CUDA device, not {_shape(t)}")
    m, n = t.shape
    ld, inner = t.stride()
    if m <= 1:
        ld = n
    if (n > 1 and inner != 1) or ld < n:
        raise ValueError(f"{name} must have contiguous rows, not {_shape(t)}")
    return m, n, ld


def _overlap(a, lda, b, ldb):
    """Whether the bytes that two matrices span have some in common."""
    a0, b0 = a.data_ptr(), b.data_ptr()
    a1 = a0 + ((a.shape[0] - 1) * lda + a.shape[1]) * a.element_size()
    b1 = b0 + ((b.shape[0] - 1) * ldb + b.shape[1]) * b.element_size()
    return a0 < b1 and b0 < a1


def _norm(ln, k, index):
    if ln is None:
        return None, None
    if ln[0].requires_grad or ln[1].requires_grad:
        _no_gradient("gamma or beta")
    return _vector(ln[0], k, index, "gamma"), _vector(ln[1], k, index, "beta")


def quantize_rows(x, ln=None):
    """x (M, K) -> (q, scale): q (M, K rounded up to 16) int8 = round(LayerNorm?(x) / scale), zeros behind K, and
    scale (M,) = max |row| * (1 / 127) in 32 bits.  ``ln`` is (gamma, beta)."""
    m, k, ld = _matrix(x, "x")
    if x.requires_grad:
        _no_gradient("x")
    q = torch.empty(m, (k + 15) // 16 * 16, dtype=torch.int8, device=x.device)
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    if m:
        index = x.get_device()
        g, b = _norm(ln, k, index)
        check(_lib.lib().w4j_op_quantize_rows(index, x.data_ptr(), _TYPES[x.dtype], m, k, ld, g, b, q.data_ptr(), q.shape[1],
                                              scale.data_ptr(), _raw_stream(index)))
    return q, scale


class Int8Linear:
    """y = activation(LayerNorm?(x) W^T + bias) with x quantised row by row in the call and W (N, K) held as int8
    ``weight`` with a float32 ``scale`` for each output channel: numbers to compute with, not parameters that learn."""

    EPILOGUES = {"store": 0, "gelu": 1, "residual": 2}

    def __init__(self, weight, scale, bias=None):
        _need(weight.dim() == 2 and weight.dtype == torch.int8 and weight.is_cuda and 0 not in weight.shape,
              "weight must be an int8 matrix on a CUDA device")
        self.n, self.k = weight.shape
        self.device, self._index = weight.device, weight.get_device()
        k16 = (self.k + 15) // 16 * 16
        if k16 != self.k or not weight.is_contiguous() or weight.data_ptr() % 16:
            # laid out once: rows of a multiple of 16 bytes, zeros behind K
            padded = torch.zeros(self.n, k16, dtype=torch.int8, device=weight.device)
            padded[:, :self.k] = weight
            weight = padded
        scale, bias = scale.detach(), None if bias is None else bias.detach()
        self._scale = _vector(scale, self.n, self._index, "scale")
        self._bias = None if bias is None else _vector(bias, self.n, self._index, "bias")
        self.weight, self.scale, self.bias = weight, scale, bias
        self._weight, self._k16, self._lib = weight.data_ptr(), k16, _lib.lib()
        self._work_bytes = {}  # scratch of a call, by its rows

    @classmethod
    def from_float(cls, weight, bias=None):
        """Quantise a float weight (N, K), channel by channel."""
        q, scale = quantize_rows(weight.detach())
        return cls(q[:, :weight.shape[1]], scale, bias)

    def __call__(self, x, ln=None, epilogue="store", out=None, out_dtype=None):
        """x (M, K) -> (M, N) of ``out_dtype`` (default: x's), or into ``out``, which may overlap x; epilogue "gelu", or
        "residual": out += ..."""
        m, k, ldx = _matrix(x, "x")
        index, code = self._index, self.EPILOGUES.get(epilogue)
        if k != self.k or x.get_device() != index:
            raise ValueError(f"x must be (M, {self.k}) on {self.device}, not {_shape(x)}")
        if code is None:
            raise ValueError(f"epilogue must be one of {sorted(self.EPILOGUES)}")
        given = out is not None
        if x.requires_grad or (given and out.requires_grad):
            _no_gradient("x or out")
        if out is None:
            _need(code != 2, "a residual needs the tensor that it is added to: out")
            _need(out_dtype is None or out_dtype in _TYPES, "out_dtype must be float32, float16 or bfloat16")
            out = torch.empty(m, self.n, dtype=out_dtype or x.dtype, device=x.device)
            ldy = self.n
        else:
            rows, n, ldy = _matrix(out, "out")
            if rows != m or n != self.n or out.get_device() != index or (out_dtype is not None and out.dtype is not out_dtype):
                raise ValueError(f"out must be ({m}, {self.n}) of out_dtype on {self.device}, not {_shape(out)}")
        if not m:
            return out
        g, b = _norm(ln, k, index)
        n_bytes = self._work_bytes.get(m)
        if n_bytes is None:
            size = ctypes.c_size_t()
            check(self._lib.w4j_op_linear_i8_layer_workspace(m, k, size))
            n_bytes = self._work_bytes[m] = size.value
        work = torch.empty(n_bytes, dtype=torch.int8, device=x.device) if n_bytes else None
        if given and not n_bytes and _overlap(x, ldx, out, ldy):
            # one launch would write over rows that some of its blocks have still to read
            q, scale = quantize_rows(x, ln)
            check(self._lib.w4j_op_linear_i8(index, q.data_ptr(), self._k16, scale.data_ptr(), m, k, self._weight, self._k16,
                                             self._scale, self.n, self._bias, code, out.data_ptr(), _TYPES[out.dtype], ldy,
                                             _raw_stream(index)))
            _changed((out,))
            return out
        check(self._lib.w4j_op_linear_i8_layer(index, x.data_ptr(), _TYPES[x.dtype], ldx, g, b, m, k, self._weight, self._k16,
                                               self._scale, self.n, self._bias, code, out.data_ptr(), _TYPES[out.dtype], ldy,
                                               work.data_ptr() if n_bytes else None, n_bytes, _raw_stream(index)))
        if given:
            _changed((out,))
        return out
