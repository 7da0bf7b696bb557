"""Op-level operators over torch tensors, for hosts that drive their own decode loop.

Thin bindings of the ``w4j_op_*`` entry points in include/whisper4j_cuda.h: they check what a tensor knows
(type, device, layout, shape), hand over the current stream of the tensors' device and allocate outputs with
torch's allocator, so calls can be captured into CUDA graphs.  Nothing is synchronised.  A refused argument is
a ValueError; what only the device can see (a row named twice, no free page) raises a bit of the cache's
``status``, which ``PagedCache.check`` reads.

    PagedCache     a key/value cache of pages that rows (beams, re-decodes of a window) share
    quantize_rows  rows to 8-bit integers, a scale for each
    Int8Linear     a Linear layer in 8-bit integers
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import GGML_BF16, GGML_F16, GGML_F32, AttnShared, IllegalStateError, Pages, check, lib

_TYPES = {torch.float32: GGML_F32, torch.float16: GGML_F16, torch.bfloat16: GGML_BF16}
_STATUS = {_lib.PAGES_BAD_ROW: "a row is out of range or named twice", _lib.PAGES_FULL: "too few free pages",
           _lib.PAGES_TOO_LONG: "a row would outgrow its table",
           _lib.PAGES_BAD_START: "start does not ascend from 0 or does not fit the rows",
           _lib.PAGES_BAD_PAGE: "a table entry names no held page",
           _lib.PAGES_BAD_SHARED: "a shared length is over max_shared or over what a row's queries see"}


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _need(ok, what):
    if not ok:
        raise ValueError(what)


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
        self.pool, self.ref, self.table, self.len, self.device = pool, ref, table, length, pool.device
        self.n_layer, self.n_rows = pool.shape[0] // 2, length.numel()
        self.n_kv_head, self.page_tokens, self.head_dim = pool.shape[2:]
        for t, shape, name in ((ref, (pool.shape[1],), "ref"), (length, (self.n_rows,), "len"),
                               (table, (self.n_rows, table.shape[-1]), "table")):
            _need(t.shape == shape, f"{name} must have shape {shape}, not {tuple(t.shape)}")
            self._int32(t, name)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        c = self._c = Pages(self.device.index, _TYPES[pool.dtype], self.n_layer, self.n_kv_head, self.head_dim,
                            self.page_tokens, pool.shape[1], self.n_rows, table.shape[1], pool.data_ptr(), ref.data_ptr(),
                            table.data_ptr(), length.data_ptr(), self.status.data_ptr())
        self._ref = ctypes.byref(c)
        c.work_bytes = lib().w4j_op_pages_workspace(self._ref)
        _need(c.work_bytes, lib().w4j_last_error().decode())
        self._work = torch.empty(c.work_bytes, dtype=torch.uint8, device=self.device)
        c.work = self._work.data_ptr()

    def _int32(self, t, name, n=None):
        _need(t.dtype == torch.int32 and t.device == self.device and t.is_contiguous(),
              f"{name} must be a contiguous int32 tensor on {self.device}")
        _need(n is None or (t.dim() == 1 and t.shape[0] == n), f"{name} must have shape ({n},), not {tuple(t.shape)}")
        return t.data_ptr()

    def _rows(self, t, name):
        _need(t.dim() == 1, f"{name} must be one-dimensional")
        return self._int32(t, name), t.shape[0]

    def extend(self, rows, start):
        """Grow row rows[i] by start[i + 1] - start[i] tokens; ``write`` brings their keys and values."""
        r, n = self._rows(rows, "rows")
        check(lib().w4j_op_pages_extend(self._ref, r, self._int32(start, "start", n + 1), n, _stream(self.device)))

    def write(self, layer, rows, start, k, v):
        """Keys and values (n_tokens, n_kv_head, head_dim) of the tokens that ``extend(rows, start)`` made room for."""
        r, n = self._rows(rows, "rows")
        for t, name in ((k, "k"), (v, "v")):
            _need(t.dtype == self.pool.dtype and t.device == self.device, f"{name} must be {self.pool.dtype} on {self.device}")
            _need(t.dim() == 3 and t.shape[0] == k.shape[0] and t.shape[1:] == (self.n_kv_head, self.head_dim) and
                  t.stride(2) == 1 and (t.stride(1) == self.head_dim or self.n_kv_head == 1),
                  f"{name} must be (n_tokens, {self.n_kv_head}, {self.head_dim}) with contiguous heads")
        check(lib().w4j_op_pages_write(self._ref, layer, r, self._int32(start, "start", n + 1), n, k.data_ptr(),
                                       self._token_stride(k), v.data_ptr(), self._token_stride(v), k.shape[0],
                                       _stream(self.device)))

    def _token_stride(self, t):
        return t.stride(0) if t.shape[0] > 1 else self.n_kv_head * self.head_dim

    def fork(self, dst, src):
        """Row dst[i] becomes what row src[i] was before the call (-1: empty), for all i at once."""
        d, n = self._rows(dst, "dst")
        check(lib().w4j_op_pages_fork(self._ref, d, self._int32(src, "src", n), n, _stream(self.device)))

    def free(self, rows):
        """Empty the rows; pages that nobody else holds become free."""
        r, n = self._rows(rows, "rows")
        check(lib().w4j_op_pages_free(self._ref, r, n, _stream(self.device)))

    def compact(self):
        """Move the held pages to the front of the pool; returns their number as a (1,) int32 tensor."""
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        check(lib().w4j_op_pages_compact(self._ref, live.data_ptr(), _stream(self.device)))
        return live

    def attend(self, layer, q, rows, group_start, shared, max_shared, max_own, scale=None, out=None):
        """Attention of one layer: q (n_seq, n_query, n_head, head_dim) -> out of the same shape.

        Sequence i is row rows[i]; its queries are the row's last n_query tokens, already written, and see their own
        token and all before it.  Group g is sequences group_start[g] .. group_start[g + 1] - 1, whose rows hold the same
        first shared[g] tokens: they are read once for the group.  max_shared and max_own are upper bounds, known on
        the host, of shared and of the rows' tokens behind it.  ``scale`` defaults to head_dim ** -0.5.
        """
        _need(q.dim() == 4 and q.dtype == self.pool.dtype and q.device == self.device,
              f"q must be (n_seq, n_query, n_head, head_dim) {self.pool.dtype} on {self.device}")
        n_seq, n_query, n_head, dim = q.shape
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == q.device, "out must be like q")
        _need(dim == self.head_dim, f"q has heads of {dim} in a cache of {self.head_dim}")
        if q.numel() == 0:
            return out
        r, _ = self._rows(rows, "rows")
        _need(rows.shape[0] == n_seq, f"rows must have shape ({n_seq},)")
        g, n = self._rows(shared, "shared")
        a = AttnShared(ctypes.pointer(self._c), layer, n_head, n_query, n_seq, n, max_shared, max_own,
                       self.head_dim ** -0.5 if scale is None else scale, q.data_ptr(), out.data_ptr(),
                       self._query_stride(q, "q"), self._query_stride(out, "out"), r,
                       self._int32(group_start, "group_start", n + 1), g)
        ref = ctypes.byref(a)
        a.work_bytes = lib().w4j_op_attn_shared_workspace(ref)
        _need(a.work_bytes, lib().w4j_last_error().decode())
        work = torch.empty(a.work_bytes, dtype=torch.uint8, device=self.device)
        a.work = work.data_ptr()
        check(lib().w4j_op_attn_shared(ref, _stream(self.device)))
        return out

    @staticmethod
    def _query_stride(t, name):
        """Elements from one query token to the next; sequences follow one another."""
        n_seq, n_query, n_head, dim = t.shape
        stride = t.stride(1) if n_query > 1 else t.stride(0) if n_seq > 1 else n_head * dim
        _need((dim == 1 or t.stride(3) == 1) and (n_head == 1 or t.stride(2) == dim) and
              (n_seq == 1 or t.stride(0) == n_query * stride), f"{name} must have contiguous heads and evenly spaced tokens")
        return stride

    def check(self):
        """Wait for the calls so far; IllegalStateError where one of them could not be done (and clear that)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise IllegalStateError("; ".join(text for bit, text in _STATUS.items() if bits & bit))


def _vector(t, n, device, name):
    _need(t.dtype == torch.float32 and t.device == device and t.is_contiguous() and t.shape == (n,),
          f"{name} must be a contiguous float32 tensor of shape ({n},) on {device}")
    return t.data_ptr()


def _ld(t):
    """Elements from one row of a matrix to the next."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _matrix(t, name):
    _need(t.dim() == 2 and t.dtype in _TYPES and t.is_cuda, f"{name} must be a float32, float16 or bfloat16 matrix on a CUDA device")
    _need((t.shape[1] == 1 or t.stride(1) == 1) and _ld(t) >= t.shape[1], f"{name} must have contiguous rows")


def quantize_rows(x, ln=None):
    """x (M, K) -> (q, scale): q (M, K rounded up to 16) int8 = round(LayerNorm?(x) / scale), zeros behind K, and
    scale (M,) = max |row| / 127.  ``ln`` is (gamma, beta)."""
    _matrix(x, "x")
    m, k = x.shape
    q = torch.empty(m, (k + 15) // 16 * 16, dtype=torch.int8, device=x.device)
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    if m:
        g, b = (None, None) if ln is None else (_vector(t, k, x.device, "ln") for t in ln)
        check(lib().w4j_op_quantize_rows(x.device.index, x.data_ptr(), _TYPES[x.dtype], m, k, _ld(x), g, b, q.data_ptr(),
                                         q.shape[1], scale.data_ptr(), _stream(x.device)))
    return q, scale


class Int8Linear:
    """y = activation(LayerNorm?(x) W^T + bias) with x quantised row by row in the call and W (N, K) held as int8
    ``weight`` with a float32 ``scale`` for each output channel."""

    EPILOGUES = {"store": 0, "gelu": 1, "residual": 2}

    def __init__(self, weight, scale, bias=None):
        _need(weight.dim() == 2 and weight.dtype == torch.int8 and weight.is_cuda and 0 not in weight.shape,
              "weight must be an int8 matrix on a CUDA device")
        self.n, self.k = weight.shape
        self.device = weight.device
        k16 = (self.k + 15) // 16 * 16
        if k16 != self.k or not weight.is_contiguous() or weight.data_ptr() % 16:
            # laid out once: rows of a multiple of 16 bytes, zeros behind K
            padded = torch.zeros(self.n, k16, dtype=torch.int8, device=weight.device)
            padded[:, :self.k] = weight
            weight = padded
        _vector(scale, self.n, self.device, "scale")
        if bias is not None:
            _vector(bias, self.n, self.device, "bias")
        self.weight, self.scale, self.bias = weight, scale, bias

    @classmethod
    def from_float(cls, weight, bias=None):
        """Quantise a float weight (N, K), channel by channel."""
        q, scale = quantize_rows(weight)
        return cls(q[:, :weight.shape[1]], scale, bias)

    def __call__(self, x, ln=None, epilogue="store", out=None, out_dtype=None):
        """x (M, K) -> (M, N) of ``out_dtype`` (default: x's), or into ``out``; epilogue "gelu", or "residual": out += ..."""
        _matrix(x, "x")
        _need(x.device == self.device and x.shape[1] == self.k, f"x must be (M, {self.k}) on {self.device}")
        _need(epilogue in self.EPILOGUES, f"epilogue must be one of {sorted(self.EPILOGUES)}")
        m = x.shape[0]
        if out is None:
            _need(epilogue != "residual", "a residual needs the tensor that it is added to: out")
            out = torch.empty(m, self.n, dtype=out_dtype or x.dtype, device=self.device)
        _matrix(out, "out")
        _need(out.shape == (m, self.n) and out.device == self.device, f"out must be ({m}, {self.n}) on {self.device}")
        _need(out_dtype is None or out.dtype == out_dtype, "out is not of out_dtype")
        if m:
            q, xs = quantize_rows(x, ln)
            check(lib().w4j_op_linear_i8(self.device.index, q.data_ptr(), q.shape[1], xs.data_ptr(), m, self.k,
                                         self.weight.data_ptr(), self.weight.shape[1], self.scale.data_ptr(), self.n,
                                         None if self.bias is None else self.bias.data_ptr(), self.EPILOGUES[epilogue],
                                         out.data_ptr(), _TYPES[out.dtype], _ld(out), _stream(self.device)))
        return out
