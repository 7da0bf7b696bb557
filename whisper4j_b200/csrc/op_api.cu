// op_api.cu — C entry points of the operators for hosts that drive their own loop: the paged cache.
// Every argument check that needs no device memory is made here, before any device call.
#include "host_api.cuh"
#include "pages.cuh"

using namespace w4j;

namespace {

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

cudaStream_t stream_of(void *s) { return reinterpret_cast<cudaStream_t>(s); }

int pages_sizes(const w4j_pages *c, const char *who, PagesArgs *out) {
    if (!c) return set_err(W4J_ERR_ARG, "%s: null cache", who);
    if (c->type != W4J_GGML_F16 && c->type != W4J_GGML_BF16)
        return set_err(W4J_ERR_ARG, "%s: the pool's type must be F16 (1) or BF16 (30), not %d", who, c->type);
    if (c->head_dim != 64 && c->head_dim != 128)
        return set_err(W4J_ERR_ARG, "%s: head_dim must be 64 or 128, not %d", who, c->head_dim);
    if (c->page_tokens < 8 || c->page_tokens > 1024 || c->page_tokens % 8)
        return set_err(W4J_ERR_ARG, "%s: page_tokens must be a multiple of 8 in [8, 1024], not %d", who, c->page_tokens);
    if (c->n_layer < 1 || c->n_layer > 1024 || c->n_kv_head < 1 || c->n_kv_head > 1024)
        return set_err(W4J_ERR_ARG, "%s: n_layer and n_kv_head must be in [1, 1024]", who);
    if (c->n_pages < 1 || c->n_pages > 1 << 21 || c->n_rows < 1 || c->n_rows > 1 << 20)
        return set_err(W4J_ERR_ARG, "%s: n_pages must be in [1, 2^21] and n_rows in [1, 2^20]", who);
    if (c->table_width < 1 || (int64_t)c->table_width * c->page_tokens > 1 << 30)
        return set_err(W4J_ERR_ARG, "%s: table_width must be positive and hold at most 2^30 tokens", who);
    if ((int64_t)c->n_pages * c->n_kv_head * c->page_tokens >= (int64_t)1 << 32)
        return set_err(W4J_ERR_ARG, "%s: a plane of the pool must have fewer than 2^32 head rows", who);
    *out = PagesArgs{c->n_layer, c->n_kv_head, c->head_dim, c->page_tokens, c->n_pages, c->n_rows, c->table_width,
                     c->pool,    c->ref,       c->table,    c->len,         c->status,  static_cast<int *>(c->work)};
    return W4J_OK;
}

}  // namespace

int w4j::pages_check(const w4j_pages *c, const char *who, PagesArgs *out) {
    TRY(pages_sizes(c, who, out));
    if (!c->pool || !c->ref || !c->table || !c->len || !c->status || !c->work)
        return set_err(W4J_ERR_ARG, "%s: a pointer of the cache is null", who);
    if (!aligned(c->pool, 16) || !aligned(c->work, 16))
        return set_err(W4J_ERR_ARG, "%s: pool and work must be 16-byte aligned", who);
    if (c->work_bytes < pages_work_bytes(*out))
        return set_err(W4J_ERR_ARG, "%s: work has %zu bytes, w4j_op_pages_workspace asks for %zu", who, c->work_bytes,
                       pages_work_bytes(*out));
    return W4J_OK;
}

// The cache and a list of n rows; 1 where there is nothing to do.
static int pages_call(const w4j_pages *c, const char *who, const void *a, const void *b, int n, PagesArgs *out) {
    TRY(pages_check(c, who, out));
    if (n < 0 || n > c->n_rows) return set_err(W4J_ERR_ARG, "%s: n = %d rows of a cache of %d", who, n, c->n_rows);
    if (n == 0) return 1;
    if (!a || !b) return set_err(W4J_ERR_ARG, "%s: null argument", who);
    return W4J_OK;
}

extern "C" size_t w4j_op_pages_workspace(const w4j_pages *c) {
    PagesArgs p;
    return pages_sizes(c, "w4j_op_pages_workspace", &p) < 0 ? 0 : pages_work_bytes(p);
}

extern "C" int w4j_op_pages_extend(const w4j_pages *c, const int32_t *rows, const int32_t *start, int n, void *stream) {
    PagesArgs p;
    const int r = pages_call(c, "w4j_op_pages_extend", rows, start, n, &p);
    if (r) return r < 0 ? r : W4J_OK;
    DeviceGuard g(c->device);
    TRY(g.rc());
    CUDA_TRY(launch_pages_extend(p, rows, start, n, stream_of(stream)));
    return W4J_OK;
}

extern "C" int w4j_op_pages_write(const w4j_pages *c, int layer, const int32_t *rows, const int32_t *start, int n,
                                  const void *k, int64_t k_stride, const void *v, int64_t v_stride, int n_tokens,
                                  void *stream) {
    PagesArgs p;
    const int r = pages_call(c, "w4j_op_pages_write", rows, start, n, &p);
    if (r < 0) return r;
    if (layer < 0 || layer >= c->n_layer) return set_err(W4J_ERR_ARG, "w4j_op_pages_write: layer %d of %d", layer, c->n_layer);
    if (n_tokens < 0) return set_err(W4J_ERR_ARG, "w4j_op_pages_write: n_tokens = %d", n_tokens);
    if (r || n_tokens == 0) return W4J_OK;
    if (!k || !v) return set_err(W4J_ERR_ARG, "w4j_op_pages_write: null argument");
    const int64_t token = (int64_t)c->n_kv_head * c->head_dim;
    if (k_stride < token || v_stride < token || k_stride % 8 || v_stride % 8)
        return set_err(W4J_ERR_ARG, "w4j_op_pages_write: strides must be multiples of 8 of at least n_kv_head * head_dim");
    if (!aligned(k, 16) || !aligned(v, 16)) return set_err(W4J_ERR_ARG, "w4j_op_pages_write: k and v must be 16-byte aligned");
    DeviceGuard g(c->device);
    TRY(g.rc());
    CUDA_TRY(launch_pages_write(p, layer, rows, start, n, k, v, k_stride, v_stride, n_tokens, stream_of(stream)));
    return W4J_OK;
}

extern "C" int w4j_op_pages_fork(const w4j_pages *c, const int32_t *dst, const int32_t *src, int n, void *stream) {
    PagesArgs p;
    const int r = pages_call(c, "w4j_op_pages_fork", dst, src, n, &p);
    if (r) return r < 0 ? r : W4J_OK;
    DeviceGuard g(c->device);
    TRY(g.rc());
    CUDA_TRY(launch_pages_fork(p, dst, src, n, stream_of(stream)));
    return W4J_OK;
}

extern "C" int w4j_op_pages_free(const w4j_pages *c, const int32_t *rows, int n, void *stream) {
    PagesArgs p;
    const int r = pages_call(c, "w4j_op_pages_free", rows, rows, n, &p);
    if (r) return r < 0 ? r : W4J_OK;
    DeviceGuard g(c->device);
    TRY(g.rc());
    CUDA_TRY(launch_pages_free(p, rows, n, stream_of(stream)));
    return W4J_OK;
}

extern "C" int w4j_op_pages_compact(const w4j_pages *c, int32_t *n_live, void *stream) {
    PagesArgs p;
    TRY(pages_check(c, "w4j_op_pages_compact", &p));
    DeviceGuard g(c->device);
    TRY(g.rc());
    CUDA_TRY(launch_pages_compact(p, n_live, stream_of(stream)));
    return W4J_OK;
}
