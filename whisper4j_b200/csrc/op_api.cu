// op_api.cu — C entry points of the operators for hosts that drive their own loop: the paged cache,
// the attention over it and the 8-bit integer Linear.
// Every argument check that needs no device memory is made here, before any device call.
#include "attn_shared.cuh"
#include "host_api.cuh"
#include "linear_i8.cuh"
#include "pages.cuh"

using namespace w4j;

namespace {

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// arrays of 32-bit numbers
template <typename... P>
bool words(const P *...p) {
    return (aligned(p, 4) && ...);
}

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
    if ((int64_t)c->n_pages * c->n_kv_head * c->page_tokens >= (int64_t)1 << 31)
        return set_err(W4J_ERR_ARG, "%s: a plane of the pool must have fewer than 2^31 head rows", who);
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
    if (!words(c->ref, c->table, c->len, c->status))
        return set_err(W4J_ERR_ARG, "%s: ref, table, len and status must be aligned to their type", who);
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
    if (!words(a, b)) return set_err(W4J_ERR_ARG, "%s: lists must be aligned to their type", who);
    return W4J_OK;
}

extern "C" int w4j_op_pages_workspace(const w4j_pages *c, size_t *bytes) {
    PagesArgs p;
    if (!bytes) return set_err(W4J_ERR_ARG, "w4j_op_pages_workspace: null argument");
    *bytes = 0;
    TRY(pages_sizes(c, "w4j_op_pages_workspace", &p));
    *bytes = pages_work_bytes(p);
    return W4J_OK;
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
    if (!words(n_live)) return set_err(W4J_ERR_ARG, "w4j_op_pages_compact: n_live must be aligned to its type");
    DeviceGuard g(c->device);
    TRY(g.rc());
    CUDA_TRY(launch_pages_compact(p, n_live, stream_of(stream)));
    return W4J_OK;
}

static int attn_sizes(const w4j_attn_shared *x, const char *who, AttnSharedArgs *a) {
    if (!x) return set_err(W4J_ERR_ARG, "%s: null argument", who);
    TRY(pages_sizes(x->cache, who, &a->p));
    if (x->n_head < 1 || x->n_head > 4096 || x->n_head % a->p.n_kv_head)
        return set_err(W4J_ERR_ARG, "%s: n_head = %d must be a multiple of n_kv_head = %d in [1, 4096]", who, x->n_head,
                       a->p.n_kv_head);
    if (x->n_query < 1 || x->n_query > 4096) return set_err(W4J_ERR_ARG, "%s: n_query must be in [1, 4096]", who);
    if (x->n_seq < 1 || x->n_seq > 1 << 16 || x->n_group < 1 || x->n_group > 1 << 16)
        return set_err(W4J_ERR_ARG, "%s: n_seq and n_group must be in [1, 65536]", who);
    if ((int64_t)x->n_seq * x->n_query * x->n_head > 1 << 24)
        return set_err(W4J_ERR_ARG, "%s: n_seq * n_query * n_head must be at most 2^24", who);
    if (x->layer < 0 || x->layer >= a->p.n_layer) return set_err(W4J_ERR_ARG, "%s: layer %d of %d", who, x->layer, a->p.n_layer);
    const int most = a->p.width * a->p.page_tokens;
    if (x->max_shared < 0 || x->max_shared > most || x->max_own < 0 || x->max_own > most)
        return set_err(W4J_ERR_ARG, "%s: max_shared and max_own must be in [0, %d], what a row can hold", who, most);
    a->layer = x->layer, a->n_head = x->n_head, a->rep = x->n_head / a->p.n_kv_head, a->n_query = x->n_query;
    a->n_seq = x->n_seq, a->n_group = x->n_group, a->max_shared = x->max_shared, a->max_own = x->max_own;
    attn_shared_plan(*a);
    return W4J_OK;
}

extern "C" int w4j_op_attn_shared_workspace(const w4j_attn_shared *x, size_t *bytes) {
    AttnSharedArgs a;
    if (!bytes) return set_err(W4J_ERR_ARG, "w4j_op_attn_shared_workspace: null argument");
    *bytes = 0;
    TRY(attn_sizes(x, "w4j_op_attn_shared_workspace", &a));
    *bytes = attn_shared_work_bytes(a);
    return W4J_OK;
}

// Test hook (w4j_test_attn_shared_waits_run_out): calls whose waits still run out.
static std::atomic<int> g_withhold_attn{0};

extern "C" int w4j_test_attn_shared_waits_run_out(int n_calls) {
    if (n_calls < 0) return set_err(W4J_ERR_ARG, "n_calls must be >= 0");
    g_withhold_attn.store(n_calls);
    return W4J_OK;
}

extern "C" int w4j_op_attn_shared(const w4j_attn_shared *x, void *stream) {
    const char *who = "w4j_op_attn_shared";
    AttnSharedArgs a;
    TRY(attn_sizes(x, who, &a));
    TRY(pages_check(x->cache, who, &a.p));
    if (!x->q || !x->out || !x->rows || !x->group_start || !x->shared)
        return set_err(W4J_ERR_ARG, "%s: null argument", who);
    const int64_t token = (int64_t)x->n_head * a.p.head_dim;
    if (x->q_stride < token || x->out_stride < token || x->q_stride % 8 || x->out_stride % 8)
        return set_err(W4J_ERR_ARG, "%s: strides must be multiples of 8 of at least n_head * head_dim", who);
    if (!aligned(x->q, 16) || !aligned(x->out, 16))
        return set_err(W4J_ERR_ARG, "%s: q and out must be 16-byte aligned", who);
    if (!words(x->rows, x->group_start, x->shared))
        return set_err(W4J_ERR_ARG, "%s: rows, group_start and shared must be aligned to their type", who);
    if (!(x->scale > 0) || x->scale > 3e38f) return set_err(W4J_ERR_ARG, "%s: scale must be positive and finite", who);
    const size_t need = attn_shared_work_bytes(a);
    if (need && (!x->work || !aligned(x->work, 16) || x->work_bytes < need))
        return set_err(W4J_ERR_ARG, "%s: work must be 16-byte aligned and hold the %zu bytes that w4j_op_attn_shared_workspace asks for",
                       who, need);
    a.scale_log2 = x->scale * 1.44269504f;
    a.q = x->q, a.out = x->out, a.q_stride = x->q_stride, a.out_stride = x->out_stride;
    a.rows = x->rows, a.group_start = x->group_start, a.shared = x->shared;
    a.part_o = static_cast<float *>(x->work);
    a.part_ml = a.part_o + (size_t)a.n_seq * a.n_query * a.n_head * a.slots * a.p.head_dim;
    int n = g_withhold_attn.load();
    while (n > 0 && !g_withhold_attn.compare_exchange_weak(n, n - 1)) {
    }
    a.withhold = n > 0 ? 16 : 0;
    DeviceGuard g(x->cache->device);
    TRY(g.rc());
    CUDA_TRY(launch_attn_shared(a, x->cache->type == W4J_GGML_BF16, stream_of(stream)));
    return W4J_OK;
}

static bool float_type(int t) { return t == W4J_GGML_F32 || t == W4J_GGML_F16 || t == W4J_GGML_BF16; }

static int check_rows(const char *who, const void *x, int x_type, int M, int K, int64_t ldx, const float *ln_g, const float *ln_b) {
    if (!float_type(x_type)) return set_err(W4J_ERR_ARG, "%s: x_type must be F32 (0), F16 (1) or BF16 (30), not %d", who, x_type);
    if (M < 1 || K < 1 || M > 1 << 24 || K > 1 << 24) return set_err(W4J_ERR_ARG, "%s: bad shape (%d x %d)", who, M, K);
    if (ldx < K) return set_err(W4J_ERR_ARG, "%s: ldx must be at least K", who);
    if (!aligned(x, x_type == W4J_GGML_F32 ? 4 : 2)) return set_err(W4J_ERR_ARG, "%s: x must be aligned to its type", who);
    if ((ln_g == nullptr) != (ln_b == nullptr)) return set_err(W4J_ERR_ARG, "LayerNorm needs both gamma and beta");
    if (!words(ln_g, ln_b)) return set_err(W4J_ERR_ARG, "%s: gamma and beta must be aligned to their type", who);
    return W4J_OK;
}

static int check_product(const char *who, int M, int K, const int8_t *w, int64_t ldw, const float *w_scale, int N, const float *bias,
                         int epilogue, const void *y, int y_type, int64_t ldy) {
    if (!float_type(y_type)) return set_err(W4J_ERR_ARG, "%s: y_type must be F32 (0), F16 (1) or BF16 (30), not %d", who, y_type);
    if (M < 1 || N < 1 || K < 1 || M > 1 << 24 || N > 1 << 24) return set_err(W4J_ERR_ARG, "%s: bad shape (%d x %d x %d)", who, M, K, N);
    if ((int64_t)M * N > (int64_t)1 << 38) return set_err(W4J_ERR_ARG, "%s: M * N must be at most 2^38", who);
    if (K > 131056) return set_err(W4J_ERR_ARG, "%s: K = %d: sums of more than 131056 products may leave 32 bits", who, K);
    if (ldw < K || ldw % 16 || !aligned(w, 16))
        return set_err(W4J_ERR_ARG, "%s: w must be 16-byte aligned with rows a multiple of 16 bytes of at least K apart", who);
    if (ldy < N || !aligned(y, y_type == W4J_GGML_F32 ? 4 : 2))
        return set_err(W4J_ERR_ARG, "%s: y must be aligned to its type with ldy at least N", who);
    if (!words(w_scale, bias)) return set_err(W4J_ERR_ARG, "%s: w_scale and bias must be aligned to their type", who);
    if (epilogue < 0 || epilogue > 2) return set_err(W4J_ERR_ARG, "epilogue must be 0, 1 or 2");
    return W4J_OK;
}

extern "C" int w4j_op_quantize_rows(int device, const void *x, int x_type, int M, int K, int64_t ldx, const float *ln_g,
                                    const float *ln_b, int8_t *q, int64_t ldq, float *scale, void *stream) {
    const char *who = "w4j_op_quantize_rows";
    if (!x || !q || !scale) return set_err(W4J_ERR_ARG, "%s: null argument", who);
    TRY(check_rows(who, x, x_type, M, K, ldx, ln_g, ln_b));
    if (ldq < K || ldq % 16 || !aligned(q, 16))
        return set_err(W4J_ERR_ARG, "%s: q must be 16-byte aligned with ldq a multiple of 16 of at least K", who);
    if (!words(scale)) return set_err(W4J_ERR_ARG, "%s: scale must be aligned to its type", who);
    DeviceGuard g(device);
    TRY(g.rc());
    CUDA_TRY(launch_quantize_rows(QuantizeArgs{x, x_type, M, K, ldx, ln_g, ln_b, q, ldq, scale}, stream_of(stream)));
    return W4J_OK;
}

extern "C" int w4j_op_linear_i8(int device, const int8_t *x, int64_t ldx, const float *x_scale, int M, int K,
                                const int8_t *w, int64_t ldw, const float *w_scale, int N, const float *bias, int epilogue,
                                void *y, int y_type, int64_t ldy, void *stream) {
    const char *who = "w4j_op_linear_i8";
    if (!x || !x_scale || !w || !w_scale || !y) return set_err(W4J_ERR_ARG, "%s: null argument", who);
    TRY(check_product(who, M, K, w, ldw, w_scale, N, bias, epilogue, y, y_type, ldy));
    if (!words(x_scale)) return set_err(W4J_ERR_ARG, "%s: x_scale must be aligned to its type", who);
    if (ldx < K || ldx % 16 || !aligned(x, 16))
        return set_err(W4J_ERR_ARG, "%s: x must be 16-byte aligned with rows a multiple of 16 bytes of at least K apart", who);
    DeviceGuard g(device);
    TRY(g.rc());
    CUDA_TRY(launch_linear_i8(LinearI8Args{x, w, ldx, ldw, x_scale, w_scale, bias, M, N, K, epilogue, y_type, y, ldy},
                              stream_of(stream)));
    return W4J_OK;
}

extern "C" int w4j_op_linear_i8_layer_workspace(int M, int K, size_t *bytes) {
    if (!bytes) return set_err(W4J_ERR_ARG, "w4j_op_linear_i8_layer_workspace: null argument");
    *bytes = 0;
    if (M < 1 || K < 1 || M > 1 << 24 || K > 131056)
        return set_err(W4J_ERR_ARG, "w4j_op_linear_i8_layer_workspace: bad shape (%d x %d)", M, K);
    *bytes = linear_i8_layer_work(M, K);
    return W4J_OK;
}

extern "C" int w4j_op_linear_i8_layer(int device, const void *x, int x_type, int64_t ldx, const float *ln_g, const float *ln_b, int M,
                                      int K, const int8_t *w, int64_t ldw, const float *w_scale, int N, const float *bias,
                                      int epilogue, void *y, int y_type, int64_t ldy, void *work, size_t work_bytes, void *stream) {
    const char *who = "w4j_op_linear_i8_layer";
    if (!x || !w || !w_scale || !y) return set_err(W4J_ERR_ARG, "%s: null argument", who);
    TRY(check_rows(who, x, x_type, M, K, ldx, ln_g, ln_b));
    TRY(check_product(who, M, K, w, ldw, w_scale, N, bias, epilogue, y, y_type, ldy));
    const size_t need = linear_i8_layer_work(M, K);
    if (need && (!work || !aligned(work, 16) || work_bytes < need))
        return set_err(W4J_ERR_ARG, "%s: work must be 16-byte aligned and hold the %zu bytes that w4j_op_linear_i8_layer_workspace asks for",
                       who, need);
    DeviceGuard g(device);
    TRY(g.rc());
    CUDA_TRY(launch_linear_i8_layer(LinearI8Args{nullptr, w, 0, ldw, nullptr, w_scale, bias, M, N, K, epilogue, y_type, y, ldy},
                                    QuantizeArgs{x, x_type, M, K, ldx, ln_g, ln_b, nullptr, 0, nullptr}, work, stream_of(stream)));
    return W4J_OK;
}
