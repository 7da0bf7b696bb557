// pages.cuh — a paged key/value cache as the kernels see it (k_pages.cu, k_attn_shared.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/whisper4j_cuda.h"

namespace w4j {

struct PagesArgs {
    int n_layer, n_kv_head, head_dim, page_tokens, n_pages, n_rows, width;
    void *pool;                      // [2 n_layer][n_pages][n_kv_head][page_tokens][head_dim], 16 bits
    int *ref, *table, *len, *status;
    int *work;
};

int pages_check(const w4j_pages *c, const char *who, PagesArgs *out);  // W4J_OK, or the error it has set (op_api.cu)
size_t pages_work_bytes(const PagesArgs &p);
cudaError_t launch_pages_fork(const PagesArgs &p, const int *dst, const int *src, int n, cudaStream_t s);
cudaError_t launch_pages_extend(const PagesArgs &p, const int *rows, const int *start, int n, cudaStream_t s);
cudaError_t launch_pages_free(const PagesArgs &p, const int *rows, int n, cudaStream_t s);
cudaError_t launch_pages_compact(const PagesArgs &p, int *live, cudaStream_t s);
cudaError_t launch_pages_write(const PagesArgs &p, int layer, const int *rows, const int *start, int n, const void *k,
                               const void *v, long long k_stride, long long v_stride, int n_tokens, cudaStream_t s);

}  // namespace w4j
