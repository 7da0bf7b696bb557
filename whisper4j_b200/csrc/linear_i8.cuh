// linear_i8.cuh — arguments of the 8-bit integer Linear (k_linear_i8.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace w4j {

// `type`: of x or y, a GGML type number (F32, F16 or BF16)
struct QuantizeArgs {
    const void *x;
    int type, M, K;
    long long ldx;
    const float *ln_g, *ln_b;  // both or none
    int8_t *q;
    long long ldq;
    float *scale;
};

struct LinearI8Args {
    const int8_t *x, *w;
    long long ldx, ldw;
    const float *xs, *ws, *bias;
    int M, N, K, epilogue, type;
    void *y;
    long long ldy;
};

cudaError_t launch_quantize_rows(const QuantizeArgs &a, cudaStream_t s);
cudaError_t launch_linear_i8(const LinearI8Args &a, cudaStream_t s);

// both in one; `work`: linear_i8_layer_work bytes (0 for a few rows, which take one launch)
size_t linear_i8_layer_work(int M, int K);
cudaError_t launch_linear_i8_layer(LinearI8Args a, QuantizeArgs q, void *work, cudaStream_t s);

}  // namespace w4j
