// k_linear_i8.cu — a Linear layer in 8-bit integers: rows quantised by their largest magnitude, the product in
// exact 32-bit integers on the 5th-generation tensor cores, one scale for each row and each output channel.
//
//   s_m = max_k |x_mk| / 127,  q_mk = round(x_mk / s_m),  y_mn = act(s_m t_n sum_k q_mk w_nk + b_n)
#include <cuda_bf16.h>
#include <cudaTypedefs.h>

#include "host_api.cuh"
#include "linear_i8.cuh"
#include "tc_common.cuh"

namespace w4j {

namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---------------------------------------------------------------------------
// rows to 8 bits: a block per row, eight neighbouring elements per thread and step, held in registers
// between the passes (sum, squares, largest magnitude, quotients) where the row fits.  Bound by HBM for
// many rows and by the latency of its block reductions for few.
// ---------------------------------------------------------------------------
constexpr int kQMax = 256;

// Eight elements from k on (zeros behind K).
template <typename T>
__device__ __forceinline__ void load8(const T *x, int k, int K, bool vec, float (&v)[8]) {
    if (vec && k + 8 <= K) {
        T t[8];
#pragma unroll
        for (size_t i = 0; i < sizeof(T) / 2; ++i)
            reinterpret_cast<uint4 *>(t)[i] = __ldg(reinterpret_cast<const uint4 *>(x + k) + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f32<T>(x[k + i]) : 0.f;
    }
}

template <typename Op>
__device__ __forceinline__ float block_reduce(float v, float *sm, Op op) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (blockDim.x == 32) return v;
    __syncthreads();  // the last call's numbers have been read
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sm[0];
    for (int w = 1; w < (int)blockDim.x / 32; ++w) v = op(v, sm[w]);
    return v;
}

// The whole number nearest to x / s, ties to even, by the exact quotient: r from the rounded reciprocal is at most
// one off, and x - r s, exact in one FMA wherever it matters, says on which side of a half x / s lies.  Within
// +-127: a subnormal scale may have been rounded far down.
__device__ __forceinline__ int nearest(float x, float s, float inv) {
    float r = rintf(x * inv);
    const float e = fmaf(-r, s, x), h = 0.5f * s;
    if (fabsf(e) > h || (fabsf(e) == h && ((int)r & 1))) r += e > 0.f ? 1.f : -1.f;
    return min(127, max(-127, (int)r));
}

// C: steps held in registers, 0: the row is read again in every pass
template <typename T, int C>
__global__ void __launch_bounds__(kQMax) k_quantize_rows(QuantizeArgs a) {
    __shared__ float sm[kQMax / 32];
    pdl_wait();
    pdl_trigger();
    const T *x = reinterpret_cast<const T *>(a.x) + (long long)blockIdx.x * a.ldx;
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0;
    const int step = blockDim.x * 8, k0 = threadIdx.x * 8, K = a.K;
    float v[C ? C : 1][8];
    if (C) {
#pragma unroll
        for (int c = 0; c < C; ++c) load8(x, k0 + c * step, K, vec, v[c]);
    }
    // f(k, eight elements): over the row
    auto pass = [&](auto f) {
        if (C) {
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (k0 + c * step < K) f(k0 + c * step, v[c]);
        } else {
            for (int k = k0; k < K; k += step) {
                load8(x, k, K, vec, v[0]);
                f(k, v[0]);
            }
        }
    };
    auto add = [](float p, float q) { return p + q; };
    float mean = 0.f, rstd = 1.f;
    if (a.ln_g) {
        float sum = 0.f, sq = 0.f;
        pass([&](int, float(&e)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += e[i];
        });
        mean = block_reduce(sum, sm, add) / K;
        pass([&](int k, float(&e)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < K) sq += (e[i] - mean) * (e[i] - mean);
        });
        rstd = 1.f / sqrtf(block_reduce(sq, sm, add) / K + 1e-5f);
    }
    auto norm = [&](int k, float(&e)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            e[i] = k + i < K ? (e[i] - mean) * rstd * __ldg(a.ln_g + k + i) + __ldg(a.ln_b + k + i) : 0.f;
    };
    float top = 0.f;
    bool odd = false;  // an infinity or a NaN
    pass([&](int k, float(&e)[8]) {
        if (a.ln_g) norm(k, e);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            top = fmaxf(top, fabsf(e[i]));
            odd |= !(fabsf(e[i]) <= 3.4028234e38f);
        }
    });
    top = block_reduce(odd ? INFINITY : top, sm, [](float p, float q) { return fmaxf(p, q); });
    const bool good = top <= 3.4028234e38f;
    const float s = __fdiv_rn(top, 127.f);
    // where the scale's reciprocal or half would not be normal, x and s are taken times 2^64: the same quotient
    const float up = s < 1e-30f ? 18446744073709551616.f : 1.f, su = s * up, inv = __fdiv_rn(1.f, su);
    if (threadIdx.x == 0) a.scale[blockIdx.x] = good ? s : __int_as_float(0x7fffffff);
    int8_t *q = a.q + (long long)blockIdx.x * a.ldq;
    auto store = [&](int k, float(&e)[8]) {
        if (a.ln_g && !C) norm(k, e);
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = good && s > 0.f && k + i < K ? nearest(e[i] * up, su, inv) : 0;
            w[i / 4] |= (uint32_t)(r & 0xff) << (i % 4 * 8);
        }
        *reinterpret_cast<uint2 *>(q + k) = make_uint2(w[0], w[1]);
    };
    pass(store);
    // the rest up to a multiple of 16 is zero: a product may read it
    if (threadIdx.x == 0 && K % 16 && K % 16 <= 8) *reinterpret_cast<uint2 *>(q + K / 16 * 16 + 8) = make_uint2(0, 0);
}

template <typename T>
cudaError_t quantize(const QuantizeArgs &a, cudaStream_t s) {
    const int units = (a.K + 7) / 8, c = (units + kQMax - 1) / kQMax;
    const int held = c <= 1 ? 1 : c <= 2 ? 2 : c <= 4 ? 4 : 0;
    const int threads = held ? (units + held - 1) / held : kQMax, block = (threads + 31) / 32 * 32;
    switch (held) {
        case 1: return launch_after(k_quantize_rows<T, 1>, a.M, block, 0, s, 1, a);
        case 2: return launch_after(k_quantize_rows<T, 2>, a.M, block, 0, s, 1, a);
        case 4: return launch_after(k_quantize_rows<T, 4>, a.M, block, 0, s, 1, a);
        default: return launch_after(k_quantize_rows<T, 0>, a.M, block, 0, s, 1, a);
    }
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------
// One output from its integer sum (exact: |sum| <= 2^14 K < 2^31).  GELU in its tanh form, as
// v / (1 + exp(-2 u)): no cancellation, and the right limits where the exponential leaves its range.
template <typename T>
__device__ __forceinline__ void finish(const LinearI8Args &a, int acc, float xs, float ws, float b, T *y) {
    float v = (float)acc * xs * ws + b;
    if (a.epilogue == 1) {
        const float u = 0.7978845608f * (v + 0.044715f * v * v * v);
        v = v / (1.f + __expf(-2.f * u));
    } else if (a.epilogue == 2) {
        v += to_f32<T>(*y);
    }
    *y = from_f32<T>(v);
}

__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// kind::i8: signed 8-bit A and B, both K-major, 32-bit integer accumulator
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// The word at the same place in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ int peer_word(const int *p, int rank) {
    uint32_t at;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

constexpr int kMmThreads = 256, kMmTile = 128, kMmK = 128;  // 128 channels x NT tokens, 128 bytes of k a stage

__host__ __device__ constexpr int mm_stages(int NT) { return NT <= 64 ? 6 : NT <= 128 ? 3 : 4; }
__host__ __device__ constexpr int mm_stage_bytes(int NT) { return (kMmTile + NT) * kMmK; }
__host__ __device__ constexpr size_t mm_smem(int NT) { return (size_t)mm_stages(NT) * mm_stage_bytes(NT) + 1024; }

// A cluster of blocks owns 128 channels x NT tokens; block q of the cluster multiplies a share of k.  The
// channels are the MMA's 128 rows (TMEM lanes), so that a warp's store of one token's column is one contiguous run
// of y, and a lane keeps its channel's scale and bias in registers.
template <int NT, typename T>
__global__ void __launch_bounds__(kMmThreads) k_linear_i8(const __grid_constant__ CUtensorMap wmap,
                                                          const __grid_constant__ CUtensorMap xmap, LinearI8Args a, int ks,
                                                          int token_tiles) {
    constexpr int S = mm_stages(NT), kStage = mm_stage_bytes(NT), kCols = NT < 32 ? 32 : NT;
    extern __shared__ unsigned char raw[];
    unsigned char *sm = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[S], empty[S], done;
    __shared__ uint32_t slot;
    __shared__ int failed, issued;
    __shared__ float xs[NT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int q = blockIdx.x % ks, tile = blockIdx.x / ks;
    const int n0 = tile / token_tiles * kMmTile, m0 = tile % token_tiles * NT;
    const int kb_all = (a.K + kMmK - 1) / kMmK, kb0 = q * kb_all / ks, kb1 = (q + 1) * kb_all / ks, nk = kb1 - kb0;
    if (tid == 0) {
        for (int i = 0; i < S; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 1);
        mbar_init(&done, 1);
        fence_mbar_init();
        failed = issued = 0;
    }
    pdl_wait();  // before the tensor memory: a kernel that waits must not hold what the one before it may need
    if (warp == 1) tmem_alloc(&slot, kCols), tmem_relinquish();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = slot;
    if (warp == 0 && lane == 0) {
        for (int i = 0; i < nk; ++i) {
            const int st = i % S;
            if (i >= S && !mbar_wait(empty + st, ((i / S) - 1) & 1, &failed)) break;
            mbar_expect_tx(full + st, kStage);
            tma_load_2d(sm + st * kStage, &wmap, (kb0 + i) * kMmK, n0, full + st);
            tma_load_2d(sm + st * kStage + kMmTile * kMmK, &xmap, (kb0 + i) * kMmK, m0, full + st);
            issued = i + 1;
        }
    } else if (warp == 1 && lane == 0) {
        constexpr uint32_t idesc = idesc_i8(kMmTile, NT);
        for (int i = 0; i < nk; ++i) {
            const int st = i % S;
            if (!mbar_wait(full + st, (i / S) & 1, &failed)) break;
            tc_fence_after();
            const uint64_t ad = sw128_desc(smem_u32(sm + st * kStage)), bd = sw128_desc(smem_u32(sm + st * kStage + kMmTile * kMmK));
#pragma unroll
            for (int k = 0; k < kMmK / 32; ++k) umma_i8(tmem, ad + 2 * k, bd + 2 * k, idesc, i || k);
            umma_commit(empty + st);
        }
        umma_commit(&done);
    }
    for (int j = tid; j < NT; j += kMmThreads) xs[j] = m0 + j < a.M ? __ldg(a.xs + m0 + j) : 0.f;
    __syncwarp();
    mbar_wait(&done, 0, &failed);
    tc_fence_after();
    __syncthreads();
    // warps w and w + 4 share lanes 32 (w % 4) .. + 31 and take every other run of 16 tokens
    const int ch = (warp & 3) * 32 + lane, n = n0 + ch;
    const bool in = n < a.N;
    const float ws = in ? __ldg(a.ws + n) : 0.f, b = in && a.bias ? __ldg(a.bias + n) : 0.f;
    T *y = reinterpret_cast<T *>(a.y) + n;
    int *part = reinterpret_cast<int *>(sm);  // [NT][128], over the stages
    for (int j0 = (warp >> 2) * 16; j0 < NT; j0 += 32) {
        float f[16];
        __syncwarp();
        tmem_ld16(tmem + ((uint32_t)(warp & 3) << 21) + j0, f);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int acc = __float_as_int(f[j]), m = m0 + j0 + j;
            if (ks > 1)
                part[(j0 + j) * kMmTile + ch] = acc;
            else if (in && m < a.M)
                finish<T>(a, acc, failed ? NAN : xs[j0 + j], ws, b, y + (long long)m * a.ldy);
        }
    }
    tc_fence_before();
    if (ks > 1) {  // token j of the tile is added up by block j % ks
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        int lost = 0;
        for (int r = 0; r < ks; ++r) lost |= peer_word(&failed, r);
        for (int j = q + (tid >> 7) * ks; j < NT; j += 2 * ks) {
            const int m = m0 + j, c = tid & 127;
            if (m >= a.M) break;
            int acc = 0;
            for (int r = 0; r < ks; ++r) acc += peer_word(part + j * kMmTile + c, r);
            const int nn = n0 + c;
            if (nn < a.N)
                finish<T>(a, acc, lost ? NAN : xs[j], __ldg(a.ws + nn), a.bias ? __ldg(a.bias + nn) : 0.f,
                          reinterpret_cast<T *>(a.y) + (long long)m * a.ldy + nn);
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    __syncthreads();
    if (failed && tid == 0) drain_ring(full, S, issued);
    if (warp == 1) tc_fence_after(), tmem_dealloc(tmem, kCols);
}

// [box rows x 128 bytes] boxes of a row-major 8-bit matrix, 128-byte swizzle; reads beyond rows or columns give zeros
bool tmap_i8(CUtensorMap *m, const int8_t *base, long long rows, int cols, long long ld, int box) {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult r;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) == cudaSuccess &&
                        r == cudaDriverEntryPointSuccess;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ok ? p : nullptr);
    }();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t boxes[2] = {(cuuint32_t)kMmK, (cuuint32_t)box}, estr[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(base), dims, strides, boxes, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NT, typename T>
cudaError_t product(const LinearI8Args &a, cudaStream_t s) {
    const int k16 = (a.K + 15) / 16 * 16, kb = (a.K + kMmK - 1) / kMmK;
    alignas(64) CUtensorMap wmap, xmap;
    if (!tmap_i8(&wmap, a.w, a.N, k16, a.ldw, kMmTile) || !tmap_i8(&xmap, a.x, a.M, k16, a.ldx, NT))
        return cudaErrorInvalidValue;
    const long long token_tiles = (a.M + NT - 1) / NT, tiles = (long long)((a.N + kMmTile - 1) / kMmTile) * token_tiles;
    // k is split while the tiles leave SMs idle and every block keeps two stages of k
    int ks = 1;
    while (ks < 8 && tiles * ks * 2 <= 148 && kb >= 4 * ks) ks *= 2;
    cudaError_t e = allow_smem<k_linear_i8<NT, T>>(mm_smem(NT));
    if (e != cudaSuccess) return e;
    return launch_after(k_linear_i8<NT, T>, (unsigned)(tiles * ks), kMmThreads, mm_smem(NT), s, ks, wmap, xmap, a, ks,
                        (int)token_tiles);
}

template <typename T>
cudaError_t product(const LinearI8Args &a, cudaStream_t s) {
    if (a.M <= 16) return product<16, T>(a, s);
    if (a.M <= 32) return product<32, T>(a, s);
    if (a.M <= 64) return product<64, T>(a, s);
    return product<128, T>(a, s);
}

}  // namespace

cudaError_t launch_quantize_rows(const QuantizeArgs &a, cudaStream_t s) {
    return a.type == W4J_GGML_F32 ? quantize<float>(a, s) : a.type == W4J_GGML_F16 ? quantize<__half>(a, s)
                                                                                  : quantize<__nv_bfloat16>(a, s);
}

cudaError_t launch_linear_i8(const LinearI8Args &a, cudaStream_t s) {
    return a.type == W4J_GGML_F32 ? product<float>(a, s) : a.type == W4J_GGML_F16 ? product<__half>(a, s)
                                                                                 : product<__nv_bfloat16>(a, s);
}

}  // namespace w4j
