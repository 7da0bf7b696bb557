// k_linear_i8.cu — a Linear layer in 8-bit integers: rows quantised by their largest magnitude, the product in
// exact 32-bit integers on the 5th-generation tensor cores, one scale for each row and each output channel.
//
//   s_m = max_k |x_mk| (1 / 127),  q_mk = round(x_mk / s_m),  y_mn = act(s_m t_n sum_k q_mk w_nk + b_n)
#include <cuda_bf16.h>
#include <cudaTypedefs.h>

#include <type_traits>

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
// rows to 8 bits: a warp per row where there are many rows, else a block, 16 bytes per thread and step, held in
// registers between the passes (sum, squares, largest magnitude, quotients) where the row fits.  12000 rows of 1280
// 32-bit numbers behind a LayerNorm take 24 us, 3.2 TB/s: bound by the passes' instructions and their latency at 24 warps
// an SM, half of what HBM would give.  Packed arithmetic, or the warp's next row fetched ahead at more registers, took as
// long or longer.  Few rows are bound by the latency of the reductions (320 rows of 5120: 3 to 5 us).
// ---------------------------------------------------------------------------
constexpr int kQMax = 1024;

// The 16 bytes of elements from k on; one by one, with zeros behind K, where rows are not whole 16-byte units.
template <typename T, bool WHOLE>
__device__ __forceinline__ void load16(const T *x, int k, int K, float (&v)[16 / sizeof(T)]) {
    constexpr int V = 16 / sizeof(T);
    if (WHOLE) {
        T t[V];
        *reinterpret_cast<uint4 *>(t) = __ldg(reinterpret_cast<const uint4 *>(x + k));
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_f32<T>(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = k + i < K ? to_f32<T>(x[k + i]) : 0.f;
    }
}

template <bool WARP, typename U, typename Op>
__device__ __forceinline__ U row_reduce(U v, U *sm, Op op) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (WARP) return v;
    __syncthreads();  // the last call's numbers have been read
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sm[0];
    for (int w = 1; w < (int)blockDim.x / 32; ++w) v = op(v, sm[w]);
    return v;
}

// A scale is the largest magnitude times this 32-bit number (where it is a multiple of 127 half steps of a 16-bit type,
// many quotients are near ties: everybody who quantises the same rows has to round it alike).
constexpr float kPerStep = 1.f / 127.f;

// The whole number nearest to x / s, ties to even, by the exact quotient: r from the rounded reciprocal is at most
// one off, and x - r s, exact in one FMA wherever it matters, says on which side of a half x / s lies.  Within
// +-127: a subnormal scale may have been rounded far down.
__device__ __noinline__ int nearest(float x, float s, float inv) {
    float r = rintf(x * inv);
    const float e = fmaf(-r, s, x), h = 0.5f * s;
    if (fabsf(e) > h || (fabsf(e) == h && ((int)r & 1))) r += e > 0.f ? 1.f : -1.f;
    return min(127, max(-127, (int)r));
}

// A row's scale s, and its reciprocal.  Where that or s / 2 would not be normal, x and s are taken times `up` = 2^64: the
// same quotient.
struct Step {
    float s, inv, up;
    bool tiny;
};
// Four of them, packed.  Adding 1.5 x 2^23 rounds to the whole number and leaves it in the low byte; `close` where x / s
// lies at or beyond a half from one of them (one in some hundred thousand): there the exact rule has to be asked.
__device__ __forceinline__ uint32_t round4(const float *x, const Step &p, bool &close) {
    const float h = 0.5f * p.s;
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float y = fmaf(x[i], p.inv, 12582912.f);
        t[i] = __float_as_uint(y);
        close |= fabsf(fmaf(12582912.f - y, p.s, x[i])) >= h;
    }
    return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t nearest4(const float *x, const Step &p) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (uint32_t)(nearest(x[i] * p.up, p.s * p.up, p.inv) & 0xff) << (8 * i);
    return w;
}

// C: steps held in registers, 0: any rows, read again in every pass (C > 0: K, x, ldx and a LayerNorm's vectors are whole
// 16-byte units); WARP: a row per warp, else per block
template <typename T, int C, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : kQMax) k_quantize_rows(QuantizeArgs a) {
    constexpr int V = 16 / sizeof(T);
    constexpr bool WHOLE = C > 0;
    __shared__ float sm[kQMax / 32];
    pdl_wait();
    pdl_trigger();
    const int row = WARP ? blockIdx.x * 4 + threadIdx.x / 32 : blockIdx.x, tid = WARP ? threadIdx.x % 32 : threadIdx.x;
    if (row >= a.M) return;
    const T *x = reinterpret_cast<const T *>(a.x) + (long long)row * a.ldx;
    const int step = (WARP ? 32 : blockDim.x) * V, k0 = tid * V, K = a.K;
    float v[C ? C : 1][V];
    if (C) {
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (k0 + c * step < K) load16<T, WHOLE>(x, k0 + c * step, K, v[c]);
    }
    // f(k, the elements from k on): over the row
    auto pass = [&](auto f) {
        if (C) {
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (k0 + c * step < K) f(k0 + c * step, v[c]);
        } else {
            for (int k = k0; k < K; k += step) {
                load16<T, WHOLE>(x, k, K, v[0]);
                f(k, v[0]);
            }
        }
    };
    auto add = [](float p, float q) { return p + q; };
    float mean = 0.f, rstd = 1.f;
    if (a.ln_g) {
        float sum = 0.f, sq = 0.f;
        pass([&](int, float(&e)[V]) {
#pragma unroll
            for (int i = 0; i < V; ++i) sum += e[i];
        });
        mean = row_reduce<WARP>(sum, sm, add) / K;
        pass([&](int k, float(&e)[V]) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (WHOLE || k + i < K) sq += (e[i] - mean) * (e[i] - mean);
        });
        rstd = 1.f / sqrtf(row_reduce<WARP>(sq, sm, add) / K + 1e-5f);
    }
    auto norm = [&](int k, float(&e)[V]) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            float g[4], b[4];
            load16<float, WHOLE>(a.ln_g, k + i, K, g);
            load16<float, WHOLE>(a.ln_b, k + i, K, b);
#pragma unroll
            for (int j = 0; j < 4; ++j) e[i + j] = (e[i + j] - mean) * rstd * g[j] + b[j];  // behind K both are 0
        }
    };
    // the largest magnitude by its bits: an infinity or a NaN is above every number
    uint32_t bits = 0;
    pass([&](int k, float(&e)[V]) {
        if (a.ln_g) norm(k, e);
#pragma unroll
        for (int i = 0; i < V; ++i) bits = max(bits, __float_as_uint(e[i]) & 0x7fffffffu);
    });
    bits = row_reduce<WARP>(bits, reinterpret_cast<uint32_t *>(sm), [](uint32_t p, uint32_t q) { return max(p, q); });
    const bool good = bits < 0x7f800000u;
    const float s = __fmul_rn(__uint_as_float(bits), kPerStep);
    Step p;
    p.s = s, p.tiny = s < 1e-30f, p.up = p.tiny ? 18446744073709551616.f : 1.f, p.inv = __fdiv_rn(1.f, s * p.up);
    const bool any = good && s > 0.f;
    if (tid == 0) a.scale[row] = good ? s : __int_as_float(0x7fffffff);
    int8_t *q = a.q + (long long)row * a.ldq;
    bool close = p.tiny;
    pass([&](int k, float(&e)[V]) {
        if (a.ln_g && !C) norm(k, e);
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const uint32_t w = round4(e + i, p, close);
            *reinterpret_cast<uint32_t *>(q + k + i) = any ? w : 0;  // (zeros behind K: x is 0 there)
        }
    });
    if (close && any)  // one branch for all of the thread's elements
        pass([&](int k, float(&e)[V]) {
            if (a.ln_g && !C) norm(k, e);
#pragma unroll
            for (int i = 0; i < V; i += 4) *reinterpret_cast<uint32_t *>(q + k + i) = nearest4(e + i, p);
        });
    // the rest up to a multiple of 16 is zero: a product may read it
    const int done = (K + V - 1) / V * V, end = (K + 15) / 16 * 16;
    if (tid * 4 < end - done) *reinterpret_cast<uint32_t *>(q + done + tid * 4) = 0;
}

// A warp per row from 8 rows for every SM's scheduler on, where a row fits its registers (12000 rows of 1280 with a
// LayerNorm: 51 us with a block per row, 24 with a warp); fewer rows get as many threads as they have units.
template <typename T>
cudaError_t quantize(const QuantizeArgs &a, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int units = (a.K + V - 1) / V, c = (units + 31) / 32;
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.ln_g) | reinterpret_cast<uintptr_t>(a.ln_b);
    const bool whole = at % 16 == 0 && a.K % V == 0 && a.ldx % V == 0;
    if (a.M >= 148 * 4 * 2 && c <= 16 && whole) {
        const unsigned blocks = (a.M + 3) / 4;
        if (c <= 4) return launch_after<k_quantize_rows<T, 4, true>>(blocks, 128, 0, s, 1, a);
        if (c <= 8) return launch_after<k_quantize_rows<T, 8, true>>(blocks, 128, 0, s, 1, a);
        if (c <= 12) return launch_after<k_quantize_rows<T, 12, true>>(blocks, 128, 0, s, 1, a);
        return launch_after<k_quantize_rows<T, 16, true>>(blocks, 128, 0, s, 1, a);
    }
    const int most = a.M >= 148 * 4 ? 256 : kQMax, held = (units + most - 1) / most;
    const int threads = held <= 4 ? (units + held - 1) / held : most, block = (threads + 31) / 32 * 32;
    if (!whole) return launch_after<k_quantize_rows<T, 0, false>>(a.M, block, 0, s, 1, a);
    if (held == 1) return launch_after<k_quantize_rows<T, 1, false>>(a.M, block, 0, s, 1, a);
    if (held == 2) return launch_after<k_quantize_rows<T, 2, false>>(a.M, block, 0, s, 1, a);
    if (held <= 4) return launch_after<k_quantize_rows<T, 4, false>>(a.M, block, 0, s, 1, a);
    return launch_after<k_quantize_rows<T, 0, false>>(a.M, block, 0, s, 1, a);
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint64_t pack(float lo, float hi) {
    return (uint64_t)__float_as_uint(hi) << 32 | __float_as_uint(lo);
}
__device__ __forceinline__ uint64_t both(float v) { return pack(v, v); }
__device__ __forceinline__ float lo(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// GELU of two numbers in its tanh form, as v / (1 + 2^t) with t = -2 log2(e) u: no cancellation, and 0 where 2^t is beyond
// 32 bits (NaN for -inf, as the formula's -inf x 0).  The XU pipe is 46 % busy with them in the pair product; one reciprocal
// for two numbers needs the exponent limited and a select to 0 behind that limit: 106 us instead of 93 for 12000 rows.
__device__ __forceinline__ uint64_t gelu2(uint64_t v) {
    const uint64_t t = mul2(v, fma2(mul2(v, v), both(-0.1029432397f), both(-2.3022081985f)));
    const uint64_t d = add2(pack(ex2(lo(t)), ex2(hi(t))), both(1.f));
    return mul2(v, pack(rcp(lo(d)), rcp(hi(d))));
}
__device__ __forceinline__ float gelu(float v) { return lo(gelu2(both(v))); }
// One output from its integer sum (exact: |sum| <= 2^14 K < 2^31).
template <int EPI>
__device__ __forceinline__ float output(int acc, float xs, float ws, float b) {
    const float v = fmaf((float)acc * xs, ws, b);
    return EPI == 1 ? gelu(v) : v;
}
// Two outputs of one channel.
template <int EPI>
__device__ __forceinline__ uint64_t output2(int a0, int a1, uint64_t xs, uint64_t ws, uint64_t b) {
    const uint64_t v = fma2(mul2(pack((float)a0, (float)a1), xs), ws, b);
    return EPI == 1 ? gelu2(v) : v;
}
template <typename T, int EPI>
__device__ __forceinline__ void finish(int acc, float xs, float ws, float b, T *y) {
    float v = output<EPI>(acc, xs, ws, b);
    if (EPI == 2) v += to_f32<T>(*y);
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

// The same place in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_address(const void *p, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ void peer_store(uint32_t at, int v) {
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                   "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                   "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at)
                 : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

constexpr int kMmThreads = 256, kMmTile = 128, kMmK = 128;  // 128 channels x NT tokens, 128 bytes of k a stage

__host__ __device__ constexpr int mm_stages(int NT) { return NT <= 64 ? 6 : 4; }
__host__ __device__ constexpr int mm_stage_bytes(int NT) { return (kMmTile + NT) * kMmK; }
// the ring, then the sums that the blocks of a cluster hand one another
__host__ __device__ constexpr size_t mm_smem(int NT) { return (size_t)mm_stages(NT) * mm_stage_bytes(NT) + NT * kMmTile * 4 + 1024; }

// A cluster of blocks owns 128 channels x NT tokens; block q of the cluster multiplies a share of k.  The
// channels are the MMA's 128 rows (TMEM lanes), so that a warp's store of one token's column is one contiguous run
// of y, and a lane keeps its channel's scale and bias in registers.  With k split, token j belongs to block j % ks: every
// block stores its sums straight into the owner's shared memory, and after one cluster barrier the owner adds them up
// (fetching them from their makers instead took 15.7 us rather than 13.8 for 320 rows x 5120 x 1280 channels with their
// quantisation).  That product is bound by its operands' way from L2 (39 MB, 5 us), the exchange and the start.
template <int NT, typename T, int EPI>
__global__ void __launch_bounds__(kMmThreads) k_linear_i8(const __grid_constant__ CUtensorMap wmap,
                                                          const __grid_constant__ CUtensorMap xmap, LinearI8Args a, int ks,
                                                          int token_tiles) {
    constexpr int S = mm_stages(NT), kStage = mm_stage_bytes(NT), kCols = NT < 32 ? 32 : NT;
    extern __shared__ unsigned char raw[];
    unsigned char *sm = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[S], empty[S], done;
    __shared__ uint32_t slot;
    __shared__ int failed, issued, lost[8];
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
    if (ks > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this block is there
    pdl_wait();  // before the tensor memory: a kernel that waits must not hold what the one before it may need
    pdl_trigger();
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
    // warps w and w + 4 share lanes 32 (w % 4) .. + 31 and take every other run of tokens
    const int ch = (warp & 3) * 32 + lane, n = n0 + ch;
    const bool in = n < a.N;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    if (ks == 1) {
        const float ws = in ? __ldg(a.ws + n) : 0.f, b = in && a.bias ? __ldg(a.bias + n) : 0.f;
        T *y = reinterpret_cast<T *>(a.y) + n;
        for (int j0 = (warp >> 2) * 16; j0 < NT; j0 += 32) {
            float f[16], v[16];
            __syncwarp();
            tmem_ld16(lanes + j0, f);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = output<EPI>(__float_as_int(f[j]), xs[j0 + j], ws, b);
            T *at = y + (long long)(m0 + j0) * a.ldy;
            if (EPI == 2) {
                T old[16];
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (in && m0 + j0 + j < a.M) old[j] = at[j * a.ldy];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] += to_f32<T>(old[j]);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (in && m0 + j0 + j < a.M) at[j * a.ldy] = from_f32<T>(failed ? NAN : v[j]);
        }
        tc_fence_before();
    } else {
        constexpr int R = NT < 32 ? NT : 32;
        const int shift = __popc(ks - 1), tk = NT >> shift;  // ks is a power of two
        int *sums = reinterpret_cast<int *>(sm + S * kStage);  // [ks][tk][128]
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every block is there
        uint32_t owner[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) owner[r] = peer_address(sums + q * tk * kMmTile + ch, r & (ks - 1));
        for (int j0 = (warp >> 2) * R; j0 < NT; j0 += 2 * R) {
            __syncwarp();
            if (NT < 32) {
                float f[16];
                tmem_ld16(lanes + j0, f);
#pragma unroll
                for (int j = 0; j < 16; ++j) peer_store(owner[j & 7] + ((j0 + j) >> shift) * kMmTile * 4, __float_as_int(f[j]));
            } else {
                uint32_t f[32];
                tmem_ld32(lanes + j0, f);
#pragma unroll
                for (int j = 0; j < 32; ++j) peer_store(owner[j & 7] + ((j0 + j) >> shift) * kMmTile * 4, (int)f[j]);
            }
        }
        if (tid < ks) peer_store(peer_address(lost + q, tid), failed);
        tc_fence_before();
        // what does not depend on the sums, while they are on their way: a thread takes four channels of a token
        constexpr int I = NT * kMmTile / 4 / 2 / kMmThreads < 1 ? 1 : NT * kMmTile / 4 / 2 / kMmThreads;  // at most, with ks = 2
        const int c4 = (tid & 31) * 4, nn = n0 + c4;
        float sc[4], bi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sc[e] = nn + e < a.N ? __ldg(a.ws + nn + e) : 0.f;
            bi[e] = nn + e < a.N && a.bias ? __ldg(a.bias + nn + e) : 0.f;
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        int any = 0;
        for (int r = 0; r < ks; ++r) any |= lost[r];
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int t = (tid >> 5) + i * (kMmThreads / 32), j = t * ks + q;  // token t of this block's
            if (t >= tk || m0 + j >= a.M) break;
            int4 acc = make_int4(0, 0, 0, 0);
            for (int r = 0; r < ks; ++r) {
                const int4 x = *reinterpret_cast<const int4 *>(sums + (r * tk + t) * kMmTile + c4);
                acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
            }
            const int sum[4] = {acc.x, acc.y, acc.z, acc.w};
            T *at = reinterpret_cast<T *>(a.y) + (long long)(m0 + j) * a.ldy + nn;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = output<EPI>(sum[e], any ? NAN : xs[j], sc[e], bi[e]);
                if (EPI == 2 && nn + e < a.N) v[e] += to_f32<T>(at[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (nn + e < a.N) at[e] = from_f32<T>(v[e]);
        }
    }
    __syncthreads();
    if (failed && tid == 0) drain_ring(full, S, issued);
    if (warp == 1) tc_fence_after(), tmem_dealloc(tmem, kCols);
}

// ---------------------------------------------------------------------------
// a few rows: a warp per channel, 16 bytes of its weights per lane and step against MT rows (dp4a), the next steps' weights
// on their way.  Bound by the latency of one trip to HBM and by its launch; no tensor memory, barriers or cluster.
// (One row x 1280 x 3840 channels, weights in L2: 2.6 us, on the tensor cores 4.3.)
// ---------------------------------------------------------------------------
constexpr int kFewWarps = 8;

template <int MT, typename T, int EPI>
__global__ void __launch_bounds__(kFewWarps * 32) k_linear_i8_few(LinearI8Args a) {
    const int n = blockIdx.x * kFewWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31, units = (a.K + 15) / 16;
    pdl_wait();
    pdl_trigger();
    if (n >= a.N) return;
    const uint4 *w = reinterpret_cast<const uint4 *>(a.w + (long long)n * a.ldw);
    const float ws = __ldg(a.ws + n), b = a.bias ? __ldg(a.bias + n) : 0.f;
    int acc[MT] = {};
    constexpr int U = 4;
    for (int u0 = lane; u0 < units; u0 += 32 * U) {
        uint4 v[U];
#pragma unroll
        for (int i = 0; i < U; ++i) v[i] = u0 + 32 * i < units ? __ldg(w + u0 + 32 * i) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (m >= a.M) break;
            const uint4 *x = reinterpret_cast<const uint4 *>(a.x + m * a.ldx);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (u0 + 32 * i >= units) break;
                const uint4 t = __ldg(x + u0 + 32 * i);
                acc[m] = __dp4a((int)v[i].x, (int)t.x, acc[m]), acc[m] = __dp4a((int)v[i].y, (int)t.y, acc[m]);
                acc[m] = __dp4a((int)v[i].z, (int)t.z, acc[m]), acc[m] = __dp4a((int)v[i].w, (int)t.w, acc[m]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int o = 16; o; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
        if (m < a.M && lane == m) finish<T, EPI>(acc[m], __ldg(a.xs + m), ws, b, reinterpret_cast<T *>(a.y) + (long long)m * a.ldy + n);
    }
}

// The whole layer for a few rows in one launch: every block quantises the rows for itself (8, 4 or 2 warps to a row)
// into shared memory while its first channels' weights are on their way.  One row x 1280 x 3840 channels
// takes 3.6 us in a graph, 1.3 TB/s of weights, where two launches take 4.5.
// Longer rows or more of them are quantised once instead, by a launch of their own (in a graph, 1280 x 3840: 2 rows 7.1 us
// against 4.6, 4 rows 17 against 5.6; 5120 x 1280: 1 row 9.3 against 6.2); below, a launch saved is 2.5 us of the host's.
constexpr size_t kLayerSmem = 1536;
constexpr int kLayerBlocks = 4;  // to an SM

__device__ __forceinline__ float load1(const void *x, int type, long long i) {
    return type == W4J_GGML_F32 ? __ldg(static_cast<const float *>(x) + i)
           : type == W4J_GGML_F16 ? __half2float(__ldg(static_cast<const __half *>(x) + i))
                                  : __bfloat162float(__ldg(static_cast<const __nv_bfloat16 *>(x) + i));
}

template <int MT, typename T, int EPI>
__global__ void __launch_bounds__(kFewWarps * 32, kLayerBlocks) k_linear_i8_layer(LinearI8Args a, QuantizeArgs in) {
    extern __shared__ __align__(16) int8_t sq[];  // [M][K rounded up to 16]
    __shared__ uint32_t sm[kFewWarps];
    __shared__ float sxs[MT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int K = a.K, units = (K + 15) / 16, k16 = 16 * units;
    int n = blockIdx.x * kFewWarps + warp;
    const int8_t *w = a.w + (long long)n * a.ldw;
    if (n < a.N)  // into L2 only: the weights may be what the kernel before this one writes
        for (int k = lane * 128; k < K; k += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(w + k));
    pdl_wait();
    pdl_trigger();
    constexpr int U = (kLayerSmem + 511) / 512;  // 16-byte units of a channel for each lane
    uint4 v[U];
    auto weights = [&]() {
#pragma unroll
        for (int i = 0; i < U; ++i)
            v[i] = n < a.N && lane + 32 * i < units ? __ldg(reinterpret_cast<const uint4 *>(w) + lane + 32 * i) : make_uint4(0, 0, 0, 0);
    };
    weights();
    // row `row` by `per` warps, E elements of a thread in registers: MT / 2 rows and one more have the longest
    constexpr int per = kFewWarps / MT, nt = 32 * per, E = (kLayerSmem / (MT / 2 + 1) + nt - 1) / nt;
    const int row = warp / per, t = tid % nt, rows = min(MT, a.M);
    const long long x0 = (long long)min(row, rows - 1) * in.ldx;
    float c[E];
#pragma unroll
    for (int e = 0; e < E; ++e) c[e] = t + e * nt < K ? load1(in.x, in.type, x0 + t + e * nt) : 0.f;
    auto pass = [&](auto f) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (t + e * nt < K) f(t + e * nt, c[e]);
    };
    auto reduce = [&](auto r, auto op) {
        using R = decltype(r);
#pragma unroll
        for (int o = 16; o; o >>= 1) r = op(r, __shfl_xor_sync(0xffffffffu, r, o));
        if (per == 1) return r;
        R *to = reinterpret_cast<R *>(sm);
        __syncthreads();
        if (lane == 0) to[warp] = r;
        __syncthreads();
        r = to[row * per];
#pragma unroll
        for (int i = 1; i < per; ++i) r = op(r, to[row * per + i]);
        return r;
    };
    auto add = [](float p, float q) { return p + q; };
    float mean = 0.f, rstd = 1.f;
    if (in.ln_g) {
        float sum = 0.f, sum2 = 0.f;
        pass([&](int, float x) { sum += x; });
        mean = reduce(sum, add) / K;
        pass([&](int, float x) { sum2 += (x - mean) * (x - mean); });
        rstd = 1.f / sqrtf(reduce(sum2, add) / K + 1e-5f);
    }
    auto value = [&](int k, float x) { return in.ln_g ? (x - mean) * rstd * __ldg(in.ln_g + k) + __ldg(in.ln_b + k) : x; };
    uint32_t bits = 0;  // the largest magnitude by its bits: an infinity or a NaN is above every number
    pass([&](int k, float x) { bits = max(bits, __float_as_uint(value(k, x)) & 0x7fffffffu); });
    bits = reduce(bits, [](uint32_t p, uint32_t q) { return max(p, q); });
    const bool good = bits < 0x7f800000u;
    Step p;
    p.s = __fmul_rn(__uint_as_float(bits), kPerStep);
    p.tiny = p.s < 1e-30f, p.up = p.tiny ? 18446744073709551616.f : 1.f, p.inv = __fdiv_rn(1.f, p.s * p.up);
    if (row < rows) {
        if (t == 0) sxs[row] = good ? p.s : __int_as_float(0x7fffffff);
        int8_t *q = sq + row * k16;
        pass([&](int k, float x) {
            x = value(k, x);
            const float y = fmaf(x, p.inv, 12582912.f);
            int r = (int)(__float_as_uint(y) & 0xffu);
            if (p.tiny || fabsf(fmaf(12582912.f - y, p.s, x)) >= 0.5f * p.s) r = nearest(x * p.up, p.s * p.up, p.inv);
            q[k] = (int8_t)(good && p.s > 0.f ? r : 0);
        });
        for (int k = K + t; k < k16; k += nt) q[k] = 0;
    }
    __syncthreads();
    while (n < a.N) {
        int acc[MT] = {};
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (m >= rows) break;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (lane + 32 * i >= units) break;
                const uint4 x = *reinterpret_cast<const uint4 *>(sq + m * k16 + 16 * (lane + 32 * i));
                acc[m] = __dp4a((int)v[i].x, (int)x.x, acc[m]), acc[m] = __dp4a((int)v[i].y, (int)x.y, acc[m]);
                acc[m] = __dp4a((int)v[i].z, (int)x.z, acc[m]), acc[m] = __dp4a((int)v[i].w, (int)x.w, acc[m]);
            }
        }
        const float ws = __ldg(a.ws + n), b = a.bias ? __ldg(a.bias + n) : 0.f;
        T *y = reinterpret_cast<T *>(a.y) + n;
        n += gridDim.x * kFewWarps;
        w = a.w + (long long)n * a.ldw;
        weights();
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int o = 16; o; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
            if (m < rows && lane == m) finish<T, EPI>(acc[m], sxs[m], ws, b, y + (long long)m * a.ldy);
        }
    }
}

// ---------------------------------------------------------------------------
// many rows: a pair of SMs owns 256 channels x 256 tokens at a time (tcgen05.mma with cta_group::2), each with 128 of the
// channels and half of the tokens in its shared memory, so that a tile's operands cross from L2 once: 64 bytes a cycle
// and SM at the integer MMAs' 8192 products, where a single SM's 128 x 256 tile would want 96.  Persistent: two
// accumulators in tensor memory, and sixteen warps turn one into outputs while the next tile's products run (12000 rows x
// 1280 x 5120 with GELU: 83 us with eight warps, 70 with sixteen; 111 when the outputs were stored one by one).  2.3
// POP/s, the integer pipe 56 % active: bound by the operands' way from L2, 616 MB at 9 TB/s.
// ---------------------------------------------------------------------------
constexpr int kPrWarps = 16, kPrThreads = 64 + 32 * kPrWarps, kPrTokens = 1024 / kPrWarps, kPrStage = 2 * kMmTile * kMmK;
constexpr int pr_stages(int bytes) { return bytes == 4 ? 4 : 5; }
constexpr int pr_out(int bytes) { return 32 * 32 * bytes; }  // a warp's outgoing box
constexpr size_t pr_smem(int bytes) { return (size_t)pr_stages(bytes) * kPrStage + kPrWarps * pr_out(bytes) + 1024; }

__device__ __forceinline__ void arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// a box into this block's shared memory, its bytes counted by a barrier of either block of the pair
__device__ __forceinline__ void tma_load_pair(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// the barrier at this place in both blocks
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void pair_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// TMA: outputs leave as boxes of 32 channels x 32 tokens through shared memory (ymap; not with a residual)
template <typename T, int EPI, bool TMA>
__global__ void __launch_bounds__(kPrThreads, 1) k_linear_i8_pair(const __grid_constant__ CUtensorMap wmap,
                                                                  const __grid_constant__ CUtensorMap xmap,
                                                                  const __grid_constant__ CUtensorMap ymap, LinearI8Args a,
                                                                  int token_tiles, int tiles) {
    constexpr int kPrStages = pr_stages(sizeof(T)), kPrOut = pr_out(sizeof(T));
    extern __shared__ unsigned char raw[];
    unsigned char *sm = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[kPrStages], empty[kPrStages], acc_full[2], acc_free[2], drained;
    __shared__ uint32_t slot;
    __shared__ int failed;
    __shared__ __align__(16) float xs[kPrWarps][kPrTokens];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x & 1;
    const int nk = (a.K + kMmK - 1) / kMmK, pairs = gridDim.x / 2;
    if (tid == 0) {
        for (int i = 0; i < kPrStages; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 1);
        for (int i = 0; i < 2; ++i) mbar_init(acc_full + i, 1), mbar_init(acc_free + i, 2 * kPrWarps);
        mbar_init(&drained, 1);
        fence_mbar_init();
        failed = 0;
    }
    pdl_wait();  // before the tensor memory: a kernel that waits must not hold what the one before it may need
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    pair_barrier();  // both blocks' barriers are there
    tc_fence_after();
    const uint32_t tmem = slot;
    if (warp == 0) {
        // the first block's `full` counts both blocks' bytes
        int it = 0;
        bool ok = true;
        for (int t = blockIdx.x / 2; t < tiles && ok; t += pairs) {
            const int n0 = t / token_tiles * 256 + 128 * rank, m0 = t % token_tiles * 256 + 128 * rank;
            for (int k = 0; k < nk; ++k, ++it) {
                const int st = it % kPrStages;
                ok = __all_sync(0xffffffffu, it < kPrStages || mbar_wait(empty + st, (it / kPrStages - 1) & 1, &failed));
                if (!ok) break;
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(full + st, 2 * kPrStage);
                    const uint32_t bar = peer_address(full + st, 0);
                    tma_load_pair(sm + st * kPrStage, &wmap, k * kMmK, n0, bar);
                    tma_load_pair(sm + st * kPrStage + kMmTile * kMmK, &xmap, k * kMmK, m0, bar);
                }
                __syncwarp();
            }
        }
        // after a wait that ran out, copies that are in flight land within microseconds: wait a good while longer
        if (*(volatile int *)&failed)
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t idesc = idesc_i8(256, 256);
            int it = 0, n = 0;
            bool ok = true;
            for (int t = blockIdx.x / 2; t < tiles && ok; t += pairs, ++n) {
                const int b = n & 1;
                ok = __all_sync(0xffffffffu, n < 2 || mbar_wait(acc_free + b, (n / 2 - 1) & 1, &failed));
                for (int k = 0; k < nk && ok; ++k, ++it) {
                    const int st = it % kPrStages;
                    ok = __all_sync(0xffffffffu, mbar_wait(full + st, (it / kPrStages) & 1, &failed));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t at = smem_u32(sm + st * kPrStage);
                    if (elect_one()) {
#pragma unroll
                        for (int i = 0; i < kMmK / 32; ++i)
                            umma_i8_pair(tmem + 256 * b, sw128_desc(at) + 2 * i, sw128_desc(at + kMmTile * kMmK) + 2 * i, idesc,
                                         k > 0 || i > 0);
                        commit_pair(empty + st);
                        if (k == nk - 1) commit_pair(acc_full + b);
                    }
                    __syncwarp();
                }
            }
            if (!ok) {  // nothing may be in flight when the tensor memory is given back
                if (elect_one()) commit_pair(&drained);
                mbar_wait(&drained, 0, &failed);
            }
        }
    } else {
        // the warps of one lane quarter share the tokens
        const int e = warp - 2, quarter = warp & 3, first = e / 4 * kPrTokens;
        float *sx = xs[e];
        unsigned char *out = sm + kPrStages * kPrStage + e * kPrOut;
        int n = 0;
        bool ok = true;
        for (int t = blockIdx.x / 2; t < tiles; t += pairs, ++n) {
            const int b = n & 1, ch = t / token_tiles * 256 + 128 * rank + 32 * quarter + lane, m0 = t % token_tiles * 256 + first;
            const int rows = min(kPrTokens, a.M - m0);
            const bool in = ch < a.N;
            float ws = in ? __ldg(a.ws + ch) : 0.f;
            const float bias = in && a.bias ? __ldg(a.bias + ch) : 0.f;
            __syncwarp();
#pragma unroll
            for (int j = lane; j < kPrTokens; j += 32) sx[j] = j < rows ? __ldg(a.xs + m0 + j) : 0.f;
            __syncwarp();
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(acc_full + b, (n / 2) & 1, &failed));
            if (!ok) ws = NAN;  // after a wait that ran out every output is NaN
            tc_fence_after();
            const uint64_t ws2 = both(ws), bias2 = both(bias);
            T *y = reinterpret_cast<T *>(a.y) + (long long)m0 * a.ldy + ch;
            for (int j0 = 0; j0 < rows; j0 += 32) {
                uint32_t acc[32];
                __syncwarp();
                tmem_ld32(tmem + ((uint32_t)quarter << 21) + 256 * b + first + j0, acc);
                if (j0 + 32 >= rows) {  // the accumulator has been read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_at(peer_address(acc_free + b, 0));
                }
                uint64_t v[16];
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(sx + j0 + 2 * j);
                    v[j] = output2<EPI>((int)acc[2 * j], (int)acc[2 * j + 1], x.x, ws2, bias2);
                    v[j + 1] = output2<EPI>((int)acc[2 * j + 2], (int)acc[2 * j + 3], x.y, ws2, bias2);
                }
                if (TMA) {
                    T *box = reinterpret_cast<T *>(out);
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        box[64 * j + lane] = from_f32<T>(lo(v[j])), box[64 * j + 32 + lane] = from_f32<T>(hi(v[j]));
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {  // rows and channels beyond y are left out by the map
                        if (ch < a.N)
                            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(&ymap),
                                         "r"(ch), "r"(m0 + j0), "r"(smem_u32(box))
                                         : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                    continue;
                }
                // each store 32 neighbouring channels of one token
                if (EPI == 2) {
                    T old[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (in && j0 + j < rows) old[j] = y[j * a.ldy];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = add2(v[j], pack(to_f32<T>(old[2 * j]), to_f32<T>(old[2 * j + 1])));
                }
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (in && j0 + j < rows) y[j * a.ldy] = from_f32<T>(j & 1 ? hi(v[j / 2]) : lo(v[j / 2]));
                y += 32 * a.ldy;
            }
            if (rows <= 0 && lane == 0) arrive_at(peer_address(acc_free + b, 0));
        }
        if (TMA && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    pair_barrier();  // no block ends, or gives back its tensor memory, while the other's products may use it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Boxes of a row-major matrix, ld bytes from row to row; reads beyond its rows or columns give zeros, writes there are
// left out.
bool tmap_2d(CUtensorMap *m, CUtensorMapDataType type, const void *base, long long rows, int cols, long long ld, int box_cols,
             int box_rows, CUtensorMapSwizzle swizzle) {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult r;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) == cudaSuccess &&
                        r == cudaDriverEntryPointSuccess;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ok ? p : nullptr);
    }();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return fn(m, type, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// [box x 128 bytes] of an operand, with the 128-byte swizzle of the MMA's K-major operands
bool tmap_i8(CUtensorMap *m, const int8_t *base, long long rows, int cols, long long ld, int box) {
    return tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rows, cols, ld, kMmK, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

long long mm_tiles(const LinearI8Args &a, int nt) {
    return (long long)((a.N + kMmTile - 1) / kMmTile) * ((a.M + nt - 1) / nt);
}
// k is split while the tiles leave SMs idle and every block keeps two stages of k
int mm_split(long long tiles, int kb) {
    int ks = 1;
    while (ks < 8 && tiles * ks * 2 <= 148 && kb >= 4 * ks) ks *= 2;
    return ks;
}

template <int NT, typename T, int EPI>
cudaError_t product(const LinearI8Args &a, cudaStream_t s) {
    const int k16 = (a.K + 15) / 16 * 16, kb = (a.K + kMmK - 1) / kMmK;
    alignas(64) CUtensorMap wmap, xmap;
    if (!tmap_i8(&wmap, a.w, a.N, k16, a.ldw, kMmTile) || !tmap_i8(&xmap, a.x, a.M, k16, a.ldx, NT))
        return cudaErrorInvalidValue;
    const long long token_tiles = (a.M + NT - 1) / NT, tiles = mm_tiles(a, NT);
    const int ks = mm_split(tiles, kb);
    return launch_after<k_linear_i8<NT, T, EPI>>((unsigned)(tiles * ks), kMmThreads, mm_smem(NT), s, ks, wmap, xmap, a, ks,
                        (int)token_tiles);
}

template <typename T, int EPI>
cudaError_t product_pair(const LinearI8Args &a, cudaStream_t s) {
    const int k16 = (a.K + 15) / 16 * 16;
    alignas(64) CUtensorMap wmap, xmap;
    if (!tmap_i8(&wmap, a.w, a.N, k16, a.ldw, kMmTile) || !tmap_i8(&xmap, a.x, a.M, k16, a.ldx, kMmTile))
        return cudaErrorInvalidValue;
    const int token_tiles = (a.M + 255) / 256;
    const long long tiles = (long long)((a.N + 255) / 256) * token_tiles;
    if (tiles > 0x7fffffff) return cudaErrorInvalidValue;
    const unsigned blocks = 2 * (unsigned)(tiles < 74 ? tiles : 74);
    CUtensorMap ymap = {};
    // (a box that ends inside 16 bytes of y would write all of them: then the last channel has to end on their border)
    if (EPI != 2 && reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && a.ldy * sizeof(T) % 16 == 0 && a.N * sizeof(T) % 16 == 0) {
        const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                         : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        if (!tmap_2d(&ymap, type, a.y, a.M, a.N, a.ldy * sizeof(T), 32, 32, CU_TENSOR_MAP_SWIZZLE_NONE)) return cudaErrorInvalidValue;
        return launch_after<k_linear_i8_pair<T, EPI, true>>(blocks, kPrThreads, pr_smem(sizeof(T)), s, 2, wmap, xmap, ymap, a, token_tiles,
                            (int)tiles);
    }
    return launch_after<k_linear_i8_pair<T, EPI, false>>(blocks, kPrThreads, pr_smem(sizeof(T)), s, 2, wmap, xmap, ymap, a, token_tiles,
                        (int)tiles);
}

constexpr int kFewRows = 8;

// Which kernel takes a product, times in a graph: the warps' one pass over the weights where it is short (K = 1280: 2 rows
// 3.3 us against 4.4, 4 rows 4.5 against 4.4; K = 384: 4 rows 2.3 against 3.4; K = 5120: 1 row 3.6 against 4.7, 2 rows 5.4
// against 4.7); the pair where single blocks of 128 x 128 would need a second turn of the SMs (K = 1280, N = 5120: 320 rows
// 9.8 us against 8.1, 512 rows 9.8 against 15.2; K = 5120, N = 1280: 1500 rows 18.1 against 17.1, 2048 rows 18.3 against 31.9);
// single blocks otherwise, with as many tokens nt as take the least time by what was measured of a block: 2.5 us + 0.02 us
// a token + (0.27 + 0.0003 nt) us for each 128 of its k + 1 us for a cluster's sums, one block to an SM (77 x 1000 x 701: 6.1 us with nt = 128, 4.1 with 32;
// 100 x 5120 x 1280: 7.3 with 128, 7.5 with 64, 9.3 with 32).
template <typename T, int EPI>
cudaError_t product(const LinearI8Args &a, cudaStream_t s) {
    const unsigned few = (a.N + kFewWarps - 1) / kFewWarps;
    if (a.M == 1) return launch_after<k_linear_i8_few<1, T, EPI>>(few, kFewWarps * 32, 0, s, 1, a);
    if (a.M <= kFewRows && a.M * (long long)a.K < 5120) {
        if (a.M <= 4) return launch_after<k_linear_i8_few<4, T, EPI>>(few, kFewWarps * 32, 0, s, 1, a);
        return launch_after<k_linear_i8_few<8, T, EPI>>(few, kFewWarps * 32, 0, s, 1, a);
    }
    if (a.M > 128 && mm_tiles(a, 128) > 148) return product_pair<T, EPI>(a, s);
    const int kb = (a.K + kMmK - 1) / kMmK;
    int nt = 16;
    float least = 0.f;
    for (const int x : {16, 32, 64, 128}) {
        const long long tiles = mm_tiles(a, x);
        const int ks = mm_split(tiles, kb), steps = (kb + ks - 1) / ks;
        const float us = (float)((tiles * ks + 147) / 148) * (2.5f + 0.02f * x + steps * (0.27f + 0.0003f * x) + (ks > 1));
        if (x == 16 || us < least) least = us, nt = x;
    }
    if (nt == 16) return product<16, T, EPI>(a, s);
    if (nt == 32) return product<32, T, EPI>(a, s);
    if (nt == 64) return product<64, T, EPI>(a, s);
    return product<128, T, EPI>(a, s);
}

template <typename T, int EPI>
cudaError_t layer(const LinearI8Args &a, const QuantizeArgs &q, cudaStream_t s) {
    // as many as find room at once: a second turn would wait for the rows a second time (1 x 1280 x 5120 in a graph: 6.9 us
    // with a block for each eight channels, 4.7 so)
    const unsigned all = (a.N + kFewWarps - 1) / kFewWarps, most = 148 * kLayerBlocks, blocks = all < most ? all : most;
    const size_t smem = (size_t)a.M * ((a.K + 15) / 16 * 16);
    if (a.M == 1) return launch_after<k_linear_i8_layer<1, T, EPI>>(blocks, kFewWarps * 32, smem, s, 1, a, q);
    if (a.M == 2) return launch_after<k_linear_i8_layer<2, T, EPI>>(blocks, kFewWarps * 32, smem, s, 1, a, q);
    return launch_after<k_linear_i8_layer<4, T, EPI>>(blocks, kFewWarps * 32, smem, s, 1, a, q);
}

template <typename T>
cudaError_t layer(const LinearI8Args &a, const QuantizeArgs &q, cudaStream_t s) {
    return a.epilogue == 0 ? layer<T, 0>(a, q, s) : a.epilogue == 1 ? layer<T, 1>(a, q, s) : layer<T, 2>(a, q, s);
}

template <typename T>
cudaError_t product(const LinearI8Args &a, cudaStream_t s) {
    return a.epilogue == 0 ? product<T, 0>(a, s) : a.epilogue == 1 ? product<T, 1>(a, s) : product<T, 2>(a, s);
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

size_t linear_i8_layer_work(int M, int K) {
    const size_t k16 = ((size_t)K + 15) / 16 * 16;
    return M <= 4 && M * k16 <= kLayerSmem ? 0 : M * (k16 + 4);
}

cudaError_t launch_linear_i8_layer(LinearI8Args a, QuantizeArgs q, void *work, cudaStream_t s) {
    if (linear_i8_layer_work(a.M, a.K) == 0)
        return a.type == W4J_GGML_F32 ? layer<float>(a, q, s) : a.type == W4J_GGML_F16 ? layer<__half>(a, q, s)
                                                                                      : layer<__nv_bfloat16>(a, q, s);
    // the integers, then the rows' scales
    q.ldq = a.ldx = ((long long)a.K + 15) / 16 * 16;
    q.q = static_cast<int8_t *>(work);
    q.scale = reinterpret_cast<float *>(q.q + a.M * q.ldq);
    a.x = q.q, a.xs = q.scale;
    const cudaError_t e = launch_quantize_rows(q, s);
    return e == cudaSuccess ? launch_linear_i8(a, s) : e;
}

}  // namespace w4j
