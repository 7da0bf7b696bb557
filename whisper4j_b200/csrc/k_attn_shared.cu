// k_attn_shared.cu — attention over a paged cache for a batch whose groups share their first tokens.
//
// Mathematics.  A query of row b sees keys [0, n_b); keys [0, s_g) are the same for all rows of its group
// g, so softmax(q K^T) V splits into a part over [0, s_g), computed for all of the group's queries against
// one reading of the keys, and a part over [s_g, n_b) of the row's own.  Every part keeps its running
// maximum m, sum l = sum exp(x - m) and o = sum exp(x - m) v in 32 bits; parts of one query join as
//   m = max m_i,  o = sum e^(m_i - m) o_i / sum e^(m_i - m) l_i,
// in the order of the parts, so results do not depend on which block ran first.  Long stretches of
// keys are split into such parts as well, so that few rows still fill the device.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "attn_shared.cuh"
#include "host_api.cuh"
#include "tc_common.cuh"

namespace w4j {

namespace {

constexpr float kNone = -INFINITY;

__device__ __forceinline__ float ex2(float x) {  // 2^x to two units in the last place; 0 below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t *a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two numbers rounded to the cache's type (half a step of it: 2^-11 or 2^-8 relative), `lo` in the low half: outputs, and the
// softmax's weights, because the tensor cores take both operands of P V in one 16-bit type.  (In place of 32-bit weights that
// takes the error of the measured cases from 2.1e-4 to 2.6e-4 .. 2.9e-4 in fp16, 1.7e-3 to 2.3e-3 in bf16.)
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// whether a pair holds an infinity or a NaN
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t v);
template <>
__device__ __forceinline__ bool not_finite<__half>(uint32_t v) {
    return (v & 0x7c00u) == 0x7c00u || (v & 0x7c000000u) == 0x7c000000u;
}
template <>
__device__ __forceinline__ bool not_finite<__nv_bfloat16>(uint32_t v) {
    return (v & 0x7f80u) == 0x7f80u || (v & 0x7f800000u) == 0x7f800000u;
}

// The last i in [0, n) with key(i) <= x (0 where there is none), 32 places at a time; the whole warp calls it.
template <typename Key>
__device__ __forceinline__ int warp_find(int n, long long x, Key key) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + (threadIdx.x & 31) * step;
        const unsigned m = __ballot_sync(0xffffffffu, at < hi && key(at) <= x);
        const int last = m ? 31 - __clz(m) : 0;
        lo += last * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// Bounded wait that never sleeps: the phases follow one another within a microsecond or two.  A test that fails takes
// 4.4 us (measured where none succeeded), so that a wait runs out after 1.2 s.
__device__ __forceinline__ bool wait_phase(uint64_t *bar, unsigned parity, int *failed) {
    for (int it = 0; it < 1 << 18; ++it)
        if (mbar_test(bar, parity)) return true;
    atomicExch(failed, 2);
    return false;
}

// ---------------------------------------------------------------------------
// one warp: 8 NT query rows against a stretch of keys
//
// The products are taken the other way round, S^T = K Q^T and O^T = V^T P^T, so that the MMA's 16 rows are keys and
// dimensions and its 8 columns the few queries; P goes from one fragment layout to the other by an 8 x 8
// transposition.  Each warp has a ring of its own: a stage holds STEP keys and their values, brought page by page
// as TMA boxes (128-byte swizzle, read back by ldmatrix), so that a stage is in flight while another is worked on
// without holding registers, and no warp waits for another.  Bound by HBM and, where rows are short, by the look-ups
// that each begins with: 256 rows x 20 heads of 64, 257 tokens each on average, 61 us, 5.5 TB/s (112 us with fragments
// loaded straight into registers); 64 x 5 rows of 111 tokens behind 227 shared ones 56 us, 4.5 TB/s.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

// A block is one warp: rows differ in length, and a block of four kept its shared memory until the last had ended (64
// streams x 5 beams: 61.2 us with four, 59.9 with two, 55.4 with one).
constexpr int kAsWarps = 1, kAsStages = 2;
constexpr int as_step(int D) { return 2048 / D; }             // keys of a stage
constexpr int as_stage(int D) { return as_step(D) * D * 4; }  // its bytes: the keys, then their values
constexpr size_t as_smem(int D, int warps) { return (size_t)warps * kAsStages * as_stage(D) + 1024; }

template <typename T, int D, int NT>
struct WarpTile {
    static constexpr int NB = D / 64, STEP = as_step(D), H = STEP / 16, kBlock = STEP * 128, kKeys = NB * kBlock, kAsStage = as_stage(D);
    uint32_t qf[NT][D / 16][2];
    float o[NT][D / 16][4];  // dimension 16 t + g + 8 (e >> 1), query 8 n + 2 q + (e & 1)
    float m[NT][2], l[NT][2];

    // row[n]: query 8 n + g, null where there is none
    __device__ __forceinline__ void load_q(const T *const (&row)[NT]) {
        const int q = threadIdx.x & 3;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    qf[n][t][i] = row[n] ? __ldg(reinterpret_cast<const uint32_t *>(row[n] + 16 * t + 8 * i + 2 * q)) : 0;
                o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.f;
            }
            m[n][0] = m[n][1] = kNone, l[n][0] = l[n][1] = 0.f;
        }
    }

    // Keys [k0, k1) of the row whose table is `table`; boxes below `shared` are found in `first`'s instead.  Query
    // 8 n + 2 q + i sees the keys below lim[n][i], all queries see those below `all`.  sm: the warp's ring, full: a
    // barrier for each stage; box: rows of a TMA box.
    __device__ __forceinline__ void run(const PagesArgs &p, const int *table, const int *first, int shared, int head, const CUtensorMap *kmap,
                                        const CUtensorMap *vmap, unsigned char *sm, uint64_t *full, int box, int k0, int k1,
                                        const int (&lim)[NT][2], int all, float scale_log2, unsigned withhold, int *bad, int *failed) {
        const int lane = threadIdx.x & 31, g = lane >> 2;
        if (k0 >= k1) return;
        const int start = k0 / box * box, n_steps = (k1 - start + STEP - 1) / STEP;  // boxes do not cross pages
        // lane b (keys) and lane 16 + b (values) bring box b of a step; page and place in it of its first key
        int key = start + (lane & 15) * box, j = key / p.page_tokens, tok = key - j * p.page_tokens;
        const int dj = STEP / p.page_tokens, dt = STEP - dj * p.page_tokens;
        const bool mine = (lane & 15) * box < STEP;
        auto page_of = [&]() { return mine && key < k1 ? __ldg((key + box <= shared ? first : table) + j) : 0; };
        int page = page_of();
        auto issue = [&](int i) {
            const int at = start + i * STEP, boxes = (min(STEP, k1 - at) + box - 1) / box, st = i % kAsStages;
            if (lane == 0) mbar_expect_tx(full + st, 2 * NB * boxes * box * 128 + withhold);
            if (page < 0 || page >= p.n_pages) *bad = 1, page = 0;
            const int y = (page * p.n_kv_head + head) * p.page_tokens + tok;
            __syncwarp();
            if ((lane & 15) < boxes) {
                unsigned char *dst = sm + st * kAsStage + (lane >> 4) * kKeys + (lane & 15) * box * 128;
                for (int b = 0; b < NB; ++b) tma_load_2d(dst + b * kBlock, lane < 16 ? kmap : vmap, 64 * b, y, full + st);
            }
            __syncwarp();
            key += STEP, j += dj, tok += dt;
            if (tok >= p.page_tokens) tok -= p.page_tokens, ++j;
            page = page_of();  // for the next call
        };
        for (int i = 0; i < kAsStages && i < n_steps; ++i) issue(i);
        // ldmatrix rows: keys as they lie, values transposed; offsets of the first 16 keys' units of dimensions 16 t on
        const int kr = lane & 15, kc = lane >> 4, vr = (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;
        uint32_t k_at[4], v_at[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) k_at[t] = kr * 128 + ((2 * t + kc) ^ (kr & 7)) * 16, v_at[t] = kKeys + vr * 128 + ((2 * t + vc) ^ (vr & 7)) * 16;
        int i = 0;
        for (; i < n_steps; ++i) {
            const int st = i % kAsStages, kb = start + i * STEP;
            if (!__all_sync(0xffffffffu, wait_phase(full + st, (i / kAsStages) & 1, failed))) break;
            const uint32_t base = smem_u32(sm + st * kAsStage);
            const bool masked = kb < k0 || kb + STEP > min(k1, all);
            if (kb + STEP > k1) {  // behind the last key there may be anything: zero
                for (int x = lane; x < (kb + STEP - k1) * 8 * NB; x += 32)
                    *reinterpret_cast<uint4 *>(sm + st * kAsStage + kKeys + x % NB * kBlock + (k1 - kb) * 128 + x / NB * 16) =
                        make_uint4(0, 0, 0, 0);
                __syncwarp();
            }
            float s[NT][H][4];  // key 16 h + g + 8 (e >> 1), query 8 n + 2 q + (e & 1)
#pragma unroll
            for (int h = 0; h < H; ++h) {
#pragma unroll
                for (int n = 0; n < NT; ++n) s[n][h][0] = s[n][h][1] = s[n][h][2] = s[n][h][3] = 0.f;
#pragma unroll
                for (int t = 0; t < D / 16; ++t) {
                    uint32_t a[4];
                    ldsm4(a, base + k_at[t & 3] + t / 4 * kBlock + h * 2048);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma<T>(s[n][h], a, qf[n][t][0], qf[n][t][1]);
                }
            }
            uint32_t pf[NT][H][2];
            float c[NT][2];
            bool grown = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int sees = min(k1, lim[n][x]) - kb - g, from = k0 - kb - g;
                    float mx = kNone;
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int e = x; e < 4; e += 2) {
                            const int at = 16 * h + 8 * (e >> 1);
                            if (masked && (at >= sees || at < from)) s[n][h][e] = kNone;
                            mx = fmaxf(mx, s[n][h][e]);
                        }
#pragma unroll
                    for (int y = 4; y < 32; y *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, y));
                    mx = fmaxf(m[n][x], mx * scale_log2);
                    c[n][x] = m[n][x] == mx ? 1.f : ex2(m[n][x] - mx);
                    grown |= c[n][x] != 1.f;
                    m[n][x] = mx;
                    if (mx == kNone) mx = 0.f;  // nothing seen so far: all weights are 0
                    float sum = 0.f;
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int e = x; e < 4; e += 2) {
                            s[n][h][e] = ex2(fmaf(s[n][h][e], scale_log2, -mx));
                            sum += s[n][h][e];
                        }
                    l[n][x] = l[n][x] * c[n][x] + sum;  // this lane's keys; summed over g at the end
                }
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int x = 0; x < 2; ++x) pf[n][h][x] = transpose8(pack2<T>(s[n][h][2 * x], s[n][h][2 * x + 1]));
            }
            if (__any_sync(0xffffffffu, grown))
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int t = 0; t < D / 16; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][t][e] *= c[n][e & 1];
            if (kb + STEP > all && hides(sm + st * kAsStage + kKeys)) {
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int t = 0; t < D / 16; ++t) {
                        uint32_t a[4];
                        ldsm4_t(a, base + v_at[t & 3] + t / 4 * kBlock + h * 2048);
#pragma unroll
                        for (int n = 0; n < NT; ++n) add_hidden(o[n][t], a, pf[n][h], lim[n], kb + 16 * h);
                    }
            } else {
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int t = 0; t < D / 16; ++t) {
                        uint32_t a[4];
                        ldsm4_t(a, base + v_at[t & 3] + t / 4 * kBlock + h * 2048);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma<T>(o[n][t], a, pf[n][h][0], pf[n][h][1]);
                    }
            }
            __syncwarp();
            if (i + kAsStages < n_steps) issue(i + kAsStages);
        }
        // after a wait that ran out: let the copies in flight land before the block's shared memory goes on
        for (int x = i; x < min(n_steps, i + kAsStages); ++x)
            for (int it = 0; it < 1 << 16 && !mbar_test(full + x % kAsStages, (x / kAsStages) & 1); ++it) {
            }
    }

    // Where a key that only some queries see holds an infinity or a NaN, 0 x v is none: the queries take their
    // turns, each with the keys that it does not see set to zero.
    __device__ __forceinline__ bool hides(const unsigned char *values) const {
        bool bad = false;
        for (int x = threadIdx.x & 31; x < kKeys / 16; x += 32) {
            const uint4 v = *reinterpret_cast<const uint4 *>(values + 16 * x);
            bad |= not_finite<T>(v.x) || not_finite<T>(v.y) || not_finite<T>(v.z) || not_finite<T>(v.w);
        }
        return __any_sync(0xffffffffu, bad);
    }
    __device__ __forceinline__ void add_hidden(float (&acc)[4], const uint32_t (&a)[4], const uint32_t (&pf)[2],
                                               const int (&lim)[2], int k16) {
        const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll 1
        for (int r = 0; r < 8; ++r) {
            const int sees = __shfl_sync(0xffffffffu, r & 1 ? lim[1] : lim[0], r >> 1) - k16 - 2 * q;
            const uint32_t lo = (sees > 0 ? 0xffffu : 0u) | (sees > 1 ? 0xffff0000u : 0u);
            const uint32_t hi = (sees > 8 ? 0xffffu : 0u) | (sees > 9 ? 0xffff0000u : 0u);
            const uint32_t ar[4] = {a[0] & lo, a[1] & lo, a[2] & hi, a[3] & hi};
            float x[4] = {};
            mma<T>(x, ar, g == r ? pf[0] : 0, g == r ? pf[1] : 0);
            // the other queries' 0 x v may be NaN here: only query r takes its sums
            if (2 * q == r) acc[0] += x[0], acc[2] += x[2];
            if (2 * q + 1 == r) acc[1] += x[1], acc[3] += x[3];
        }
    }

    // o, m (base 2) and l of query 8 n + 2 q + i to their places; null: no such query
    __device__ __forceinline__ void store(float *const (&po)[NT][2], float *const (&pm)[NT][2]) {
        const int g = (threadIdx.x & 31) >> 2;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int x = 4; x < 32; x *= 2) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], x);
                if (!po[n][i]) continue;
                if (g == 0) *reinterpret_cast<float2 *>(pm[n][i]) = make_float2(m[n][i], l[n][i]);
                if (l[n][i] == 0.f) continue;
#pragma unroll
                for (int t = 0; t < D / 16; ++t) po[n][i][16 * t + g] = o[n][t][i], po[n][i][16 * t + 8 + g] = o[n][t][2 + i];
            }
    }
};

// Whether sequences first .. last are of group gr, found as warp_find does.  Groups that do not ascend may lay claim to the
// same sequences: a tile of shared keys leaves those of another group alone.  (What warp_find finds does not fall as the
// sequence grows: where the first and the last one's is gr, so is that of all between.)
__device__ __forceinline__ bool of_group(const AttnSharedArgs &a, int first, int last, int gr) {
    int lo = 0, hi = a.n_group;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + (threadIdx.x & 31) * step;
        const int start = at < hi ? __ldg(a.group_start + at) : 0x7fffffff;
        const unsigned m0 = __ballot_sync(0xffffffffu, start <= first), m1 = __ballot_sync(0xffffffffu, start <= last);
        if (__clz(m0 | 1) != __clz(m1 | 1)) return false;
        lo += (31 - __clz(m0 | 1)) * step;
        hi = min(hi, lo + step);
    }
    return lo == gr;
}

// ---------------------------------------------------------------------------
// items: (group tile, head, split) of the shared keys, then (row, head, tile, split) of the rows' own
// ---------------------------------------------------------------------------
// Row, its group's first row, length and shared length of sequence `seq`, 0 or what is wrong with it (then rows 0); the whole warp calls it.
// first: whether this call also looks at all of the groups, and reports what is wrong with them.  A sequence is of the group
// where warp_find finds it; where that is right, it gets its results whatever is wrong with others.
__device__ __forceinline__ int find_row(const AttnSharedArgs &a, int seq, bool first, int &row, int &row0, int &len, int &shared) {
    const PagesArgs &p = a.p;
    const int r = __ldg(a.rows + seq);
    const int gr = warp_find(a.n_group, seq, [&](int i) { return (long long)__ldg(a.group_start + i); });
    const int lo = __ldg(a.group_start + gr), hi = __ldg(a.group_start + gr + 1), s = __ldg(a.shared + gr);
    const bool row_ok = r >= 0 && r < p.n_rows;
    row = row_ok ? r : 0;
    len = row_ok ? max(0, min(__ldg(p.len + r), p.width * p.page_tokens)) : 0;
    shared = s;
    // the shared keys are read through the group's first row: what is wrong there concerns all of them
    const bool group_ok = lo >= 0 && lo <= seq && seq < hi && hi <= a.n_seq;
    const int r0 = group_ok ? __ldg(a.rows + lo) : -1;
    row0 = r0 >= 0 && r0 < p.n_rows ? r0 : 0;
    const int len0 = r0 >= 0 && r0 < p.n_rows ? __ldg(p.len + r0) : -1;
    int bad = !group_ok ? W4J_PAGES_BAD_START : !row_ok || len0 < 0 ? W4J_PAGES_BAD_ROW
              : s < 0 || s > a.max_shared || s > max(0, min(len, len0) - a.n_query + 1) ? W4J_PAGES_BAD_SHARED : 0;
    if (first) {  // the groups as a whole
        bool out = __ldg(a.group_start) != 0 || __ldg(a.group_start + a.n_group) != a.n_seq;
        for (int i = threadIdx.x & 31; i < a.n_group; i += 32) out |= __ldg(a.group_start + i) > __ldg(a.group_start + i + 1);
        if (out) atomicOr(p.status, W4J_PAGES_BAD_START);
    }
    return bad;
}

// (12 of these blocks' rings fit an SM: registers for as many, and for 16 where that costs nothing)
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kAsWarps * 32, NT == 1 ? 16 : 12) k_attn_shared(const __grid_constant__ CUtensorMap kmap,
                                                               const __grid_constant__ CUtensorMap vmap, AttnSharedArgs a,
                                                               int box) {
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[kAsWarps][kAsStages];
    __shared__ int failed[kAsWarps];
    // Behind k_attn_shared_tc this kernel starts while that one runs (all of its blocks have waited for whatever came
    // before, so that is done): the two read the same inputs, write different parts, and one is bound by its
    // exponentials, the other by HBM.  It then waits for it before it ends, so that the join need only wait for this one.
    if (!a.tc_tiles) pdl_wait();
    pdl_trigger();
    constexpr int R = 8 * NT;  // query rows of a tile
    const PagesArgs &p = a.p;
    const int lane = threadIdx.x & 31, g = lane >> 2, qd = lane & 3;
    const int c = a.n_query * a.rep;  // query rows of one sequence and one key/value head
    const T *q = reinterpret_cast<const T *>(a.q);
    unsigned item = blockIdx.x * kAsWarps + (threadIdx.x >> 5);
    int seq0, n_rows, head, split, tile, slot, k0, k1, own_len, bad = 0;
    unsigned mine = 0xffffffffu;  // the tile's rows
    const int *table;
    if (item < a.shared_items) {
        tile = (int)(item % a.shared_tiles);
        split = (int)(item / a.shared_tiles % a.shared_splits);
        head = (int)(item / a.shared_tiles / a.shared_splits);
        // group gr has tiles gs c / R + gr on (rounded down), one more than it may need
        const int gr = warp_find(a.n_group, tile, [&](int i) { return (long long)__ldg(a.group_start + i) * c / R + i; });
        seq0 = __ldg(a.group_start + gr);
        const int seq1 = __ldg(a.group_start + gr + 1);
        if (seq0 < 0 || seq1 <= seq0 || seq1 > a.n_seq) return;  // (no such items behind k_attn_shared_tc)
        tile -= (int)((long long)seq0 * c / R) + gr;
        n_rows = (seq1 - seq0) * c;
        const int r = __ldg(a.rows + seq0), s = min(__ldg(a.shared + gr), a.max_shared);
        if (tile < 0 || tile * R >= n_rows || r < 0 || r >= p.n_rows) return;
        if (!of_group(a, seq0 + tile * R / c, seq0 + min(n_rows - 1, tile * R + R - 1) / c, gr)) {
            mine = 0;
            for (int x = 0; x < R; ++x)
                if (tile * R + x < n_rows && of_group(a, seq0 + (tile * R + x) / c, seq0 + (tile * R + x) / c, gr)) mine |= 1u << x;
        }
        table = p.table + (size_t)r * p.width;
        const int len = max(0, min(min(s, __ldg(p.len + r)), p.width * p.page_tokens));
        const int step = ((len + a.shared_splits - 1) / a.shared_splits + 31) / 32 * 32;
        k0 = min(len, split * step), k1 = min(len, k0 + step);
        own_len = len + a.n_query - 1;  // every row sees every shared key
        slot = split;
    } else {
        item -= a.shared_items;
        if (item >= a.own_items) {
            if (a.tc_tiles) pdl_wait();
            return;
        }
        tile = (int)(item % a.own_tiles);
        split = (int)(item / a.own_tiles % a.own_splits);
        head = (int)(item / a.own_tiles / a.own_splits % p.n_kv_head);
        seq0 = (int)(item / a.own_tiles / a.own_splits / p.n_kv_head);
        n_rows = c;
        int r, r0, shared;
        bad = find_row(a, seq0, seq0 + head + split + tile == 0, r, r0, own_len, shared);
        table = p.table + (size_t)r * p.width;
        const int from = bad ? 0 : shared, n = bad ? 0 : own_len - shared;
        // pieces of one size whatever the row's length (a long row's would be the last to end), the last one to the end
        const int step = ((a.max_own + a.own_splits - 1) / a.own_splits + 31) / 32 * 32;
        k0 = from + min(n, split * step), k1 = split + 1 == (int)a.own_splits ? from + n : min(from + n, k0 + step);
        slot = a.shared_splits + split;
    }
    // query r of the tile: (sequence, query token, head)
    auto token_of = [&](int r) { return (size_t)(seq0 + r / c) * a.n_query + r % c / a.rep; };
    const T *qr[NT];
    float *po[NT][2], *pm[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = tile * R + 8 * n + g;
        qr[n] = r < n_rows && mine >> (8 * n + g) & 1 ? q + token_of(r) * a.q_stride + (size_t)(head * a.rep + r % a.rep) * D : nullptr;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int x = tile * R + 8 * n + 2 * qd + i;
            po[n][i] = pm[n][i] = nullptr, lim[n][i] = 0;
            if (x >= n_rows || !(mine >> (8 * n + 2 * qd + i) & 1)) continue;
            lim[n][i] = own_len - a.n_query + x % c / a.rep + 1;
            const size_t part = (token_of(x) * a.n_head + head * a.rep + x % a.rep) * a.slots + slot;
            po[n][i] = a.part_o + part * D;
            pm[n][i] = a.part_ml + part * 2;
        }
    }
    const int wi = threadIdx.x >> 5;
    if (lane == 0) {
        for (int i = 0; i < kAsStages; ++i) mbar_init(&full[wi][i], 1);
        fence_mbar_init();
        failed[wi] = 0;
    }
    __syncwarp();
    unsigned char *sm = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    WarpTile<T, D, NT> w;
    int bad_page = 0;
    w.load_q(qr);
    w.run(p, table, nullptr, 0, head, &kmap, &vmap, sm + wi * kAsStages * as_stage(D), full[wi], box, k0, k1, lim, own_len - a.n_query + 1,
          a.scale_log2, a.withhold, &bad_page, &failed[wi]);
    if (__any_sync(0xffffffffu, bad_page)) bad |= W4J_PAGES_BAD_PAGE;
    __syncwarp();
    if (failed[wi]) bad |= W4J_PAGES_TIMEOUT;
    if (bad) {
#pragma unroll
        for (int n = 0; n < NT; ++n) w.m[n][0] = w.m[n][1] = w.l[n][0] = w.l[n][1] = NAN;  // the join hands it on
        if (lane == 0) atomicOr(p.status, bad);
    }
    w.store(po, pm);
    if (a.tc_tiles) pdl_wait();
}

// ---------------------------------------------------------------------------
// a few rows: a block, or for longer rows a cluster of blocks, takes a row, head and tile; its warps share all of the row's
// keys (the group's among them: read again by every row, from L2) and join their sums in shared memory, the blocks' over
// the cluster's.  One launch and no scratch; bound by latency (5 rows x 8 heads x 284 tokens: 4.8 us in a graph, 8.4 with
// parts and a join; x 1500 tokens 7.8 and 11.1).
// ---------------------------------------------------------------------------
constexpr int kDirectWarps = 8, kDirectMost = 8;  // warps of a block, blocks of a cluster

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What block `rank` of the cluster has at this place of its shared memory.
__device__ __forceinline__ float2 ld_cluster(const float2 *p, int rank) {
    uint32_t at;
    float2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kDirectWarps * 32) k_attn_direct(const __grid_constant__ CUtensorMap kmap,
                                                                   const __grid_constant__ CUtensorMap vmap, AttnSharedArgs a,
                                                                   int box) {
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[kDirectWarps][kAsStages];
    __shared__ int failed, wrong;
    __shared__ float2 ml[kDirectWarps][8 * NT], block_ml[8 * NT];
    pdl_wait();
    pdl_trigger();
    constexpr int R = 8 * NT;
    const PagesArgs &p = a.p;
    const int tid = threadIdx.x, wi = tid >> 5, lane = tid & 31, g = lane >> 2, qd = lane & 3;
    const int c = a.n_query * a.rep;
    const int rank = blockIdx.x % a.direct, item = blockIdx.x / a.direct;
    const int tile = item % a.own_tiles, head = item / a.own_tiles % p.n_kv_head, seq = item / a.own_tiles / p.n_kv_head;
    if (tid == 0) failed = wrong = 0;
    if (lane == 0) {
        for (int i = 0; i < kAsStages; ++i) mbar_init(&full[wi][i], 1);
        fence_mbar_init();
    }
    __syncthreads();
    int row, row0, len, shared;
    int bad = find_row(a, seq, blockIdx.x == 0, row, row0, len, shared);
    const int n = bad ? 0 : len, warps = a.direct * kDirectWarps, step = ((n + warps - 1) / warps + 31) / 32 * 32;
    const int k0 = min((long long)n, (long long)(rank * kDirectWarps + wi) * step), k1 = min(n, k0 + step);
    const T *q = reinterpret_cast<const T *>(a.q);
    const T *qr[NT];
    int lim[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = tile * R + 8 * t + g;
        qr[t] = r < c ? q + ((size_t)seq * a.n_query + r / a.rep) * a.q_stride + (size_t)(head * a.rep + r % a.rep) * D : nullptr;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int x = tile * R + 8 * t + 2 * qd + i;
            lim[t][i] = x < c ? len - a.n_query + x / a.rep + 1 : 0;
        }
    }
    unsigned char *sm = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023) +
                        wi * kAsStages * as_stage(D);
    WarpTile<T, D, NT> w;
    int bad_page = 0;
    w.load_q(qr);
    w.run(p, p.table + (size_t)row * p.width, p.table + (size_t)row0 * p.width, bad ? 0 : shared, head, &kmap, &vmap, sm, full[wi], box, k0, k1, lim, len - a.n_query + 1, a.scale_log2,
          a.withhold, &bad_page, &failed);
    if (__any_sync(0xffffffffu, bad_page)) bad |= W4J_PAGES_BAD_PAGE;
    if (bad && lane == 0) atomicOr(&wrong, bad);
    __syncwarp();
    // the warp's o over its ring, [8 NT][D]
    float *po[NT][2], *pm[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            po[t][i] = reinterpret_cast<float *>(sm) + (8 * t + 2 * qd + i) * D;
            pm[t][i] = reinterpret_cast<float *>(&ml[wi][8 * t + 2 * qd + i]);
        }
    w.store(po, pm);
    __syncthreads();
    const bool lost = failed || wrong;
    if (tid == 0 && lost) atomicOr(p.status, wrong | (failed ? W4J_PAGES_TIMEOUT : 0));
    float *o0 = reinterpret_cast<float *>(sm - wi * kAsStages * as_stage(D));
    auto put = [&](int r, int d, float l, float u, float v) {
        const int qi = tile * R + r;
        if (qi >= c) return;
        const float inv = l == 0.f ? 0.f : 1.f / l;  // a query that sees nothing gets zeros
        T *out = reinterpret_cast<T *>(a.out) + ((size_t)seq * a.n_query + qi / a.rep) * a.out_stride + (size_t)(head * a.rep + qi % a.rep) * D;
        *reinterpret_cast<uint32_t *>(out + d) = pack2<T>(u * inv, v * inv);
    };
    for (int x = tid; x < R * D / 2; x += kDirectWarps * 32) {
        const int r = x / (D / 2), d = 2 * (x % (D / 2));
        float m = kNone, l = 0.f, u = 0.f, v = 0.f;
#pragma unroll
        for (int y = 0; y < kDirectWarps; ++y) m = fmaxf(m, ml[y][r].x);
#pragma unroll
        for (int y = 0; y < kDirectWarps; ++y) {
            const float2 part = ml[y][r];
            if (part.y == 0.f) continue;
            const float f = ex2(part.x - m);
            const float2 o = *reinterpret_cast<const float2 *>(o0 + y * (kAsStages * as_stage(D) / 4) + r * D + d);
            l += f * part.y, u += f * o.x, v += f * o.y;
        }
        if (lost) m = 0.f, l = NAN;
        if (a.direct == 1) {
            put(r, d, l, u, v);
            continue;
        }
        // over the first warp's, whose two numbers of this place no other thread reads
        *reinterpret_cast<float2 *>(o0 + r * D + d) = make_float2(u, v);
        if (d == 0) block_ml[r] = make_float2(m, l);
    }
    if (a.direct == 1) return;
    cluster_sync();
    for (int x = rank * kDirectWarps * 32 + tid; x < R * D / 2; x += a.direct * kDirectWarps * 32) {
        const int r = x / (D / 2), d = 2 * (x % (D / 2));
        float2 part[kDirectMost], o[kDirectMost];
        float m = kNone, l = 0.f, u = 0.f, v = 0.f;
#pragma unroll
        for (int y = 0; y < kDirectMost; ++y) {
            const int from = min(y, a.direct - 1);
            part[y] = y < a.direct ? ld_cluster(block_ml + r, from) : make_float2(kNone, 0.f);
            o[y] = ld_cluster(reinterpret_cast<const float2 *>(o0 + r * D + d), from);
            m = fmaxf(m, part[y].x);
        }
#pragma unroll
        for (int y = 0; y < kDirectMost; ++y) {
            if (part[y].y == 0.f) continue;
            const float f = ex2(part[y].x - m);
            l += f * part[y].y, u += f * o[y].x, v += f * o[y].y;
        }
        put(r, d, l, u, v);
    }
    cluster_sync();  // the others have read this block's
}

// ---------------------------------------------------------------------------
// shared keys on the 5th-generation tensor cores: 128 query rows of a group against 128 keys at a time
//
// S = Q K^T (tcgen05.mma, operands in shared memory) and O += P V (P from tensor memory).  Two warpgroups take the first
// and the second 64 keys of every tile, each with a maximum, sum and O of its own; a thread owns a row, so the softmax
// needs no shuffle.  There are two S buffers, P overwrites its S.  O is rescaled only when a row's maximum has grown by
// more than 2^8 (weights up to 2^8 are as good as weights up to 1 in either type), by its owner, once the products so far
// are in.  Keys and values come page by page through TMA boxes (128-byte swizzle) into two rings; V is the MMA's B
// operand as it lies in the pages (MN-major).
//
// 128 x 128 exponentials take the 16 a cycle of an SM's special function units 1024 cycles, the MMAs of a tile 512 (head
// 64) or 1024 (head 128); a tile takes 1850 to 2500 (4 x 256 rows x 16381 keys x 8 heads of 128: 86 us, 0.8 PFLOP/s),
// bound by the round from S over P to the S that comes after the
// next (softmax 1500, P V and Q K^T 600 to 900 with their hand-overs).  Moving 4 to 16 of every 32 exponentials to a
// polynomial on the FMA pipes made that round longer (142 -> 143 .. 150 us on 4 x 256 rows x 16381 keys x 8 heads of
// 128) and was not kept.
// ---------------------------------------------------------------------------
constexpr int kTcThreads = 384, kTcKeys = 128, kTcBlock = 128 * 128;  // bytes of 64 numbers of 128 rows

constexpr int tc_stages(int D) { return D == 64 ? 4 : 3; }
constexpr size_t tc_smem(int D) { return (size_t)(D / 64) * kTcBlock * (1 + 2 * tc_stages(D)) + 1024; }

__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),
                   "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]),
                   "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]),
                   "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at), "r"(v[0]),
                   "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                   "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
                   "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]),
                   "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]) : "memory");
}
// two 32-bit numbers at a time
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One lane of a warp that runs as one.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}

// A from tensor memory
__device__ __forceinline__ void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// An operand whose rows (128 bytes, 64 numbers of the M or N dimension) follow one another along K, 128-byte
// swizzle: groups of 8 rows 1024 bytes apart, the next 64 numbers of M or N `next` bytes on.
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t saddr, uint32_t next) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(next >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 1) k_attn_shared_tc(const __grid_constant__ CUtensorMap kmap,
                                                                  const __grid_constant__ CUtensorMap vmap, AttnSharedArgs a,
                                                                  int box) {
    constexpr int NB = D / 64, NS = tc_stages(D), kTile = NB * kTcBlock;
    constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
    extern __shared__ unsigned char raw[];
    unsigned char *sq = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *sk = sq + NB * kTcBlock, *sv = sk + NS * kTile;
    __shared__ uint64_t k_full[NS], k_empty[NS], v_full[NS], v_empty[NS], q_full, s_full[2], p_full[4], pv_done[4], drained[2];
    __shared__ uint32_t slot_word;
    __shared__ int failed, bad_page;
    __shared__ float m1[128], l1[128];
    pdl_wait();
    pdl_trigger();
    const PagesArgs &p = a.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int c = a.n_query * a.rep;
    int tile = blockIdx.x % a.tc_tiles;
    const int split = blockIdx.x / a.tc_tiles % a.shared_splits, head = blockIdx.x / a.tc_tiles / a.shared_splits;
    const int gr = warp_find(a.n_group, tile, [&](int i) { return (long long)__ldg(a.group_start + i) * c / 128 + i; });
    const int seq0 = __ldg(a.group_start + gr), seq1 = __ldg(a.group_start + gr + 1);
    if (seq0 < 0 || seq1 <= seq0 || seq1 > a.n_seq) return;
    tile -= (int)((long long)seq0 * c / 128) + gr;
    const int n_rows = (seq1 - seq0) * c, r0 = __ldg(a.rows + seq0);
    if (tile < 0 || tile * 128 >= n_rows || r0 < 0 || r0 >= p.n_rows) return;
    const int *table = p.table + (size_t)r0 * p.width;
    const int len = max(0, min(min(min(__ldg(a.shared + gr), a.max_shared), __ldg(p.len + r0)), p.width * p.page_tokens));
    const int all = (len + kTcKeys - 1) / kTcKeys, per = (all + a.shared_splits - 1) / a.shared_splits;
    const int t0 = min(all, split * per), n = min(all, t0 + per) - t0;
    // the row of this thread: (sequence, query token, head)
    const int r = tile * 128 + (tid & 127);
    bool mine = r < n_rows && tid < 256;
    if (!of_group(a, seq0 + tile * 128 / c, seq0 + min(n_rows - 1, tile * 128 + 127) / c, gr))
        for (int x = 0; x < 32; ++x) {
            const int seq = seq0 + (r - lane + x) / c;
            const bool of = of_group(a, seq, seq, gr);
            if (lane == x && !of) mine = false;
        }
    size_t part = 0;
    const T *qr = nullptr;
    if (mine) {
        const size_t token = (size_t)(seq0 + r / c) * a.n_query + r % c / a.rep;
        const int h = head * a.rep + r % a.rep;
        qr = reinterpret_cast<const T *>(a.q) + token * a.q_stride + (size_t)h * D;
        part = (token * a.n_head + h) * a.slots + split;
    }
    if (n <= 0) {
        if (qr && tid < 128) a.part_ml[part * 2] = kNone, a.part_ml[part * 2 + 1] = 0.f;
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < NS; ++i) mbar_init(k_full + i, 1), mbar_init(k_empty + i, 1), mbar_init(v_full + i, 1), mbar_init(v_empty + i, 2);
        for (int i = 0; i < 4; ++i) mbar_init(p_full + i, 4), mbar_init(pv_done + i, 1);
        for (int i = 0; i < 2; ++i) mbar_init(s_full + i, 1), mbar_init(drained + i, 1);
        mbar_init(&q_full, 256);
        fence_mbar_init();
        failed = bad_page = 0;
    }
    if (warp == 9) tmem_alloc(&slot_word, 512), tmem_relinquish();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // S of tile i at columns 128 (i % 2), a half for each warpgroup, O of warpgroup w at 256 + w D;
    // p_full and pv_done: of warpgroup w and tile i at 2 (i % 2) + w
    const uint32_t tmem = slot_word;
    if (warp >= 8) {
        // every warp of these runs as one (its descriptors stay uniform); one lane issues
        bool ok = true;
        if (warp == 8 || warp == 11) {
            // warp 8 brings the keys, warp 11 the values, lane b box b of each tile
            const CUtensorMap *map = warp == 8 ? &kmap : &vmap;
            uint64_t *full = warp == 8 ? k_full : v_full, *empty = warp == 8 ? k_empty : v_empty;
            unsigned char *ring = warp == 8 ? sk : sv;
            int key = t0 * kTcKeys + lane * box, issued = 0;
            auto page_of = [&]() { return lane * box < kTcKeys && key < len ? __ldg(table + key / p.page_tokens) : 0; };
            int page = page_of();
            for (int i = 0; i < n; ++i) {
                const int st = i % NS, boxes = (min(kTcKeys, len - (t0 + i) * kTcKeys) + box - 1) / box;
                if (page < 0 || page >= p.n_pages) bad_page = 1, page = 0;
                const int y = (page * p.n_kv_head + head) * p.page_tokens + key % p.page_tokens;
                key += kTcKeys;
                page = page_of();  // for the next tile
                if (!__all_sync(0xffffffffu, i < NS || wait_phase(empty + st, (i / NS - 1) & 1, &failed))) break;
                if (lane == 0) mbar_expect_tx(full + st, boxes * box * 128 * NB + a.withhold);
                __syncwarp();
                if (lane < boxes)
                    for (int b = 0; b < NB; ++b)
                        tma_load_2d(ring + st * kTile + b * kTcBlock + lane * box * 128, map, 64 * b, y, full + st);
                __syncwarp();
                issued = i + 1;
            }
            // after a wait that ran out: let the copies in flight land before the block's shared memory goes on
            if (lane == 0 && *(volatile int *)&failed) drain_ring(full, NS, issued);
        } else if (warp == 9) {  // S = Q K^T
            constexpr uint32_t id = idesc_f16(128, kTcKeys) | kType;
            ok = __all_sync(0xffffffffu, wait_phase(&q_full, 0, &failed));
            for (int i = 0; i < n && ok; ++i) {
                const int st = i % NS, b = i & 1;
                ok = wait_phase(k_full + st, (i / NS) & 1, &failed);
                if (i >= 2)  // both halves of P of tile i - 2 have been read
                    ok = ok && wait_phase(pv_done + 2 * b, ((i >> 1) - 1) & 1, &failed) &&
                         wait_phase(pv_done + 2 * b + 1, ((i >> 1) - 1) & 1, &failed);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t q0 = smem_u32(sq), k0 = smem_u32(sk + st * kTile);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        umma_f16(tmem + 128 * b, sw128_desc(q0 + k / 4 * kTcBlock) + 2 * (k % 4),
                                 sw128_desc(k0 + k / 4 * kTcBlock) + 2 * (k % 4), id, k > 0);
                    umma_commit(s_full + b);
                    umma_commit(k_empty + st);
                }
                __syncwarp();
            }
        } else {  // O += P V, the two halves of a tile in turn
            constexpr uint32_t id = idesc_f16(128, D) | kType | (1u << 16);
            for (int i = 0; i < 2 * n && ok; ++i) {
                const int t = i >> 1, w = i & 1, st = t % NS, bi = 2 * (t & 1) + w;
                ok = wait_phase(v_full + st, (t / NS) & 1, &failed) && wait_phase(p_full + bi, (t >> 1) & 1, &failed);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t v0 = smem_u32(sv + st * kTile) + w * 64 * 128;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_f16_ta(tmem + 256 + w * D, tmem + 64 * bi + 8 * k, sw128_desc_mn(v0 + 2048 * k, kTcBlock), id,
                                    t > 0 || k > 0);
                    umma_commit(pv_done + bi);
                    umma_commit(v_empty + st);
                }
                __syncwarp();
            }
        }
        if (warp == 9 || warp == 10) {
            __syncwarp();
            if (*(volatile int *)&failed) {  // nothing may be in flight when the tensor memory is given back
                if (elect_one()) umma_commit(drained + warp - 9);
                wait_phase(drained + warp - 9, 0, &failed);
            }
        }
    } else {
        const int w = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21, o_at = tmem + lanes + 256 + w * D;
        // the query tile, rows behind the group's last as zeros: warpgroup w lays out every other 16-byte unit
#pragma unroll
        for (int u = w; u < D / 8; u += 2) {
            const uint4 v = qr ? __ldg(reinterpret_cast<const uint4 *>(qr) + u) : make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4 *>(sq + u / 8 * kTcBlock + row * 128 + ((u % 8 ^ (row & 7)) << 4)) = v;
        }
        fence_proxy_async();
        mbar_arrive(&q_full);
        const uint64_t scale2 = pair(__float_as_uint(a.scale_log2), __float_as_uint(a.scale_log2));
        float m = 0.f, l = 0.f;
        bool ok = true;
        for (int i = 0; i < n; ++i) {
            const int valid = max(0, min(64, len - (t0 + i) * kTcKeys - 64 * w)), bi = 2 * (i & 1) + w;  // of this half
            const uint32_t s_at = tmem + lanes + 64 * bi;
            ok = __all_sync(0xffffffffu, wait_phase(s_full + (i & 1), (i >> 1) & 1, &failed));
            if (!ok) break;
            tc_fence_after();
            uint32_t s[64];
            tmem_load32(s_at, s);
            tmem_load32(s_at + 32, s + 32);
            tmem_wait_ld();
            if (valid < 64)
#pragma unroll
                for (int x = 0; x < 64; ++x)
                    if (x >= valid) s[x] = __float_as_uint(kNone);
            float mx[4] = {kNone, kNone, kNone, kNone};
#pragma unroll
            for (int x = 0; x < 64; x += 2)
                mx[x / 2 & 3] = max3(mx[x / 2 & 3], __uint_as_float(s[x]), __uint_as_float(s[x + 1]));
            const float top = max3(mx[0], mx[1], fmaxf(mx[2], mx[3])) * a.scale_log2;
            if (i == 0) {
                m = top;  // kNone until a key has scored more than -inf
            } else if (__any_sync(0xffffffffu, top > m + 8.f)) {
                ok = __all_sync(0xffffffffu, wait_phase(pv_done + (bi ^ 2), ((i - 1) >> 1) & 1, &failed));
                if (!ok) break;
                tc_fence_after();
                const float f = top > m ? ex2(m - top) : 1.f;
                m = fmaxf(m, top);
                l *= f;
#pragma unroll 1
                for (int x = 0; x < D; x += 32) {
                    uint32_t o[32];
                    tmem_load32(o_at + x, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tmem_store32(o_at + x, o);
                }
            }
            const float from = m == kNone ? 0.f : -m;
            const uint64_t base2 = pair(__float_as_uint(from), __float_as_uint(from));
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int x = 0; x < 64; x += 2) {
                const uint64_t e = fma2(pair(s[x], s[x + 1]), scale2, base2);
                const float e0 = ex2(__uint_as_float((uint32_t)e)), e1 = ex2(__uint_as_float((uint32_t)(e >> 32)));
                sum[x / 2 & 1] = add2(sum[x / 2 & 1], pair(__float_as_uint(e0), __float_as_uint(e1)));
                s[x / 2] = pack2<T>(e0, e1);
            }
            tmem_store32(s_at, s);
            sum[0] = add2(sum[0], sum[1]);
            l += __uint_as_float((uint32_t)sum[0]) + __uint_as_float((uint32_t)(sum[0] >> 32));
            if (valid < 64) {  // behind the last key there may be anything: 0 x NaN is none
                const int st = i % NS;
                ok = __all_sync(0xffffffffu, wait_phase(v_full + st, (i / NS) & 1, &failed));
                if (!ok) break;
                for (int x = row; x < (64 - valid) * 8 * NB; x += 128) {
                    const int at = 64 * w + valid + x / (8 * NB), u = x % (8 * NB);
                    *reinterpret_cast<uint4 *>(sv + st * kTile + u / 8 * kTcBlock + at * 128 + u % 8 * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + bi);
        }
        // both warpgroups' sums, joined by the first
        ok = ok && wait_phase(pv_done + 2 * ((n - 1) & 1) + w, ((n - 1) >> 1) & 1, &failed);
        __syncwarp();
        tc_fence_after();
        float *other = reinterpret_cast<float *>(sk);  // [D][128], over the keys: every S is there
        if (w == 1) {
#pragma unroll 1
            for (int x = 0; x < D; x += 32) {
                uint32_t o[32];
                tmem_load32(o_at + x, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) other[(x + e) * 128 + row] = __uint_as_float(o[e]);
            }
            m1[row] = m, l1[row] = l;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (w == 0) {
            const bool lost = *(volatile int *)&failed || *(volatile int *)&bad_page;
            // (a warpgroup whose keys all scored -inf, or without one, has l = 0 and O = 0, and nothing to say about the maximum)
            const bool none0 = l == 0.f, none1 = l1[row] == 0.f;
            const float top = none0 ? m1[row] : none1 ? m : fmaxf(m, m1[row]);
            const float f0 = none0 ? 0.f : ex2(m - top), f1 = none1 ? 0.f : ex2(m1[row] - top);
            l = l * f0 + l1[row] * f1;
            m = top;
            if (qr) a.part_ml[part * 2] = lost ? NAN : m, a.part_ml[part * 2 + 1] = lost ? NAN : l;
            if (tid == 0 && lost)
                atomicOr(p.status, (*(volatile int *)&bad_page ? W4J_PAGES_BAD_PAGE : 0) | (*(volatile int *)&failed ? W4J_PAGES_TIMEOUT : 0));
#pragma unroll 1
            for (int x = 0; x < D; x += 32) {
                uint32_t o[32];
                tmem_load32(o_at + x, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    o[e] = __float_as_uint(__uint_as_float(o[e]) * f0 + other[(x + e) * 128 + row] * f1);
                if (qr)
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4 *>(a.part_o + part * D + x + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 9) tc_fence_after(), tmem_dealloc(tmem, 512);
}

// The parts of one query joined, a warp per query and head, lane i dimensions i D / 32 on.  Bound by latency: 5 us for
// 5120 queries of 5 parts, most of it beside the kernel before it.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_attn_shared_join(AttnSharedArgs a) {
    pdl_wait();
    pdl_trigger();
    const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (r >= (long long)a.n_seq * a.n_query * a.n_head) return;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + r * a.slots;
    const float *po = a.part_o + r * a.slots * D;
    float mx = kNone;
    for (int i = lane; i < a.slots; i += 32) {
        const float2 v = __ldg(ml + i);
        mx = v.x != v.x || mx != mx ? NAN : fmaxf(mx, v.x);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float y = __shfl_xor_sync(0xffffffffu, mx, o);
        mx = y != y || mx != mx ? NAN : fmaxf(mx, y);
    }
    constexpr int N = D / 32;
    float acc[N] = {}, l = 0.f;
#pragma unroll 8
    for (int i = 0; i < a.slots; ++i) {
        const float2 v = __ldg(ml + i);
        const bool none = v.y == 0.f;  // then its place holds nothing
        const float f = none ? 0.f : ex2(v.x - mx);
        l += f * v.y;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = fmaf(f, none ? 0.f : po[(size_t)i * D + lane * N + e], acc[e]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a query that sees nothing gets zeros
    uint32_t w[N / 2];
#pragma unroll
    for (int e = 0; e < N / 2; ++e) w[e] = pack2<T>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    T *out = reinterpret_cast<T *>(a.out) + (r / a.n_head) * a.out_stride + (r % a.n_head) * D + lane * N;
#pragma unroll
    for (int e = 0; e < N / 2; ++e) reinterpret_cast<uint32_t *>(out)[e] = w[e];
}

template <typename T, int D>
cudaError_t launch(const AttnSharedArgs &a, cudaStream_t s) {
    const long long rows = (long long)a.n_seq * a.n_query * a.n_head;
    const PagesArgs &p = a.p;
    const int head_rows = p.n_pages * p.n_kv_head * p.page_tokens;
    const T *pk = reinterpret_cast<const T *>(p.pool) + (size_t)2 * a.layer * head_rows * D, *pv = pk + (size_t)head_rows * D;
    alignas(64) CUtensorMap km, vm;
    // boxes of up to `most` rows that do not cross pages
    auto maps = [&](int most) {
        int box = most;
        while (p.page_tokens % box) box /= 2;
        return make_tmap_f16_box(&km, pk, head_rows, D, box) && make_tmap_f16_box(&vm, pv, head_rows, D, box) ? box : 0;
    };
    cudaError_t e;
    if (a.direct) {
        const int box = maps(as_step(D));
        if (!box) return cudaErrorInvalidValue;
        const unsigned blocks = a.n_seq * p.n_kv_head * a.own_tiles * a.direct;
        const size_t smem = as_smem(D, kDirectWarps);
        return a.tile_rows == 8 ? launch_after<k_attn_direct<T, D, 1>>(blocks, kDirectWarps * 32, smem, s, a.direct, km, vm, a, box)
                                : launch_after<k_attn_direct<T, D, 2>>(blocks, kDirectWarps * 32, smem, s, a.direct, km, vm, a, box);
    }
    if (a.tc_tiles) {
        const int box = maps(kTcKeys);
        if (!box) return cudaErrorInvalidValue;
        e = launch_after<k_attn_shared_tc<T, D>>(a.tc_tiles * a.shared_splits * p.n_kv_head, kTcThreads, tc_smem(D), s, 1, km, vm,
                         a, box);
        if (e != cudaSuccess) return e;
    }
    const int box = maps(as_step(D));
    if (!box) return cudaErrorInvalidValue;
    const unsigned blocks = (a.shared_items + a.own_items + kAsWarps - 1) / kAsWarps;
    if (a.tile_rows == 8) {
        e = launch_after<k_attn_shared<T, D, 1>>(blocks, kAsWarps * 32, as_smem(D, kAsWarps), s, 1, km, vm, a, box);
    } else {
        e = launch_after<k_attn_shared<T, D, 2>>(blocks, kAsWarps * 32, as_smem(D, kAsWarps), s, 1, km, vm, a, box);
    }
    if (e != cudaSuccess) return e;
    return launch_after<k_attn_shared_join<T, D>>((unsigned)((rows + 7) / 8), 256, 0, s, 1, a);
}

}  // namespace

// From so many query rows of a group on, the tensor cores' tiles of 128 rows take the shared keys (64 groups and heads x
// 4096 keys, in a graph: head 64, 16 rows 30.3 us against the warps' 25.8, 24 rows 31.3 against 34.2; head 128, 8 rows 35.9
// against 36.1, 16 rows 37.6 against 49).
constexpr int tc_rows(int D) { return D == 64 ? 24 : 16; }

void attn_shared_plan(AttnSharedArgs &a) {
    const PagesArgs &p = a.p;
    const long long c = a.n_query * a.rep, want = 148 * 16;  // warps in flight on the device
    auto splits = [&](long long items, int keys) {
        // a step costs a warp 0.85 us, a part its row's join 0.18 us: no more parts than where both are
        // equal, nor of fewer than 64 keys
        const long long n = (want + items - 1) / items, steps = (keys + as_step(p.head_dim) - 1) / as_step(p.head_dim);
        long long most = 1;
        while (most < n && most * 64 < keys && most * most < 5 * steps) ++most;
        return (int)(n < most ? n : most);
    };
    // tiles of 16 query rows where a row's own part or, on the warps, a group has more than 8
    const bool tc = a.max_shared > 0 && a.n_seq * c / a.n_group >= tc_rows(p.head_dim);
    a.tile_rows = c <= 8 && (tc || a.max_shared == 0 || a.n_seq * c / a.n_group <= 8) ? 8 : 16;
    a.tc_tiles = a.shared_tiles = a.shared_splits = 0;
    if (a.max_shared > 0) {
        const long long avg = a.n_seq * c / a.n_group;  // query rows of a group and key/value head
        if (tc) {
            a.tc_tiles = (unsigned)(a.n_seq * c / 128 + a.n_group);
            // fewest rounds of blocks over the SMs times key tiles of a block (and about four more to start and join)
            const long long blocks = (avg + 127) / 128 * a.n_group * p.n_kv_head, tiles = (a.max_shared + 127) / 128;
            long long best = 0;
            for (int n = 1; n <= tiles && n <= 64; ++n) {
                const long long cost = (blocks * n + 147) / 148 * ((tiles + n - 1) / n + 4);
                if (n == 1 || cost < best) best = cost, a.shared_splits = n;
            }
        } else {
            a.shared_tiles = (unsigned)(a.n_seq * c / a.tile_rows + a.n_group);
            a.shared_splits = splits((long long)a.shared_tiles * p.n_kv_head, a.max_shared);
        }
    }
    a.shared_items = a.shared_tiles * a.shared_splits * p.n_kv_head;
    a.own_tiles = (unsigned)((c + a.tile_rows - 1) / a.tile_rows);
    // pieces of 256 keys, as long as they are not many times more than the device takes at once
    const long long own_items = (long long)a.n_seq * p.n_kv_head * a.own_tiles, most = 6 * want / own_items;
    const int own = a.max_own > 0 ? splits(own_items, a.max_own) : 1, pieces = (a.max_own + 255) / 256, some = most < pieces ? (int)most : pieces;
    a.own_splits = own > some ? own : some < 1 ? 1 : some;
    a.own_items = (unsigned)a.n_seq * p.n_kv_head * a.own_tiles * a.own_splits;
    a.slots = a.shared_splits + a.own_splits;
    // A row, head and tile to a block, or to a cluster of as many as find room at once (clusters of 7 or 5 fill the SMs'
    // groups badly), up to 16 steps a warp, on clusters of eight 32.  One row x 8 heads x 64, in a graph: 300 tokens 5.1 us
    // on a block, 5.8 on eight, 8.7 with parts and a join; 1500 tokens 9.7, 5.8, 10.3; 24000 tokens 82, 15.4, 26.8.  16 rows,
    // one block each: 1500 tokens 10.2 against 12.6, 6000 tokens 24.5 against 18.
    a.direct = 0;
    const unsigned direct_tiles = (unsigned)((c + (c <= 8 ? 7 : 15)) / (c <= 8 ? 8 : 16));
    const long long items = (long long)a.n_seq * p.n_kv_head * direct_tiles, keys = (long long)a.max_shared + a.max_own;
    int blocks = items <= 148 ? 1 : 0;
    if (keys > 512)
        for (const int n : {2, 3, 4, 6, 8})
            if (items * n <= (n == 2 ? 148 : 128)) blocks = n;
    if (blocks && keys <= (long long)blocks * kDirectWarps * (blocks < 8 ? 16 : 32) * as_step(p.head_dim)) {
        a.direct = blocks, a.slots = 0;
        a.tile_rows = c <= 8 ? 8 : 16, a.own_tiles = direct_tiles;
    }
}

size_t attn_shared_work_bytes(const AttnSharedArgs &a) {
    return (size_t)a.n_seq * a.n_query * a.n_head * a.slots * (a.p.head_dim + 2) * 4;
}

cudaError_t launch_attn_shared(const AttnSharedArgs &a, bool bf16, cudaStream_t s) {
    if (a.p.head_dim == 64) return bf16 ? launch<__nv_bfloat16, 64>(a, s) : launch<__half, 64>(a, s);
    return bf16 ? launch<__nv_bfloat16, 128>(a, s) : launch<__half, 128>(a, s);
}

}  // namespace w4j
