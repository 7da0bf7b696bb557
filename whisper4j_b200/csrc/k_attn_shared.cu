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

#include "attn_shared.cuh"
#include "host_api.cuh"
#include "w4j_internal.cuh"

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
// Two numbers rounded to the cache's type (half a step of it: 2^-11 or 2^-8 relative), `lo` in the low half.
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

// ---------------------------------------------------------------------------
// one warp: up to 16 query rows against a stretch of keys
//
// Fragments come from global memory straight into registers.  The contraction order over the head's
// dimensions is free, so lane (g, q) = (lane / 4, lane % 4) takes dimensions 32 u + 8 q .. + 7 of key g
// as one 16-byte load and feeds them to two MMA steps (the queries are laid out alike); the order of the
// output's columns is free too, so the same lane takes dimensions 8 g .. 8 g + 7 of keys 2 q, 2 q + 1,
// 2 q + 8, 2 q + 9 and column c of MMA tile t is dimension 8 c + t.  Every load of a warp covers whole
// 128-byte rows, and no shared memory or transposition is needed.  Bound by HBM as long as rows are few:
// 16 rows cost 16 flop per byte of the cache.
// ---------------------------------------------------------------------------
template <typename T, int D>
struct WarpTile {
    static constexpr int KU = D / 32, NW = D / 64;
    uint32_t qf[2 * KU][4];
    float o[NW][8][4];
    float m[2], l[2];

    // rows g and g + 8 of the tile, null where there is none
    __device__ __forceinline__ void load_q(const T *r0, const T *r1) {
        const int q = threadIdx.x & 3;
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            uint4 a = make_uint4(0, 0, 0, 0), b = a;
            if (r0) a = __ldg(reinterpret_cast<const uint4 *>(r0 + 32 * u + 8 * q));
            if (r1) b = __ldg(reinterpret_cast<const uint4 *>(r1 + 32 * u + 8 * q));
            qf[2 * u][0] = a.x, qf[2 * u][1] = b.x, qf[2 * u][2] = a.y, qf[2 * u][3] = b.y;
            qf[2 * u + 1][0] = a.z, qf[2 * u + 1][1] = b.z, qf[2 * u + 1][2] = a.w, qf[2 * u + 1][3] = b.w;
        }
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int t = 0; t < 8; ++t) o[w][t][0] = o[w][t][1] = o[w][t][2] = o[w][t][3] = 0.f;
        m[0] = m[1] = kNone;
        l[0] = l[1] = 0.f;
    }

    // o += P V for 16 keys; p: the A fragment, v0 .. v3: keys 2 q, 2 q + 1, 2 q + 8, 2 q + 9
    __device__ __forceinline__ void pv(const uint32_t (&p)[4], const uint4 (&v)[NW][4]) {
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const uint32_t *x0 = &v[w][0].x, *x1 = &v[w][1].x, *x2 = &v[w][2].x, *x3 = &v[w][3].x;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const uint32_t sel = t & 1 ? 0x7632u : 0x5410u;
                mma<T>(o[w][t], p, __byte_perm(x0[t / 2], x1[t / 2], sel), __byte_perm(x2[t / 2], x3[t / 2], sel));
            }
        }
    }

    // Keys [k0, k1) of the row whose table is `table`; row r of the tile sees those below lim[r] (r = g, g + 8)
    // and all rows see those below `all`.  plane_k / plane_v: the head rows of the layer.
    __device__ __forceinline__ void run(const PagesArgs &p, const int *table, int head, const T *plane_k, const T *plane_v,
                                        int k0, int k1, const int (&lim)[2], int all, float scale_log2, int *bad) {
        const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
        for (int kb = k0; kb < k1; kb += 32) {
            // lane i finds head row kb + i
            const int key = kb + lane;
            uint32_t at = 0;
            if (key < k1) {
                const int j = key / p.page_tokens;
                int page = __ldg(table + j);
                if (page < 0 || page >= p.n_pages) *bad = 1, page = 0;
                at = ((uint32_t)page * p.n_kv_head + head) * p.page_tokens + (key - j * p.page_tokens);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int k16 = kb + 16 * c;
                if (k16 >= k1) break;
                uint4 kf[2][KU], vf[NW][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const size_t r = __shfl_sync(0xffffffffu, at, 16 * c + 8 * i + g);
#pragma unroll
                    for (int u = 0; u < KU; ++u)
                        kf[i][u] = __ldg(reinterpret_cast<const uint4 *>(plane_k + r * D + 32 * u + 8 * q));
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int kk = (i >> 1) * 8 + 2 * q + (i & 1);
                    const size_t r = __shfl_sync(0xffffffffu, at, 16 * c + kk);
#pragma unroll
                    for (int w = 0; w < NW; ++w)  // behind the last key there may be anything: zero
                        vf[w][i] = k16 + kk < k1 ? __ldg(reinterpret_cast<const uint4 *>(plane_v + r * D + 64 * w + 8 * g))
                                                 : make_uint4(0, 0, 0, 0);
                }
                float s[2][4] = {};
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int u = 0; u < KU; ++u) {
                        mma<T>(s[i], qf[2 * u], kf[i][u].x, kf[i][u].y);
                        mma<T>(s[i], qf[2 * u + 1], kf[i][u].z, kf[i][u].w);
                    }
                // s[i][e]: key k16 + 8 i + 2 q + (e & 1), row g + 8 (e >> 1)
                float mx[2] = {m[0], m[1]};
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[i][e] = k16 + 8 * i + 2 * q + (e & 1) < min(k1, lim[e >> 1]) ? s[i][e] * scale_log2 : kNone;
                        mx[e >> 1] = fmaxf(mx[e >> 1], s[i][e]);
                    }
                float f[2], sum[2] = {0.f, 0.f};
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                    f[r] = m[r] == mx[r] ? 1.f : ex2(m[r] - mx[r]);
                    m[r] = mx[r];
                    if (mx[r] == kNone) mx[r] = 0.f;  // nothing seen so far: all weights are 0
                }
                uint32_t pf[4];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[i][e] = ex2(s[i][e] - mx[e >> 1]);
                        sum[e >> 1] += s[i][e];
                    }
                pf[0] = pack2<T>(s[0][0], s[0][1]), pf[1] = pack2<T>(s[0][2], s[0][3]);
                pf[2] = pack2<T>(s[1][0], s[1][1]), pf[3] = pack2<T>(s[1][2], s[1][3]);
#pragma unroll
                for (int r = 0; r < 2; ++r) l[r] = l[r] * f[r] + sum[r];  // this lane's keys; summed over q at the end
                if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f))
#pragma unroll
                    for (int w = 0; w < NW; ++w)
#pragma unroll
                        for (int t = 0; t < 8; ++t)
                            o[w][t][0] *= f[0], o[w][t][1] *= f[0], o[w][t][2] *= f[1], o[w][t][3] *= f[1];
                if (k16 + 16 > all && hides(vf))
                    pv_hidden(pf, vf, k16, lim);
                else
                    pv(pf, vf);
            }
        }
    }

    // Where a key that only some rows see holds an infinity or a NaN, 0 x v is none: the rows take their
    // turns, each with the keys that it does not see set to zero.
    __device__ __forceinline__ bool hides(const uint4 (&v)[NW][4]) {
        bool bad = false;
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                bad |= not_finite<T>(v[w][i].x) || not_finite<T>(v[w][i].y) || not_finite<T>(v[w][i].z) ||
                       not_finite<T>(v[w][i].w);
        return __any_sync(0xffffffffu, bad);
    }
    __device__ __forceinline__ void pv_hidden(const uint32_t (&p)[4], const uint4 (&v)[NW][4], int k16,
                                              const int (&lim)[2]) {
        const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const uint32_t *x0 = &v[w][0].x, *x1 = &v[w][1].x, *x2 = &v[w][2].x, *x3 = &v[w][3].x;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const uint32_t sel = t & 1 ? 0x7632u : 0x5410u;
                const uint32_t b0 = __byte_perm(x0[t / 2], x1[t / 2], sel), b1 = __byte_perm(x2[t / 2], x3[t / 2], sel);
#pragma unroll 1
                for (int r = 0; r < 16; ++r) {
                    const int sees = __shfl_sync(0xffffffffu, r < 8 ? lim[0] : lim[1], (r & 7) * 4) - k16 - 2 * q;
                    const uint32_t lo = (sees > 0 ? 0xffffu : 0u) | (sees > 1 ? 0xffff0000u : 0u);
                    const uint32_t hi = (sees > 8 ? 0xffffu : 0u) | (sees > 9 ? 0xffff0000u : 0u);
                    const bool mine0 = g == r, mine1 = g + 8 == r;
                    const uint32_t pr[4] = {mine0 ? p[0] : 0, mine1 ? p[1] : 0, mine0 ? p[2] : 0, mine1 ? p[3] : 0};
                    float acc[4] = {};
                    mma<T>(acc, pr, b0 & lo, b1 & hi);
                    // the other rows' 0 x v may be NaN here: only row r takes its sums
                    if (mine0) o[w][t][0] += acc[0], o[w][t][1] += acc[1];
                    if (mine1) o[w][t][2] += acc[2], o[w][t][3] += acc[3];
                }
            }
        }
    }

    // o, m (base 2) and l of rows g and g + 8 to their places; null: no such row
    __device__ __forceinline__ void store(float *o0, float *o1, float *ml0, float *ml1) {
        const int q = threadIdx.x & 3;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            float *po = r ? o1 : o0, *pm = r ? ml1 : ml0;
            if (!po) continue;
            if (q == 0) pm[0] = m[r], pm[1] = l[r];
            if (l[r] == 0.f) continue;
#pragma unroll
            for (int w = 0; w < NW; ++w)
#pragma unroll
                for (int c = 0; c < 2; ++c)  // column 2 q + c of tiles 0 .. 7: dimensions 64 w + 16 q + 8 c .. + 7
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        *reinterpret_cast<float4 *>(po + 64 * w + 16 * q + 8 * c + 4 * h) =
                            make_float4(o[w][4 * h][2 * r + c], o[w][4 * h + 1][2 * r + c], o[w][4 * h + 2][2 * r + c],
                                        o[w][4 * h + 3][2 * r + c]);
        }
    }
};

// ---------------------------------------------------------------------------
// items: (group tile, head, split) of the shared keys, then (row, head, tile, split) of the rows' own
// ---------------------------------------------------------------------------
constexpr int kAsWarps = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kAsWarps * 32) k_attn_shared(AttnSharedArgs a) {
    pdl_wait();
    pdl_trigger();
    const PagesArgs &p = a.p;
    const int lane = threadIdx.x & 31, g = lane >> 2;
    const int c = a.n_query * a.rep;  // query rows of one sequence and one key/value head
    const size_t plane = (size_t)p.n_pages * p.n_kv_head * p.page_tokens * D;
    const T *pk = reinterpret_cast<const T *>(p.pool) + 2 * a.layer * plane, *pv = pk + plane;
    const T *q = reinterpret_cast<const T *>(a.q);
    unsigned item = blockIdx.x * kAsWarps + (threadIdx.x >> 5);
    int seq0, n_rows, head, split, tile, slot, k0, k1, own_len, bad = 0;
    const int *table;
    if (item < a.shared_items) {
        tile = (int)(item % a.shared_tiles);
        split = (int)(item / a.shared_tiles % a.shared_splits);
        head = (int)(item / a.shared_tiles / a.shared_splits);
        // group gr has tiles gs c / 16 + gr on (rounded down), one more than it may need
        const int gr = warp_find(a.n_group, tile, [&](int i) { return (long long)__ldg(a.group_start + i) * c / 16 + i; });
        seq0 = __ldg(a.group_start + gr);
        const int seq1 = __ldg(a.group_start + gr + 1);
        if (seq0 < 0 || seq1 <= seq0 || seq1 > a.n_seq) return;
        tile -= (int)((long long)seq0 * c / 16) + gr;
        n_rows = (seq1 - seq0) * c;
        const int r = __ldg(a.rows + seq0), s = min(__ldg(a.shared + gr), a.max_shared);
        if (tile < 0 || tile * 16 >= n_rows || r < 0 || r >= p.n_rows) return;
        table = p.table + (size_t)r * p.width;
        const int len = max(0, min(min(s, __ldg(p.len + r)), p.width * p.page_tokens));
        const int step = ((len + a.shared_splits - 1) / a.shared_splits + 31) / 32 * 32;
        k0 = min(len, split * step), k1 = min(len, k0 + step);
        own_len = len + a.n_query - 1;  // every row sees every shared key
        slot = split;
    } else {
        item -= a.shared_items;
        if (item >= a.own_items) return;
        tile = (int)(item % a.own_tiles);
        split = (int)(item / a.own_tiles % a.own_splits);
        head = (int)(item / a.own_tiles / a.own_splits % p.n_kv_head);
        seq0 = (int)(item / a.own_tiles / a.own_splits / p.n_kv_head);
        n_rows = c;
        const int r = __ldg(a.rows + seq0);
        const int gr = warp_find(a.n_group, seq0, [&](int i) { return (long long)__ldg(a.group_start + i); });
        const int lo = __ldg(a.group_start + gr), hi = __ldg(a.group_start + gr + 1), s = __ldg(a.shared + gr);
        const bool row_ok = r >= 0 && r < p.n_rows;
        own_len = row_ok ? max(0, min(__ldg(p.len + r), p.width * p.page_tokens)) : 0;
        table = p.table + (size_t)(row_ok ? r : 0) * p.width;
        // the shared keys are read through the group's first row: what is wrong there concerns all of them
        const bool group_ok = lo >= 0 && lo <= seq0 && seq0 < hi && hi <= a.n_seq;
        const int r0 = group_ok ? __ldg(a.rows + lo) : -1;
        const int len0 = r0 >= 0 && r0 < p.n_rows ? __ldg(p.len + r0) : -1;
        bad = !group_ok ? W4J_PAGES_BAD_START : !row_ok || len0 < 0 ? W4J_PAGES_BAD_ROW
              : s < 0 || s > a.max_shared || s > max(0, min(own_len, len0) - a.n_query + 1) ? W4J_PAGES_BAD_SHARED : 0;
        if (seq0 + head + split + tile == 0 && (lo != 0 || __ldg(a.group_start + a.n_group) != a.n_seq))
            bad |= W4J_PAGES_BAD_START;
        const int from = bad ? 0 : s, n = bad ? 0 : own_len - s;
        const int step = ((n + a.own_splits - 1) / a.own_splits + 31) / 32 * 32;
        k0 = from + min(n, split * step), k1 = min(from + n, k0 + step);
        slot = a.shared_splits + split;
    }
    WarpTile<T, D> w;
    // rows g and g + 8 of the tile: (sequence, query token, head) of each
    const T *qr[2];
    float *po[2], *pm[2];
    int lim[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = tile * 16 + g + 8 * i;
        qr[i] = nullptr, po[i] = pm[i] = nullptr, lim[i] = 0;
        if (r >= n_rows) continue;
        const int seq = seq0 + r / c, t = r % c / a.rep, h = head * a.rep + r % a.rep;
        const size_t token = (size_t)seq * a.n_query + t;
        qr[i] = q + token * a.q_stride + (size_t)h * D;
        lim[i] = own_len - a.n_query + t + 1;
        const size_t part = (token * a.n_head + h) * a.slots + slot;
        po[i] = a.part_o + part * D;
        pm[i] = a.part_ml + part * 2;
    }
    int bad_page = 0;
    w.load_q(qr[0], qr[1]);
    w.run(p, table, head, pk, pv, k0, k1, lim, own_len - a.n_query + 1, a.scale_log2, &bad_page);
    if (__any_sync(0xffffffffu, bad_page)) bad |= W4J_PAGES_BAD_PAGE;
    if (bad) {
        w.m[0] = w.m[1] = w.l[0] = w.l[1] = NAN;  // the join hands it on to the whole row
        if (lane == 0) atomicOr(p.status, bad);
    }
    w.store(po[0], po[1], pm[0], pm[1]);
}

// The parts of one query joined, a warp per query and head, lane i dimensions i D / 32 on.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_attn_shared_join(AttnSharedArgs a) {
    pdl_wait();
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
    for (int i = 0; i < a.slots; ++i) {
        const float2 v = __ldg(ml + i);
        if (v.y == 0.f) continue;
        const float f = ex2(v.x - mx);
        l += f * v.y;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += f * po[(size_t)i * D + lane * N + e];
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
    cudaError_t e = launch_after(k_attn_shared<T, D>, (a.shared_items + a.own_items + kAsWarps - 1) / kAsWarps, kAsWarps * 32, 0, s, 1, a);
    if (e != cudaSuccess) return e;
    return launch_after(k_attn_shared_join<T, D>, (unsigned)((rows + 7) / 8), 256, 0, s, 1, a);
}

}  // namespace

void attn_shared_plan(AttnSharedArgs &a) {
    const PagesArgs &p = a.p;
    const long long c = a.n_query * a.rep, want = 148 * 16;  // warps in flight on the device
    auto splits = [&](long long items, int keys) {
        const long long n = (want + items - 1) / items, most = (keys + 63) / 64;
        return (int)(n < most ? n : most);
    };
    a.shared_tiles = (int)(a.n_seq * c / 16 + a.n_group);
    a.shared_splits = a.max_shared > 0 ? splits((long long)a.shared_tiles * p.n_kv_head, a.max_shared) : 0;
    a.shared_items = (unsigned)a.shared_tiles * a.shared_splits * p.n_kv_head;
    a.own_tiles = (int)((c + 15) / 16);
    const int own = a.max_own > 0 ? splits((long long)a.n_seq * p.n_kv_head * a.own_tiles, a.max_own) : 1;
    a.own_splits = own < 1 ? 1 : own;
    a.own_items = (unsigned)a.n_seq * p.n_kv_head * a.own_tiles * a.own_splits;
    a.slots = a.shared_splits + a.own_splits;
}

size_t attn_shared_work_bytes(const AttnSharedArgs &a) {
    return (size_t)a.n_seq * a.n_query * a.n_head * a.slots * (a.p.head_dim + 2) * 4;
}

cudaError_t launch_attn_shared(const AttnSharedArgs &a, bool bf16, cudaStream_t s) {
    if (a.p.head_dim == 64) return bf16 ? launch<__nv_bfloat16, 64>(a, s) : launch<__half, 64>(a, s);
    return bf16 ? launch<__nv_bfloat16, 128>(a, s) : launch<__half, 128>(a, s);
}

}  // namespace w4j
