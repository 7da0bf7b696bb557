// k_pages.cu — pages of a key/value cache: growing, writing, forking, freeing and compacting.
//
// A cache is a pool of pages [2 n_layer][n_pages][n_kv_head][page_tokens][head_dim] (plane 2 l holds layer
// l's keys, 2 l + 1 its values), the number of rows that hold each page (ref), and each row's page table
// and length.  A page is free when nobody holds it; new pages are the lowest free ones, in the order of
// the call's rows, so that every call has one answer.
//
// Mathematics.  A call is a permutation-like update of integers (who holds which page) plus the tokens it
// has to move.  The integers go through one thread-block cluster: a few passes over the call's rows and
// over `ref` with a cluster barrier between them (barrier.cluster, no grid barrier and no second launch),
// the free list by prefix sums over slices of `ref`.  The tokens are moved by a second kernel on all SMs
// from a list of (source, destination, tokens) that the first one leaves.  The first is bound by the
// latency of its four or five dependent passes over L2, the second by HBM.
//
// Every call is all or nothing: the cluster checks all rows, lengths and the number of free pages before
// its first write, and a call that cannot be done raises a bit of `status` and changes nothing else.
#include "host_api.cuh"
#include "pages.cuh"
#include "w4j_internal.cuh"

namespace w4j {

namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanCluster = 8;

// what a call leaves for its second kernel and for the next pass of its own, in the caller's workspace
enum { H_PAIRS = 0, H_BAD = 1, H_COUNT = 8, H_MORE = 16, H_SIZE = 32 };  // H_COUNT, H_MORE: one word per block

struct Work {
    int *head, *list, *mark, *owner, *rank, *slen, *from, *to, *tokens, *stage;
    __host__ __device__ Work(const PagesArgs &p) {
        const size_t r = p.n_rows, n = p.n_pages, most = r > n ? r : n;
        head = p.work;
        list = head + H_SIZE;      // free pages, or the holes of a compaction
        mark = list + n;           // the call's index of each row, -1 where it has none
        owner = mark + r;          // fork: the first destination that takes a row over
        rank = owner + r;
        slen = rank + r;
        from = slen + r;
        to = from + most;
        tokens = to + most;
        stage = tokens + most;     // fork: the source rows' tables; compaction: the high pages, then the map
    }
};

__device__ __forceinline__ int cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return (int)r;
}
__device__ __forceinline__ int cluster_size() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return (int)r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive prefix sum over the block's threads; `total` gets the sum.  All threads call it.
__device__ __forceinline__ int block_scan(int v, int *sm, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the last call's sums have been read
    if (lane == 31) sm[warp] = x;
    __syncthreads();
    int base = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) {
        const int t = sm[w];
        if (w < warp) base += t;
        sum += t;
    }
    total = sum;
    return base + x - v;
}

__device__ __forceinline__ int held_pages(const PagesArgs &p, int len) { return (len + p.page_tokens - 1) / p.page_tokens; }
__device__ __forceinline__ int row_len(const PagesArgs &p, int r) {
    const int n = __ldcg(p.len + r);
    return n < 0 ? 0 : min(n, p.width * p.page_tokens);
}

// Marks the rows of the call (mark[row] = its index) and finds rows that are out of range or named twice.
// `mark` is -1 everywhere before.
__device__ __forceinline__ void mark_rows(const PagesArgs &p, const Work &w, const int *rows, int n, int gid, int nt) {
    for (int i = gid; i < n; i += nt) {
        const int r = rows[i];
        if (r < 0 || r >= p.n_rows || atomicExch(w.mark + r, i) != -1) atomicOr(w.head + H_BAD, W4J_PAGES_BAD_ROW);
    }
}

// The block's slice of the pages.
__device__ __forceinline__ void page_slice(const PagesArgs &p, int &lo, int &hi) {
    const int per = (p.n_pages + cluster_size() - 1) / cluster_size();
    lo = min(p.n_pages, cluster_rank() * per);
    hi = min(p.n_pages, lo + per);
}

__device__ __forceinline__ void count_free(const PagesArgs &p, const Work &w, int *sm) {
    int lo, hi, n = 0, total;
    page_slice(p, lo, hi);
    for (int i = lo + threadIdx.x; i < hi; i += kPlanThreads) n += __ldcg(p.ref + i) <= 0;
    block_scan(n, sm, total);
    if (threadIdx.x == 0) w.head[H_COUNT + cluster_rank()] = total;
}

// The lowest `need` free pages into w.list (after count_free and a barrier).
__device__ __forceinline__ void list_free(const PagesArgs &p, const Work &w, int need, int *sm) {
    int lo, hi, base = 0;
    page_slice(p, lo, hi);
    for (int b = 0; b < cluster_rank(); ++b) base += __ldcg(w.head + H_COUNT + b);
    for (int i0 = lo; i0 < hi && base < need; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x;
        const int f = i < hi && __ldcg(p.ref + i) <= 0;
        int total;
        const int at = base + block_scan(f, sm, total);
        if (f && at < need) w.list[at] = i;
        base += total;
    }
}

__device__ __forceinline__ int all_free(const Work &w) {
    int n = 0;
    for (int b = 0; b < cluster_size(); ++b) n += __ldcg(w.head + H_COUNT + b);
    return n;
}

__device__ __forceinline__ void start_plan(const PagesArgs &p, const Work &w, int gid, int nt) {
    pdl_wait();
    pdl_trigger();
    for (int i = gid; i < p.n_rows; i += nt) w.mark[i] = -1, w.owner[i] = 0x7fffffff;
    if (gid == 0) w.head[H_PAIRS] = 0, w.head[H_BAD] = 0;
}

// Whether the call can go on; raises its status bits where it cannot.  The same answer in every thread.
__device__ __forceinline__ bool go_on(const PagesArgs &p, const Work &w, int more, int gid) {
    const int bad = __ldcg(w.head + H_BAD) | more;
    if (bad && gid == 0) atomicOr(p.status, bad);
    return bad == 0;
}

// ---------------------------------------------------------------------------
// fork: row dst[i] becomes what row src[i] was before the call (src -1: empty).  Full pages are held by
// both; a last page that is not full stays with one holder (the source row if it goes on, else the first
// row that takes it over) and every other one gets a copy of its tokens on a page of its own.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kPlanThreads) k_pages_fork(PagesArgs p, const int *__restrict__ dst,
                                                             const int *__restrict__ src, int n) {
    __shared__ int sm[kPlanWarps];
    const Work w(p);
    const int nt = cluster_size() * kPlanThreads, gid = cluster_rank() * kPlanThreads + threadIdx.x;
    const int lane = threadIdx.x & 31, gw = gid >> 5, nw = nt >> 5;
    start_plan(p, w, gid, nt);
    cluster_barrier();
    mark_rows(p, w, dst, n, gid, nt);
    for (int i = gid; i < n; i += nt) {
        const int s = src[i];
        if (s < -1 || s >= p.n_rows)
            atomicOr(w.head + H_BAD, W4J_PAGES_BAD_ROW);
        else if (s >= 0)
            atomicMin(w.owner + s, i);
    }
    for (int i = gw; i < n; i += nw) {  // the source rows as they were
        const int s = src[i];
        const bool ok = s >= 0 && s < p.n_rows;
        const int len = ok ? row_len(p, s) : 0, np = held_pages(p, len);
        if (lane == 0) w.slen[i] = len;
        for (int j = lane; j < np; j += 32) {
            const int page = __ldcg(p.table + (size_t)s * p.width + j);
            if (page < 0 || page >= p.n_pages) atomicOr(w.head + H_BAD, W4J_PAGES_BAD_PAGE);
            w.stage[(size_t)i * p.width + j] = page;
        }
    }
    for (int i = gw; i < n; i += nw) {  // the pages that the call lets go of
        const int d = dst[i];
        if (d < 0 || d >= p.n_rows) continue;
        const int np = held_pages(p, row_len(p, d));
        for (int j = lane; j < np; j += 32) {
            const int page = __ldcg(p.table + (size_t)d * p.width + j);
            if (page < 0 || page >= p.n_pages) atomicOr(w.head + H_BAD, W4J_PAGES_BAD_PAGE);
        }
    }
    count_free(p, w, sm);
    cluster_barrier();
    if (!go_on(p, w, 0, gid)) return;
    // who needs a page: every block counts all rows, each writes the ranks of its own chunks
    int need = 0;
    for (int i0 = 0, c = 0; i0 < n; i0 += kPlanThreads, ++c) {
        const int i = i0 + threadIdx.x;
        int copy = 0;
        if (i < n) {
            const int s = src[i], d = dst[i];
            if (s >= 0 && s != d && __ldcg(w.slen + i) % p.page_tokens) {
                const int at = __ldcg(w.mark + s);  // -1: the source row goes on by itself
                copy = at < 0 || src[at] == s || __ldcg(w.owner + s) != i;
            }
        }
        int total;
        const int r = need + block_scan(copy, sm, total);
        if (i < n && c % cluster_size() == cluster_rank()) w.rank[i] = copy ? r : -1;
        need += total;
    }
    const int lack = need > all_free(w) ? W4J_PAGES_FULL : 0;
    if (!go_on(p, w, lack, gid)) return;
    list_free(p, w, need, sm);
    cluster_barrier();
    for (int i = gw; i < n; i += nw) {
        const int s = src[i], d = dst[i];
        if (s == d) continue;
        const int np_old = held_pages(p, row_len(p, d)), len = __ldcg(w.slen + i), np = held_pages(p, len);
        const int r = __ldcg(w.rank + i);
        int *row = p.table + (size_t)d * p.width;
        for (int j = lane; j < max(np_old, np); j += 32) {
            if (j < np_old) atomicSub(p.ref + __ldcg(row + j), 1);
            if (j < np) {
                int page = __ldcg(w.stage + (size_t)i * p.width + j);
                if (r >= 0 && j == np - 1) {
                    const int mine = __ldcg(w.list + r);
                    w.from[r] = page, w.to[r] = mine, w.tokens[r] = len - j * p.page_tokens;
                    page = mine;
                }
                row[j] = page;
                atomicAdd(p.ref + page, 1);
            }
        }
        __syncwarp();
        if (lane == 0) p.len[d] = len;
    }
    if (gid == 0) w.head[H_PAIRS] = need;
}

// ---------------------------------------------------------------------------
// extend: row rows[i] grows by start[i + 1] - start[i] tokens; free: the rows become empty
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kPlanThreads) k_pages_extend(PagesArgs p, const int *__restrict__ rows,
                                                               const int *__restrict__ start, int n) {
    __shared__ int sm[kPlanWarps];
    const Work w(p);
    const int nt = cluster_size() * kPlanThreads, gid = cluster_rank() * kPlanThreads + threadIdx.x;
    const int lane = threadIdx.x & 31, gw = gid >> 5, nw = nt >> 5;
    start_plan(p, w, gid, nt);
    cluster_barrier();
    mark_rows(p, w, rows, n, gid, nt);
    if (gid == 0 && start[0] != 0) atomicOr(w.head + H_BAD, W4J_PAGES_BAD_START);
    for (int i = gid; i < n; i += nt) {
        const int r = rows[i];
        if (r < 0 || r >= p.n_rows) continue;
        const int len = row_len(p, r);
        const long long add = (long long)start[i + 1] - start[i];
        if (add < 0)
            atomicOr(w.head + H_BAD, W4J_PAGES_BAD_START);
        else if (len + add > (long long)p.width * p.page_tokens)
            atomicOr(w.head + H_BAD, W4J_PAGES_TOO_LONG);
        else
            w.slen[i] = held_pages(p, (int)(len + add)) - held_pages(p, len);
    }
    count_free(p, w, sm);
    cluster_barrier();
    if (!go_on(p, w, 0, gid)) return;
    const int have = all_free(w);
    int need = 0;
    for (int i0 = 0, c = 0; i0 < n; i0 += kPlanThreads, ++c) {
        const int i = i0 + threadIdx.x;
        int total;
        // a row asks for `width` pages at most and n rows for more than `have` are refused: no overflow
        const int r = need + block_scan(i < n ? min(__ldcg(w.slen + i), have + 1) : 0, sm, total);
        if (i < n && c % cluster_size() == cluster_rank()) w.rank[i] = r;
        need = min(need + total, have + 1);
    }
    if (!go_on(p, w, need > have ? W4J_PAGES_FULL : 0, gid)) return;
    list_free(p, w, need, sm);
    cluster_barrier();
    for (int i = gw; i < n; i += nw) {
        const int r = rows[i], len = row_len(p, r), had = held_pages(p, len), more = __ldcg(w.slen + i);
        const int at = __ldcg(w.rank + i);
        for (int j = lane; j < more; j += 32) {
            const int page = __ldcg(w.list + at + j);
            p.table[(size_t)r * p.width + had + j] = page;
            p.ref[page] = 1;
        }
        __syncwarp();
        if (lane == 0) p.len[r] = len + start[i + 1] - start[i];
    }
}

__global__ void __launch_bounds__(kPlanThreads) k_pages_free(PagesArgs p, const int *__restrict__ rows, int n) {
    const Work w(p);
    const int nt = cluster_size() * kPlanThreads, gid = cluster_rank() * kPlanThreads + threadIdx.x;
    const int lane = threadIdx.x & 31, gw = gid >> 5, nw = nt >> 5;
    start_plan(p, w, gid, nt);
    cluster_barrier();
    mark_rows(p, w, rows, n, gid, nt);
    for (int i = gw; i < n; i += nw) {
        const int r = rows[i];
        if (r < 0 || r >= p.n_rows) continue;
        const int np = held_pages(p, row_len(p, r));
        for (int j = lane; j < np; j += 32) {
            const int page = __ldcg(p.table + (size_t)r * p.width + j);
            if (page < 0 || page >= p.n_pages) atomicOr(w.head + H_BAD, W4J_PAGES_BAD_PAGE);
        }
    }
    cluster_barrier();
    if (!go_on(p, w, 0, gid)) return;
    for (int i = gw; i < n; i += nw) {
        const int r = rows[i], np = held_pages(p, row_len(p, r));
        for (int j = lane; j < np; j += 32) atomicSub(p.ref + __ldcg(p.table + (size_t)r * p.width + j), 1);
        __syncwarp();
        if (lane == 0) p.len[r] = 0;
    }
}

// ---------------------------------------------------------------------------
// compact: with n pages held, the i-th lowest free page below n gets the i-th lowest held page from n on
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kPlanThreads) k_pages_compact(PagesArgs p, int *__restrict__ live_out) {
    __shared__ int sm[kPlanWarps];
    const Work w(p);
    const int nt = cluster_size() * kPlanThreads, gid = cluster_rank() * kPlanThreads + threadIdx.x;
    const int lane = threadIdx.x & 31, gw = gid >> 5, nw = nt >> 5;
    int *map = w.stage;  // the new place of the pages from `live` on
    start_plan(p, w, gid, nt);
    cluster_barrier();
    count_free(p, w, sm);
    for (int r = gw; r < p.n_rows; r += nw) {
        const int np = held_pages(p, row_len(p, r));
        for (int j = lane; j < np; j += 32) {
            const int page = __ldcg(p.table + (size_t)r * p.width + j);
            if (page < 0 || page >= p.n_pages || __ldcg(p.ref + page) <= 0) atomicOr(w.head + H_BAD, W4J_PAGES_BAD_PAGE);
        }
    }
    cluster_barrier();
    if (!go_on(p, w, 0, gid)) return;
    const int live = p.n_pages - all_free(w);
    int lo, hi, a = 0, b = 0, holes, highs;
    page_slice(p, lo, hi);
    for (int i = lo + threadIdx.x; i < hi; i += kPlanThreads) {
        const bool f = __ldcg(p.ref + i) <= 0;
        a += f && i < live;
        b += !f && i >= live;
    }
    block_scan(a, sm, holes);
    block_scan(b, sm, highs);
    cluster_barrier();  // all_free's words have been read
    if (threadIdx.x == 0) w.head[H_COUNT + cluster_rank()] = holes, w.head[H_MORE + cluster_rank()] = highs;
    cluster_barrier();
    int hole0 = 0, high0 = 0, moves = 0;
    for (int c = 0; c < cluster_size(); ++c) {
        const int x = __ldcg(w.head + H_COUNT + c), y = __ldcg(w.head + H_MORE + c);
        if (c < cluster_rank()) hole0 += x, high0 += y;
        moves += x;
    }
    for (int i0 = lo; i0 < hi; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x;
        const bool f = i < hi && __ldcg(p.ref + i) <= 0;
        const int hole = f && i < live, high = i < hi && !f && i >= live;
        int n1, n2;
        const int r1 = hole0 + block_scan(hole, sm, n1), r2 = high0 + block_scan(high, sm, n2);
        if (hole) w.to[r1] = i, w.tokens[r1] = p.page_tokens;
        if (high) w.from[r2] = i, map[i] = r2;
        hole0 += n1, high0 += n2;
    }
    cluster_barrier();
    for (int k = gid; k < moves; k += nt) {
        const int from = __ldcg(w.from + k), to = __ldcg(w.to + k);
        p.ref[to] = __ldcg(p.ref + from);
        p.ref[from] = 0;
    }
    for (int r = gw; r < p.n_rows; r += nw) {
        const int np = held_pages(p, row_len(p, r));
        for (int j = lane; j < np; j += 32) {
            int *e = p.table + (size_t)r * p.width + j;
            const int page = __ldcg(e);
            if (page >= live) *e = __ldcg(w.to + __ldcg(map + page));
        }
    }
    if (gid == 0) {
        w.head[H_PAIRS] = moves;
        if (live_out) *live_out = live;
    }
}

// ---------------------------------------------------------------------------
// the tokens of the pairs that a plan has left: an item is one plane of one pair
// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 256, kMoveUnroll = 4;

__global__ void __launch_bounds__(kMoveThreads) k_pages_move(PagesArgs p) {
    pdl_wait();
    const Work w(p);
    const int pairs = __ldcg(w.head + H_PAIRS), planes = 2 * p.n_layer;
    const int unit = p.head_dim / 8;  // 16-byte units of a token of one head
    const size_t page_units = (size_t)p.n_kv_head * p.page_tokens * unit, plane_units = page_units * p.n_pages;
    uint4 *pool = reinterpret_cast<uint4 *>(p.pool);
    for (long long item = blockIdx.x; item < (long long)pairs * planes; item += gridDim.x) {
        const int k = (int)(item / planes), plane = (int)(item % planes);
        const uint4 *from = pool + plane * plane_units + __ldcg(w.from + k) * page_units;
        uint4 *to = pool + plane * plane_units + __ldcg(w.to + k) * page_units;
        const int run = __ldcg(w.tokens + k) * unit, whole = p.page_tokens * unit, n = p.n_kv_head * run;
        for (int u0 = threadIdx.x; u0 < n; u0 += kMoveThreads * kMoveUnroll) {
            uint4 v[kMoveUnroll];
            int at[kMoveUnroll];
#pragma unroll
            for (int i = 0; i < kMoveUnroll; ++i) {
                const int u = u0 + i * kMoveThreads;
                at[i] = u / run * whole + u % run;  // the held tokens of each head
                if (u < n) v[i] = from[at[i]];
            }
#pragma unroll
            for (int i = 0; i < kMoveUnroll; ++i)
                if (u0 + i * kMoveThreads < n) to[at[i]] = v[i];
        }
    }
}

// ---------------------------------------------------------------------------
// write: the keys and values of the last start[i + 1] - start[i] tokens of row rows[i], a warp per token
// ---------------------------------------------------------------------------
constexpr int kWriteWarps = 8;

__global__ void __launch_bounds__(kWriteWarps * 32) k_pages_write(PagesArgs p, int layer, const int *__restrict__ rows,
                                                                  const int *__restrict__ start, int n,
                                                                  const uint4 *__restrict__ k, const uint4 *__restrict__ v,
                                                                  long long k_stride, long long v_stride, int n_tokens) {
    pdl_wait();
    const int t = blockIdx.x * kWriteWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (t >= n_tokens) return;
    if (t == 0 && lane == 0 && (start[0] != 0 || start[n] != n_tokens)) atomicOr(p.status, W4J_PAGES_BAD_START);
    // the last i with start[i] <= t, 32 places at a time
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, at < hi && start[at] <= t);
        const int last = m ? 31 - __clz(m) : 0;
        lo += last * step;
        hi = min(hi, lo + step);
    }
    const int r = rows[lo], s0 = start[lo], s1 = start[lo + 1];
    if (t < s0 || t >= s1) return;  // behind the last sequence, or a start that does not ascend (reported above)
    const bool row_ok = r >= 0 && r < p.n_rows;
    const long long pos = row_ok ? (long long)row_len(p, r) - s1 + t : -1;
    if (pos < 0) {
        if (lane == 0) atomicOr(p.status, row_ok ? W4J_PAGES_BAD_START : W4J_PAGES_BAD_ROW);
        return;
    }
    const int j = (int)(pos / p.page_tokens), tok = (int)(pos % p.page_tokens);
    const int page = __ldcg(p.table + (size_t)r * p.width + j);
    if (page < 0 || page >= p.n_pages) {
        if (lane == 0) atomicOr(p.status, W4J_PAGES_BAD_PAGE);
        return;
    }
    const int unit = p.head_dim / 8, n_units = p.n_kv_head * unit;
    const size_t page_units = (size_t)n_units * p.page_tokens;
    uint4 *pool = reinterpret_cast<uint4 *>(p.pool);
    uint4 *kd = pool + ((size_t)(2 * layer) * p.n_pages + page) * page_units + (size_t)tok * unit;
    uint4 *vd = kd + (size_t)p.n_pages * page_units;
    const uint4 *ks = k + t * k_stride, *vs = v + t * v_stride;
    const int whole = p.page_tokens * unit;
    for (int u = lane; u < n_units; u += 32) {
        const int at = u / unit * whole + u % unit;
        kd[at] = ks[u];
        vd[at] = vs[u];
    }
}

int plan_blocks(const PagesArgs &p, long long entries) {
    // one block answers sooner while its passes are short (a cluster barrier costs more than a block's)
    return entries <= 4096 && p.n_pages <= 8192 && p.n_rows <= 4096 ? 1 : kPlanCluster;
}

int move_blocks(const PagesArgs &p, long long pairs) {
    const long long items = pairs * 2 * p.n_layer, most = 148 * 8;
    return (int)(items < most ? (items < 1 ? 1 : items) : most);
}

}  // namespace

size_t pages_work_bytes(const PagesArgs &p) {
    const size_t r = p.n_rows, n = p.n_pages, most = r > n ? r : n;
    const size_t stage = r * p.width > n ? r * p.width : n;
    return 4 * (H_SIZE + n + 4 * r + 3 * most + stage);
}

cudaError_t launch_pages_fork(const PagesArgs &p, const int *dst, const int *src, int n, cudaStream_t s) {
    const int nb = plan_blocks(p, (long long)n * p.width);
    cudaError_t e = launch_after(k_pages_fork, nb, kPlanThreads, 0, s, nb, p, dst, src, n);
    if (e != cudaSuccess) return e;
    return launch_after(k_pages_move, move_blocks(p, n), kMoveThreads, 0, s, 1, p);
}

cudaError_t launch_pages_extend(const PagesArgs &p, const int *rows, const int *start, int n, cudaStream_t s) {
    const int nb = plan_blocks(p, (long long)n * p.width);
    return launch_after(k_pages_extend, nb, kPlanThreads, 0, s, nb, p, rows, start, n);
}

cudaError_t launch_pages_free(const PagesArgs &p, const int *rows, int n, cudaStream_t s) {
    const int nb = plan_blocks(p, (long long)n * p.width);
    return launch_after(k_pages_free, nb, kPlanThreads, 0, s, nb, p, rows, n);
}

cudaError_t launch_pages_compact(const PagesArgs &p, int *live, cudaStream_t s) {
    const int nb = plan_blocks(p, (long long)p.n_rows * p.width);
    cudaError_t e = launch_after(k_pages_compact, nb, kPlanThreads, 0, s, nb, p, live);
    if (e != cudaSuccess) return e;
    return launch_after(k_pages_move, move_blocks(p, p.n_pages / 2), kMoveThreads, 0, s, 1, p);
}

cudaError_t launch_pages_write(const PagesArgs &p, int layer, const int *rows, const int *start, int n, const void *k,
                               const void *v, long long k_stride, long long v_stride, int n_tokens, cudaStream_t s) {
    return launch_after(k_pages_write, (n_tokens + kWriteWarps - 1) / kWriteWarps, kWriteWarps * 32, 0, s, 1, p, layer, rows,
                        start, n, reinterpret_cast<const uint4 *>(k), reinterpret_cast<const uint4 *>(v), k_stride / 8,
                        v_stride / 8, n_tokens);
}

}  // namespace w4j
