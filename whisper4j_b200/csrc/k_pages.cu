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
// latency of its dependent passes over L2, the second by HBM.  A call whose lists fit one block's registers and
// shared memory takes one block that reads everything once (k_pages_small), a fork of more rows a cluster of such blocks:
// three passes instead of five.
//
// Every call but a write is all or nothing: the cluster checks all rows, lengths and the number of free pages before
// its first write, and a call that cannot be done raises a bit of `status` and changes nothing else.  A write leaves out
// the tokens that have no place.
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

// What a row's last extension leaves for the writes that follow it: the row's index in its list, or this number and the bits
// that refused it.  The row's length has not grown then, and its new tokens' places would be those of its last ones, on
// pages that other rows may hold too.  (Scratch that nobody has set to zero looks refused once in 2^24.)
constexpr int kRefused = 0x57346a00, kRefusedBits = 0xff;

struct Work {
    int *head, *outcome, *list, *mark, *owner, *rank, *slen, *from, *to, *tokens, *stage;
    __host__ __device__ Work(const PagesArgs &p) {
        const size_t r = p.n_rows, n = p.n_pages, most = r > n ? r : n;
        head = p.work;
        outcome = head + H_SIZE;   // of each row's last extension, kept from call to call: nothing else writes it
        list = outcome + r;        // free pages, or the holes of a compaction
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

// A table entry that names no page that somebody holds.
__device__ __forceinline__ bool no_page(const PagesArgs &p, int page) {
    return page < 0 || page >= p.n_pages || __ldcg(p.ref + page) <= 0;
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

// The outcome of an extension for the rows it names (threads gid of nt), `bad` the bits that refused it.
__device__ __forceinline__ void note_outcome(const PagesArgs &p, const Work &w, const int *rows, int n, int bad, int gid, int nt) {
    for (int i = gid; i < n; i += nt) {
        const int r = rows[i];
        if (r >= 0 && r < p.n_rows) w.outcome[r] = bad ? kRefused | bad : i;
    }
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
            if (no_page(p, page)) atomicOr(w.head + H_BAD, W4J_PAGES_BAD_PAGE);
            w.stage[(size_t)i * p.width + j] = page;
        }
    }
    for (int i = gw; i < n; i += nw) {  // the pages that the call lets go of
        const int d = dst[i];
        if (d < 0 || d >= p.n_rows) continue;
        const int np = held_pages(p, row_len(p, d));
        for (int j = lane; j < np; j += 32) {
            const int page = __ldcg(p.table + (size_t)d * p.width + j);
            if (no_page(p, page)) atomicOr(w.head + H_BAD, W4J_PAGES_BAD_PAGE);
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
    if (!go_on(p, w, 0, gid)) return note_outcome(p, w, rows, n, __ldcg(w.head + H_BAD), gid, nt);
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
    const int lack = need > have ? W4J_PAGES_FULL : 0;
    note_outcome(p, w, rows, n, lack, gid, nt);
    if (!go_on(p, w, lack, gid)) return;
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
            if (no_page(p, page)) atomicOr(w.head + H_BAD, W4J_PAGES_BAD_PAGE);
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
            if (no_page(p, page)) atomicOr(w.head + H_BAD, W4J_PAGES_BAD_PAGE);
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
// the same calls by one block: the call's lists, the marks of the rows and the free list in shared memory, `ref` (kRefs
// neighbouring pages a thread) and the tables' entries (32 neighbouring ones a warp and step, kEntries steps) in
// registers, each read once.  As many warps as that takes and no more: with all 32 every instruction holds a scheduler
// for eight cycles (a beam reorder of 5 rows: 8.4 us with 1024 threads, 7.4 with as many as it needs).
// ---------------------------------------------------------------------------
enum PagesOp { OP_FORK, OP_EXTEND, OP_FREE, OP_COMPACT };
constexpr int kSmallThreads = 1024, kRefs = 8 /* the bits of a byte */, kEntries = 12;

// Exclusive prefix sum over the block's threads.
__device__ __forceinline__ int small_scan(int v, int *sm, int &total) {
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
    int y = lane < (int)blockDim.x / 32 ? sm[lane] : 0;
    const int mine = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    total = __shfl_sync(0xffffffffu, y, 31);
    return __shfl_sync(0xffffffffu, y - mine, warp) + x - v;
}

struct SmallRows {  // of the n rows of a call, and of all rows
    int *a, *b, *len_a, *len_b, *rank, *mark, *owner, *list, *more;  // more: what the call adds to each page's count
    __device__ SmallRows(int *sm, int n, int n_rows, int n_pages) {
        a = sm, b = a + n, len_a = b + n, len_b = len_a + n, rank = len_b + n, mark = rank + n, owner = mark + n_rows, list = owner + n_rows;
        more = list + n_pages;
    }
};
size_t small_bytes(const PagesArgs &p, int n) { return 4 * (5 * (size_t)n + 2 * (size_t)p.n_rows + 2 * (size_t)p.n_pages); }

// a, b: dst and src (fork), rows and start (extend), rows (free), n_live (compact: the call's rows are all of them)
template <PagesOp OP, bool MANY>
__global__ void __launch_bounds__(kSmallThreads) k_pages_small(PagesArgs p, const int *__restrict__ a, const int *__restrict__ b,
                                                               int *live_out, int n) {
    extern __shared__ int dyn[];
    __shared__ int sm[32], bad;
    __shared__ unsigned char held[kSmallThreads];  // bit i of byte t: somebody holds page t kRefs + i
    const Work w(p);
    const SmallRows s(dyn, n, p.n_rows, p.n_pages);
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, T = p.page_tokens, W = p.width;
    // step x of a warp: 32 entries (runs of 32 in each row) of row i from j0 on
    const int blocks = MANY ? cluster_size() : 1, block = MANY ? cluster_rank() : 0;
    const int runs = (W + 31) / 32, steps = n * runs, warps = blocks * (threads / 32), first = block * (threads / 32) + tid / 32;
    auto row_of = [&](int step, int &j) {
        const int i = runs == 1 ? step : step / runs;
        j = (step - i * runs) * 32 + lane;
        return i;
    };
    pdl_wait();
    pdl_trigger();
    int ref[kRefs];
    if (tid * kRefs + kRefs <= p.n_pages && reinterpret_cast<uintptr_t>(p.ref) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < kRefs; i += 4) *reinterpret_cast<int4 *>(ref + i) = *reinterpret_cast<const int4 *>(p.ref + tid * kRefs + i);
    } else {
#pragma unroll
        for (int i = 0; i < kRefs; ++i) ref[i] = tid * kRefs + i < p.n_pages ? p.ref[tid * kRefs + i] : 1;
    }
    if (OP != OP_EXTEND) {
        int bits = 0;
#pragma unroll
        for (int i = 0; i < kRefs; ++i) bits |= (ref[i] > 0) << i;
        held[tid] = (unsigned char)bits;
    }
    if (OP != OP_COMPACT) {
        for (int i = tid; i < n; i += threads) {
            s.a[i] = a[i];
            if (OP != OP_FREE) s.b[i] = b[i];
        }
        for (int i = tid; i < p.n_rows; i += threads) s.mark[i] = -1, s.owner[i] = 0x7fffffff;
        for (int i = tid; i < p.n_pages; i += threads) s.more[i] = 0;
    }
    if (tid == 0) bad = OP == OP_EXTEND && b[0] != 0 ? W4J_PAGES_BAD_START : 0;
    if (tid == 0 && block == 0) w.head[H_PAIRS] = 0;
    __syncthreads();
    if (MANY) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this block's `bad` is there
    for (int i = tid; i < n; i += threads) {
        const int r = OP == OP_COMPACT ? i : s.a[i];
        if (r < 0 || r >= p.n_rows || (OP != OP_COMPACT && atomicExch(s.mark + r, i) != -1)) {
            atomicOr(&bad, W4J_PAGES_BAD_ROW);
            s.len_a[i] = s.len_b[i] = 0;
            continue;
        }
        s.len_a[i] = row_len(p, r);
        if (OP == OP_FORK) {
            const int from = s.b[i];
            if (from < -1 || from >= p.n_rows) atomicOr(&bad, W4J_PAGES_BAD_ROW);
            const bool ok = from >= 0 && from < p.n_rows;
            if (ok) atomicMin(s.owner + from, i);
            s.len_b[i] = ok ? row_len(p, from) : 0;
        }
        if (OP == OP_EXTEND) {
            const long long add = (long long)(i + 1 < n ? s.b[i + 1] : b[n]) - s.b[i], len = s.len_a[i] + add;
            if (add < 0) atomicOr(&bad, W4J_PAGES_BAD_START);
            if (len > (long long)W * T) atomicOr(&bad, W4J_PAGES_TOO_LONG);
            s.len_b[i] = add < 0 || len > (long long)W * T ? s.len_a[i] : (int)len;
        }
    }
    __syncthreads();
    // what row a holds at the entries of this thread's steps, and what it shall hold (-1: nothing): all of them on
    // their way before the first is looked at
    int was[kEntries], shall[kEntries];
#pragma unroll
    for (int x = 0; x < kEntries; ++x) {
        was[x] = shall[x] = -1;
        const int step = first + x * warps;
        if (OP == OP_EXTEND || step >= steps) continue;
        int j;
        const int i = row_of(step, j), r = OP == OP_COMPACT ? i : s.a[i];
        if (j * T < s.len_a[i]) was[x] = __ldcg(p.table + (size_t)r * W + j);
        if (OP == OP_FORK && j * T < s.len_b[i]) shall[x] = __ldcg(p.table + (size_t)s.b[i] * W + j);
    }
    if (OP != OP_EXTEND) {
        bool out = false;
        auto no_page = [&](int page) { return page < 0 || page >= p.n_pages || !(held[page / kRefs] >> page % kRefs & 1); };
#pragma unroll
        for (int x = 0; x < kEntries; ++x) {
            const int step = first + x * warps;
            if (step >= steps) continue;
            int j;
            const int i = row_of(step, j);
            const bool in_a = j * T < s.len_a[i], in_b = OP == OP_FORK && j * T < s.len_b[i];
            if (in_a && no_page(was[x])) out = true, was[x] = -1;
            if (in_b && no_page(shall[x])) out = true, shall[x] = -1;
        }
        if (out) atomicOr(&bad, W4J_PAGES_BAD_PAGE);
    }
    auto add_more = [&]() {
#pragma unroll
        for (int i = 0; i < kRefs; ++i) {
            const int page = tid * kRefs + i;
            if (page >= p.n_pages || !s.more[page]) continue;
            if (MANY)
                atomicAdd(p.ref + page, s.more[page]);
            else
                p.ref[page] = ref[i] + s.more[page];
        }
    };
    if (OP == OP_FREE) {
        __syncthreads();
        if (bad) {
            if (tid == 0) atomicOr(p.status, bad);
            return;
        }
#pragma unroll
        for (int x = 0; x < kEntries; ++x)
            if (was[x] >= 0) atomicSub(s.more + was[x], 1);
        for (int i = tid; i < n; i += threads) p.len[s.a[i]] = 0;
        __syncthreads();
        add_more();
        return;
    }
    // free pages below this thread's
    int mine = 0, free_pages;
#pragma unroll
    for (int i = 0; i < kRefs; ++i) mine += ref[i] <= 0;
    const int free_before = small_scan(mine, sm, free_pages);
    if (OP == OP_COMPACT) {
        const int live = p.n_pages - free_pages;
        __syncthreads();
        if (bad) {
            if (tid == 0) atomicOr(p.status, bad);
            return;
        }
        // the i-th hole below `live` and the i-th held page from it on, by their places in the list
        int *to = s.list, hole = free_before, moves, highs = 0;
#pragma unroll
        for (int i = 0; i < kRefs; ++i) {
            const int page = tid * kRefs + i;
            if (page < live && ref[i] <= 0) to[hole++] = page;
            highs += page >= live && page < p.n_pages && ref[i] > 0;
        }
        int high = small_scan(highs, sm, moves);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRefs; ++i) {
            const int page = tid * kRefs + i;
            if (page < live || page >= p.n_pages || ref[i] <= 0) continue;
            w.from[high] = page, w.to[high] = to[high], w.tokens[high] = T;
            p.ref[to[high]] = ref[i];
            p.ref[page] = 0;
            w.stage[page] = to[high++];
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < kEntries; ++x)
            if (was[x] >= live) {
                int j;
                const int i = row_of(first + x * warps, j);
                p.table[(size_t)i * W + j] = w.stage[was[x]];
            }
        if (tid == 0) {
            w.head[H_PAIRS] = moves;
            if (live_out) *live_out = live;
        }
        return;
    }
    // pages that each row needs
    int need = 0;
    for (int i0 = 0; i0 < n; i0 += threads) {
        const int i = i0 + tid;
        int want = 0, total;
        if (i < n && OP == OP_FORK) {
            const int from = s.b[i];
            if (from >= 0 && from < p.n_rows && from != s.a[i] && s.len_b[i] % T) {
                const int at = s.mark[from];  // -1: the source row goes on by itself
                want = at < 0 || s.b[at] == from || s.owner[from] != i;
            }
        }
        if (i < n && OP == OP_EXTEND) want = min(held_pages(p, s.len_b[i]) - held_pages(p, s.len_a[i]), free_pages + 1);
        const int r = need + small_scan(want, sm, total);
        if (i < n) s.rank[i] = OP == OP_FORK && !want ? -1 : r;
        need = min(need + total, free_pages + 1);
    }
    int at = free_before;
#pragma unroll
    for (int i = 0; i < kRefs; ++i)
        if (ref[i] <= 0 && at < need) s.list[at++] = tid * kRefs + i;
    if (need > free_pages && tid == 0) atomicOr(&bad, W4J_PAGES_FULL);
    __syncthreads();
    if (MANY) {  // what one has found holds for all; and all have read what follows writes
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (tid < blocks && bad) {
            uint32_t at;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&bad)), "r"(tid));
            asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(at), "r"(bad) : "memory");
        }
        cluster_barrier();
    }
    if (OP == OP_EXTEND) note_outcome(p, w, s.a, n, bad, tid, threads);
    if (bad) {
        if (tid == 0 && block == 0) atomicOr(p.status, bad);
        return;
    }
#pragma unroll
    for (int x = 0; x < kEntries; ++x) {
        const int step = first + x * warps;
        if (step >= steps) break;
        int j;
        const int i = row_of(step, j);
        if (j >= W) continue;
        int *entry = p.table + (size_t)s.a[i] * W + j;
        if (OP == OP_EXTEND) {
            const int had = held_pages(p, s.len_a[i]);
            if (j < had || j >= held_pages(p, s.len_b[i])) continue;
            const int page = s.list[s.rank[i] + j - had];
            *entry = page;
            p.ref[page] = 1;
        }
        if (OP == OP_FORK && s.a[i] != s.b[i]) {
            const int r = s.rank[i];
            if (r >= 0 && shall[x] >= 0 && (j + 1) * T > s.len_b[i]) {  // the last page, not full
                w.from[r] = shall[x], w.to[r] = s.list[r], w.tokens[r] = s.len_b[i] - j * T;
                shall[x] = s.list[r];
            }
            if (was[x] == shall[x]) continue;  // what beams have in common
            if (was[x] >= 0) atomicSub(s.more + was[x], 1);
            if (shall[x] >= 0) *entry = shall[x], atomicAdd(s.more + shall[x], 1);
        }
    }
    if (block == 0)
        for (int i = tid; i < n; i += threads) p.len[s.a[i]] = s.len_b[i];
    if (OP == OP_FORK) {
        if (tid == 0 && block == 0) w.head[H_PAIRS] = need;
        __syncthreads();
        add_more();
    }
}

// ---------------------------------------------------------------------------
// the tokens of the pairs that a plan has left: an item is one plane of one pair, four 16-byte units of a thread on their
// way at a time.  Bound by HBM: 928 pages of 327 KB move in 97 us, 6.3 TB/s both ways.
// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 256, kMoveUnroll = 4;

__global__ void __launch_bounds__(kMoveThreads) k_pages_move(PagesArgs p) {
    pdl_wait();
    pdl_trigger();
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
// write: the keys and values of the last start[i + 1] - start[i] tokens of row rows[i], a warp per token.  Bound by
// HBM (14368 tokens of 20 heads of 64: 25 us, 5.9 TB/s both ways); few tokens by the four dependent look-ups of their
// place, which their data does not wait for.
//
// A row named twice would have two tokens at one place, in no fixed order.  Its last extension knew it by one index, so at
// most one of its places in this call's list is that one, and writes; a row at any other index is looked up among all rows
// of the call.  (Looking all of them up took 4.4 us instead of 3.0 for 64 rows of one token, marking them in a launch
// before this one 5.4.)
//
// Blocks behind the tokens' look whether start ascends, kStartRun places each, so that no token waits for that.
// ---------------------------------------------------------------------------
constexpr int kWriteWarps = 8, kStartRun = 4096;

__device__ __forceinline__ bool named_twice(const int *rows, int n, int r) {
    constexpr int L = 2;  // (more would cost the kernel registers)
    int named = 0;
    for (int i0 = threadIdx.x & 31; i0 < n; i0 += 32 * L) {
        int other[L];
#pragma unroll
        for (int x = 0; x < L; ++x) other[x] = i0 + 32 * x < n ? rows[i0 + 32 * x] : -1;
#pragma unroll
        for (int x = 0; x < L; ++x) named += other[x] == r;
    }
    return __reduce_add_sync(0xffffffffu, named) > 1;
}

__global__ void __launch_bounds__(kWriteWarps * 32) k_pages_write(PagesArgs p, int layer, const int *__restrict__ rows,
                                                                  const int *__restrict__ start, int n,
                                                                  const uint4 *__restrict__ k, const uint4 *__restrict__ v,
                                                                  long long k_stride, long long v_stride, int n_tokens) {
    pdl_wait();
    pdl_trigger();
    const int token_blocks = (n_tokens + kWriteWarps - 1) / kWriteWarps;
    if ((int)blockIdx.x >= token_blocks) {
        const int i0 = ((int)blockIdx.x - token_blocks) * kStartRun, i1 = min(n, i0 + kStartRun);
        bool wrong = i0 == 0 && (start[0] != 0 || start[n] != n_tokens);
        for (int i = i0 + threadIdx.x; i < i1; i += kWriteWarps * 32) wrong |= start[i] > start[i + 1];
        if (wrong) atomicOr(p.status, W4J_PAGES_BAD_START);
        return;
    }
    const int t = blockIdx.x * kWriteWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (t >= n_tokens) return;
    const int unit = p.head_dim / 8, n_units = p.n_kv_head * unit;
    const uint4 *ks = k + t * k_stride, *vs = v + t * v_stride;
    // the data is on its way while its place is looked up
    constexpr int U = 4;
    uint4 kd[U], vd[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (lane + 32 * i < n_units) kd[i] = __ldg(ks + lane + 32 * i), vd[i] = __ldg(vs + lane + 32 * i);
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
    if (t < s0 || t >= s1) return;  // behind the last sequence, or a start that does not ascend: the last blocks report both
    const bool row_ok = r >= 0 && r < p.n_rows;
    const int outcome = row_ok ? __ldcg(Work(p).outcome + r) : lo, have = row_ok ? row_len(p, r) : 0;
    if ((outcome & ~kRefusedBits) == kRefused) {  // its extension did not take place
        if (lane == 0) atomicOr(p.status, outcome & kRefusedBits);
        return;
    }
    if (outcome != lo && named_twice(rows, n, r)) {
        if (lane == 0) atomicOr(p.status, W4J_PAGES_BAD_ROW);
        return;
    }
    const long long pos = row_ok ? (long long)have - s1 + t : -1;
    if (pos < 0) {
        if (lane == 0) atomicOr(p.status, row_ok ? W4J_PAGES_BAD_START : W4J_PAGES_BAD_ROW);
        return;
    }
    const int j = (int)pos / p.page_tokens, tok = (int)pos - j * p.page_tokens;
    const int page = __ldcg(p.table + (size_t)r * p.width + j);
    if (page < 0 || page >= p.n_pages) {
        if (lane == 0) atomicOr(p.status, W4J_PAGES_BAD_PAGE);
        return;
    }
    const size_t page_units = (size_t)n_units * p.page_tokens;
    uint4 *kp = reinterpret_cast<uint4 *>(p.pool) + ((size_t)(2 * layer) * p.n_pages + page) * page_units + (size_t)tok * unit;
    uint4 *vp = kp + (size_t)p.n_pages * page_units;
    const int whole = p.page_tokens * unit;
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = lane + 32 * i, at = u / unit * whole + u % unit;
        if (u < n_units) kp[at] = kd[i], vp[at] = vd[i];
    }
    for (int u = lane + 32 * U; u < n_units; u += 32) {
        const int at = u / unit * whole + u % unit;
        kp[at] = __ldg(ks + u);
        vp[at] = __ldg(vs + u);
    }
}

// The threads of the one block that takes a call of n rows; 0 where it is too much for one.
int small_threads(const PagesArgs &p, int n) {
    const long long steps = (long long)n * ((p.width + 31) / 32), warps = (steps + kEntries - 1) / kEntries,
                    by_pages = (p.n_pages + 32 * kRefs - 1) / (32 * kRefs), need = warps > by_pages ? warps : by_pages;
    if (need > kSmallThreads / 32 || small_bytes(p, n) > 160 * 1024) return 0;
    return 32 * (int)(need < 4 ? 4 : need);
}

// A fork of more rows: the same by a cluster, whose blocks all plan for all rows and pages and share the tables'
// entries out.  One block's time is its instructions (4 layers of large-v3-turbo, with the move: 5 rows 8.1 us on one, 8.7
// on eight, 40 rows 12.0 and 10.0, 320 rows 19.4 and 14.7; 640 rows 23.4 where k_pages_fork took 37.4;
// the look at who holds the pages has since added 0.1 to 0.5 us, to k_pages_fork 3).
constexpr int kForkBlocks = 8, kForkSteps = 6;
int fork_threads(const PagesArgs &p, int n, int &blocks) {
    const long long steps = (long long)n * ((p.width + 31) / 32), by_pages = (p.n_pages + 32 * kRefs - 1) / (32 * kRefs);
    blocks = 1;
    if (steps < 32) return small_threads(p, n);
    if (by_pages > kSmallThreads / 32 || small_bytes(p, n) > 160 * 1024 || steps > kForkBlocks * kSmallThreads / 32 * kEntries) return 0;
    blocks = kForkBlocks;
    const long long share = (steps + kForkBlocks * kForkSteps - 1) / (kForkBlocks * kForkSteps), need = share > by_pages ? share : by_pages;
    return 32 * (int)(need < 4 ? 4 : need > kSmallThreads / 32 ? kSmallThreads / 32 : need);
}

template <PagesOp OP>
cudaError_t launch_small(const PagesArgs &p, const int *a, const int *b, int *live, int n, int threads, cudaStream_t s, int blocks = 1) {
    if (OP == OP_FORK && blocks > 1)
        return launch_after<k_pages_small<OP, OP == OP_FORK>>(blocks, threads, small_bytes(p, n), s, blocks, p, a, b, live, n);
    return launch_after<k_pages_small<OP, false>>(1, threads, small_bytes(p, n), s, 1, p, a, b, live, n);
}

int move_blocks(const PagesArgs &p, long long pairs) {
    const long long items = pairs * 2 * p.n_layer, most = 148 * 8;
    return (int)(items < most ? (items < 1 ? 1 : items) : most);
}

}  // namespace

size_t pages_work_bytes(const PagesArgs &p) {
    const size_t r = p.n_rows, n = p.n_pages, most = r > n ? r : n;
    const size_t stage = r * p.width > n ? r * p.width : n;
    return 4 * (H_SIZE + n + 5 * r + 3 * most + stage);
}

cudaError_t launch_pages_fork(const PagesArgs &p, const int *dst, const int *src, int n, cudaStream_t s) {
    int blocks;
    const int t = fork_threads(p, n, blocks);
    const cudaError_t e = t ? launch_small<OP_FORK>(p, dst, src, nullptr, n, t, s, blocks)
                            : launch_after<k_pages_fork>(kPlanCluster, kPlanThreads, 0, s, kPlanCluster, p, dst, src, n);
    if (e != cudaSuccess) return e;
    return launch_after<k_pages_move>(move_blocks(p, n), kMoveThreads, 0, s, 1, p);
}

cudaError_t launch_pages_extend(const PagesArgs &p, const int *rows, const int *start, int n, cudaStream_t s) {
    const int t = small_threads(p, n);
    return t ? launch_small<OP_EXTEND>(p, rows, start, nullptr, n, t, s)
             : launch_after<k_pages_extend>(kPlanCluster, kPlanThreads, 0, s, kPlanCluster, p, rows, start, n);
}

cudaError_t launch_pages_free(const PagesArgs &p, const int *rows, int n, cudaStream_t s) {
    const int t = small_threads(p, n);
    return t ? launch_small<OP_FREE>(p, rows, nullptr, nullptr, n, t, s)
             : launch_after<k_pages_free>(kPlanCluster, kPlanThreads, 0, s, kPlanCluster, p, rows, n);
}

cudaError_t launch_pages_compact(const PagesArgs &p, int *live, cudaStream_t s) {
    const int t = small_threads(p, p.n_rows);
    const cudaError_t e = t ? launch_small<OP_COMPACT>(p, nullptr, nullptr, live, p.n_rows, t, s)
                            : launch_after<k_pages_compact>(kPlanCluster, kPlanThreads, 0, s, kPlanCluster, p, live);
    if (e != cudaSuccess) return e;
    return launch_after<k_pages_move>(move_blocks(p, p.n_pages / 2), kMoveThreads, 0, s, 1, p);
}

cudaError_t launch_pages_write(const PagesArgs &p, int layer, const int *rows, const int *start, int n, const void *k,
                               const void *v, long long k_stride, long long v_stride, int n_tokens, cudaStream_t s) {
    const int blocks = (n_tokens + kWriteWarps - 1) / kWriteWarps + (n + kStartRun - 1) / kStartRun;
    return launch_after<k_pages_write>(blocks, kWriteWarps * 32, 0, s, 1, p, layer, rows,
                        start, n, reinterpret_cast<const uint4 *>(k), reinterpret_cast<const uint4 *>(v), k_stride / 8,
                        v_stride / 8, n_tokens);
}

}  // namespace w4j
