// attn_shared.cuh — arguments of the shared-prefix attention (k_attn_shared.cu).
#pragma once
#include "pages.cuh"

namespace w4j {

struct AttnSharedArgs {
    PagesArgs p;
    int layer, n_head, rep, n_query, n_seq, n_group, max_shared, max_own;
    float scale_log2;                // scale x log2 e
    const void *q;
    void *out;
    long long q_stride, out_stride;
    const int *rows, *group_start, *shared;
    float *part_o, *part_ml;         // [query token][head][slot][head_dim], [..][slot][2] (maximum in base 2, sum)
    // the split of the work (attn_shared_plan)
    int direct;                      // all by k_attn_direct on clusters of so many blocks, no scratch (0: not)
    int tile_rows;                   // query rows of a warp's tile, 8 or 16
    unsigned tc_tiles;               // shared keys by k_attn_shared_tc, in tiles of 128 rows (0: warp tiles)
    unsigned shared_tiles, shared_splits, own_tiles, own_splits, slots;
    unsigned withhold;               // test hook: bytes that every wait for keys or values counts on in vain
    unsigned shared_items, own_items;  // below 2^28: at most 2^24 query rows, and more splits only where there are few
};

void attn_shared_plan(AttnSharedArgs &a);
size_t attn_shared_work_bytes(const AttnSharedArgs &a);
cudaError_t launch_attn_shared(const AttnSharedArgs &a, bool bf16, cudaStream_t s);

}  // namespace w4j
