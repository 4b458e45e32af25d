// sdpa_kv_append.h -- arguments and launcher of the append to a paged cache
// (sdpa_kv_append.hip), and the batch description that it shares with the
// attention over such a cache (sdpa_paged.h).
#pragma once

#include "sdpa_launch.h"
#include "sdpa_rope.h"

namespace sdpa {

// N sequences.  Sequence s has the new tokens q_starts[s] .. q_starts[s + 1] - 1
// of the T packed ones and kv_lens[s] cached ones, the new ones last; cached
// token j lies in row j % page of page page_table[s][j / page].
// All three arrays are device memory; what they hold is checked where it is
// used: nothing outside the T tokens, the table's `width` columns and the
// `pages` pages is touched.
struct PagedBatch {
    const int32_t* page_table;  // [N, width], rows table_stride apart
    const int32_t* q_starts;    // [N + 1]
    const int32_t* kv_lens;     // [N]
    long long table_stride;
    int N, T, width, pages;
    int page_log2;  // tokens per page
};

// Strides, in elements, of a [T, H, D] tensor whose features are dense.
struct TokenStrides {
    long long t, h;
};

struct AppendParams {
    PagedBatch batch;
    const void* q;  // [T, H_q, D_qk] or null, and where it goes
    void* q_out;
    const void* k;  // [T, H_kv, D_qk]
    const void* v;  // [T, H_kv, D_v]
    void* k_cache;  // [pages, H_kv, page, D_qk]
    void* v_cache;  // [pages, H_kv, page, D_v]
    const void* q_weight;
    const void* k_weight;
    TokenStrides qs, qos, ks, vs;
    RopeArgs r;
    int H_kv;           // heads of the caches
    int H_q, H_k, H_v;  // heads whose rows are taken: none of those without features
    int D_qk, D_v;
    int interleaved, w32, vec;
};

hipError_t launch_kv_append(const AppendParams& p, DType dtype, hipStream_t stream);

}  // namespace sdpa
