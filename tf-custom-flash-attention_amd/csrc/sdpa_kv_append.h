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
    AxesArgs axes;  // (positions [axes][T] instead of the places, where some are used)
};

// Queries without keys are taken by four rows per group of lanes from so many waves of such on,
// where seven eighths of the rows are heads.  us by one row and by four, D 128:
//   waves (fp16, 32 heads): 512 4.8 and 5.6, 1024 6.5 and 7.1, 2048 11.7 and 10.7, 4096 18.0 and 14.7, 8643 35.4 and
//     33.9; fp32 (two waves a token): 1024 6.0 and 6.4, 2048 10.1 and 10.0, 4096 16.1 and 14.1
//   heads (fp16, 32 rows a wave, 8643 tokens): 8 11.8 and 16.4, 16 18.5 and 20.6, 24 25.2 and 24.2, 28 29.3 and
//     27.0, 40 43 and 43, 48 50 and 48.7, 96 97 and 88; 2100 tokens: 24 9.1 and 9.9, 28 11.2 and 10.6, 40 12.5 and 13.9
constexpr int kAppendFewWaves = 2048;
hipError_t launch_kv_append(const AppendParams& p, DType dtype, hipStream_t stream);

// The same into a cache in 4 bits (sdpa_kv_fp4.hip; all bytes of a page's head in
// a row), and its tokens out again.  D_qk and D_v are multiples of 32.
struct Fp4ReadParams {
    PagedBatch batch;
    const void* k_cache;
    const void* v_cache;
    void* k;  // [T, H_kv, D_qk]
    void* v;  // [T, H_kv, D_v]
    int H_kv, D_qk, D_v;
};
// From so many windows of 8 tokens (and heads) on a wave takes 8 tokens, else one.  us of the
// append by one token and by 8, 32 query heads on 8, D 128: a prompt of 512 tokens (512 windows) 18 and
// 21, 1024 23 and 20.5, 2048 44 and 23; single tokens of as many sequences 18 and 35, 38 and 41,
// 102 and 69.
constexpr int kFp4FewWindows = 1024;
hipError_t launch_kv_append_fp4(const AppendParams& p, DType dtype, hipStream_t stream);
hipError_t launch_kv_read_fp4(const Fp4ReadParams& p, DType dtype, hipStream_t stream);

}  // namespace sdpa
