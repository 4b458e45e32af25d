// sdpa_reserve.h -- arguments and launcher of the page tables made on the GPU
// (sdpa_reserve.hip).
#pragma once

#include "sdpa_launch.h"

namespace sdpa {

struct ReserveParams {
    int32_t* page_table;  // [N, width], rows table_stride apart
    long long table_stride;
    const int32_t* kv_lens;   // [N] cached tokens before the call
    const int32_t* new_lens;  // [N]
    const uint8_t* finished;  // [N] or null
    int32_t* free_pages;      // [capacity] stack: the first free_count entries
    const int32_t* free_count;
    int32_t* q_starts;        // [N + 1]
    int32_t* kv_lens_out;     // [N], maybe kv_lens
    int32_t* free_count_out;  // [1], maybe free_count
    int32_t* pages_short;     // [1] or null
    int32_t* positions;       // [T]
    int64_t* slots;           // [T]
    int N, T, width, capacity, page_log2;
    int fill;  // the first kernel writes positions and slots too
};

hipError_t launch_kv_reserve(const ReserveParams& p, hipStream_t stream);

}  // namespace sdpa
