// sdpa_paged.h -- attention of new tokens over a paged cache: arguments, and
// how its work is divided over workgroups.
//
// Rows.  The G = H_q / H_kv query heads that share a key head read the same
// keys, so a sequence of n new tokens has, for each key head, n G rows: row
// i G + g is token i, head h G + g.  A tile is up to BM of them.
//
// Division.  The lengths are on the device, so every workgroup forms the plan
// itself, from sums over the sequences; the grid and the workspace go by the call's
// sizes alone.  Two forms, both merged in order by a second kernel:
//   parts   The cost of a tile is the number of key blocks it walks on
//           average; the keys of a tile are divided into parts of at most `chunk`
//           blocks, chunk being the larger of min_chunk and the whole cost over
//           target = 2^target_log2 workgroups.  So at most target workgroups more than there
//           are tiles have work, whatever the lengths, and at most 2 target parts
//           are of divided tiles.
//   shares  The key blocks of all tiles, one tile after the other, are cut into
//           equal shares, one for each of target workgroups, which walks the
//           tiles that its share meets.  It leaves at most two partial tiles: slot
//           2 w holds one that began before its share, 2 w + 1 one that it begins
//           and does not end.  For generation, where a workgroup's time is the
//           keys it reads.
#pragma once

#include "sdpa_kv_append.h"

namespace sdpa {

struct PagedParams {
    PagedBatch batch;
    const void* q;        // [T, H_q, D_qk]
    const void* k_cache;  // [pages, H_kv, page, D_qk]
    const void* v_cache;  // [pages, H_kv, page, D_v]
    void* o;              // [T, H_q, D_v]
    float* stats;         // [T, H_q] dense
    TokenStrides qs, os;
    float* part_o;   // [slot][BM][D_v]: unnormalised O of a part
    float* part_ml;  // [slot][BM][2]: its running maximum (log2) and sum
    int H_kv, G, D_qk, D_v;
    float scale;
    int causal;
    int target_log2;  // workgroups to divide for: 2^target_log2
    int divide;       // parts: whether tiles may be divided
    int min_chunk;    // parts: key blocks of a part, at least
};

// Key blocks of 64 of a part, at least.  fp16, 300 tokens over 2300, 16 heads on 4, D
// 64: 2 blocks 31.2 us, 4 29.3, 6 25.7, 8 25.8, 16 27.7; over 1150: 24.8, 21.1, 21.9,
// 23.6, 29.6.
constexpr int kPagedMinChunk = 6;
constexpr int kPagedMaxParts = 64;  // (the merge walks a row's parts one batch after the other)

// One sequence's part of the plan.
struct SeqPlan {
    int q0, n, len;             // first new token, new tokens, cached tokens
    int tiles, blocks, parts;  // per key head; blocks of a tile on average
    bool bad;                  // more cached tokens than the table has columns for
};

// tiles = 0: nothing to do.  chunk = 0: parts are left at 1.
__host__ __device__ inline SeqPlan seq_plan(int q0, int q1, int kv_len, const PagedBatch& b, int G, bool causal, int BM,
                                            int BN, int chunk) {
    SeqPlan s{q0, 0, 0, 0, 0, 1, false};
    if (q0 < 0 || q1 <= q0 || q1 > b.T) return s;
    const int n = q1 - q0;
    const long long rows = (long long)n * G;
    const int cap = b.width << b.page_log2;
    s.n = n;
    s.bad = kv_len > cap;
    s.len = kv_len < 0 ? 0 : (kv_len > cap ? cap : kv_len);
    s.tiles = (int)((rows + BM - 1) / BM);
    const int mean = causal ? s.len - n / 2 : s.len;
    s.blocks = mean < BN ? 1 : (mean - 1) / BN + 1;
    if (chunk > 0) {
        const unsigned p = ((unsigned)s.blocks + (unsigned)chunk - 1) / (unsigned)chunk;
        s.parts = p < (unsigned)kPagedMaxParts ? (int)p : kPagedMaxParts;
    }
    return s;
}

// (Divisions of 64 bits take a microsecond here, which every workgroup would spend:
// the number of workgroups is a power of two.)
__host__ __device__ inline int plan_chunk(long long cost, int target_log2, int min_chunk) {
    const long long c = (cost + (1LL << target_log2) - 1) >> target_log2;
    return c < min_chunk ? min_chunk : (c < 0x3FFFFFFF ? (int)c : 0x3FFFFFFF);
}
// a / b for 0 <= a, 0 < b
__host__ __device__ inline int div_small(long long a, int b) {
    return a <= 0xFFFFFFFFLL ? (int)((unsigned)a / (unsigned)b) : (int)(a / b);
}

// Tiles of a launch, at most: every sequence with rows ends in one that is not full.
inline long long paged_max_tiles(const PagedParams& p, int BM) {
    const long long rows = (long long)p.batch.T * p.G;
    return (rows / BM + (rows < p.batch.N ? rows : p.batch.N)) * p.H_kv;
}

// Calls whose sequences have one tile of 32 rows, as far as is known, take the
// kernels of such tiles, by shares; others, by parts, those of 128-row tiles.
constexpr int kPagedSmallRows = 32;

// Shares: of `total` blocks, workgroup w of n takes [share_begin(w), share_begin(w + 1)); n
// is total itself or a power of two, 2^n_log2, below it.
__host__ __device__ inline long long share_begin(long long total, int w, int n, int n_log2) {
    return n == total ? w : (total * w) >> n_log2;
}
// The workgroup whose share holds block u: the largest w with total w / n < u + 1.
__host__ __device__ inline int share_owner(long long total, long long u, int n, int n_log2) {
    if (n == total) return (int)u;
    int w = (int)((double)u * n / (double)total);  // right or off by one
    if (share_begin(total, w, n, n_log2) > u) --w;
    else if (share_begin(total, w + 1, n, n_log2) <= u) ++w;
    return w;
}

// Workgroups the launches divide for, and the workspace of one launch's parts.
constexpr int kPagedTargetLog2 = 9;
constexpr int kPagedSmallBM = 32, kPagedBM = 128;
inline bool paged_small(long long T, int G, int max_q_len) {
    const long long most = max_q_len > 0 && max_q_len < T ? max_q_len : T;
    return most * G <= kPagedSmallRows;
}
inline size_t paged_part_bytes(int D_v, int BM) {
    return ((size_t)2 << kPagedTargetLog2) * BM * ((size_t)D_v + 2) * sizeof(float);
}

hipError_t launch_paged_f16_small(const PagedParams& p, hipStream_t stream);
hipError_t launch_paged_f16(const PagedParams& p, hipStream_t stream);
hipError_t launch_paged_f32_small(const PagedParams& p, hipStream_t stream);
hipError_t launch_paged_f32(const PagedParams& p, hipStream_t stream);

}  // namespace sdpa
