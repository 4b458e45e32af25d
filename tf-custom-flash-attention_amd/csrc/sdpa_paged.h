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
//           blocks (plan_chunk), at least the whole cost over target = 2^target_log2
//           workgroups.  So at most target workgroups more than there are tiles have
//           work, whatever the lengths, and at most 2 target parts are of divided tiles.
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
    float* part_ml;  // [slot][BM][2]: the reference of its weights (log2) and their sum
    int H_kv, G, D_qk, D_v;
    float scale;
    int causal;
    int most_rows;    // rows of a sequence and key head, at most as far as is known
    int target_log2;  // workgroups to divide for: 2^target_log2
    int divide;       // parts: whether tiles may be divided
    int min_chunk;    // parts: key blocks of a part, at least
    int one_per_cu;   // parts: chunks up to this come for half the workgroups (0: not)
};

// Key blocks of 64 of a part, at least.  16 tokens of 8 heads on one, D 128, over 2300:
// 4 blocks 14.9 us, 6 16.0, 8 17.9; fp32 23.4, 27.0, 31.1.
constexpr int kPagedMinChunk = 4;
// Where two workgroups share a CU and chunks would be shorter than this, they are up to
// twice as long, which leaves one a CU: 300 tokens over 2300, 16 heads on 4, chunks of 4
// blocks 28.1 us, 6 23.3; 64 over 30000, 8 heads on 4, of 6 28.7, 8 25.8.
constexpr int kPagedOnePerCu = 8;
// Parts of a tile.  16 tokens of 8 heads on one over 120000, one tile: 64 parts 50 us, 128
// 36, 256 27; fp32 202, 114 and 42.
constexpr int kPagedMaxParts = 256;

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
__host__ __device__ inline int plan_chunk(long long cost, int target_log2, int min_chunk, int one_per_cu = 0) {
    long long c = (cost + (1LL << target_log2) - 1) >> target_log2;
    if (c < one_per_cu) c = 2 * c < one_per_cu ? 2 * c : one_per_cu;
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

// Calls whose sequences have up to so many rows, as far as is known, take the kernels of
// 32-row tiles, by shares; others, by parts, those of 128-row tiles.  us by 32-row and by
// 128-row tiles, D 128:
//   fp16, 16 rows: 64 sequences of 600 to 16384, 4 key heads 131, 161; 64 of 5120 124, 132;
//         4 of 2000 19, 22; 32 of 4096 58, 53; 256 of 500 67, 61; one of 30000 36, 24
//   fp16, 32 rows: 146, 168; 129, 137; 26, 22; 63, 58; 73, 62; 51, 25
//   fp32, 32 rows: 32 of 4096 126, 215; 4 of 2000 31, 52; one of 30000 62, 64 (D 64: 73,
//         91; 28, 30; 49, 37); 64 rows, 4 of 2000 37, 53; 32 of 4096 214, 220; one 73, 65
// At 16 fp16 rows each wins three of the six (435 and 453 us together), at 32 the 128-row
// tiles four of six; one long sequence loses most by the small ones (36 for 24).  The rule goes
// by rows alone: lengths are on the device.
constexpr int kPagedSmallRowsF16 = 16, kPagedSmallRowsF32 = 32;

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
// The slot of part k of a tile that begins in the share of workgroup w and is cut.
__host__ __device__ inline int share_slot(int w, int k) { return k == 0 ? 2 * w + 1 : 2 * (w + k); }
// What workgroup w does with the tile of blocks [t0, t1) that holds block `at` of its share,
// which ends before block `end`: blocks [u0, u1) of the tile; the walk goes on at `stop`.
// Without `divide` the tiles that begin in the share, whole.
struct ShareStep {
    long long stop;
    int u0, u1, slot;
    bool divided, skip;
};
__host__ __device__ inline ShareStep share_step(long long at, long long end, long long t0, long long t1, int w,
                                                bool divide) {
    const long long stop = divide && end < t1 ? end : t1;
    const int u0 = (int)(at - t0);
    return {stop, u0, (int)(stop - t0), u0 == 0 ? share_slot(w, 0) : share_slot(w - 1, 1), u0 != 0 || stop != t1,
            !divide && t0 != at};
}
// The parts that workgroup w merges: those of the tile of `blocks` blocks from t0 on, which holds
// block `at`, the first of share w + 1, if the tile begins in share w and reaches across; else 0.
__host__ __device__ inline int share_merge(long long total, long long at, long long t0, int blocks, int w, int n,
                                           int n_log2) {
    if (t0 == at || share_owner(total, t0, n, n_log2) != w) return 0;
    return share_owner(total, t0 + blocks - 1, n, n_log2) - w + 1;
}

// Rows of a sequence and key head, at most as far as is known; workgroups the launches
// divide for, and the workspace of one launch's parts: by the kernel and D_v alone (D_v 128:
// 17 MB and 68 MB), as much for a short call as for a long one.  Launches that divide for
// half as many workgroups (fp32 chunks, fp32 generation of more than 128 features in all) use
// half of it.
constexpr int kPagedTargetLog2 = 9;
constexpr int kPagedSmallBM = 32, kPagedBM = 128;
inline long long paged_most_rows(long long T, int G, int max_q_len) {
    return (max_q_len > 0 && max_q_len < T ? max_q_len : T) * G;
}
inline bool paged_small(bool f16, long long most_rows) {
    return most_rows <= (f16 ? kPagedSmallRowsF16 : kPagedSmallRowsF32);
}
inline size_t paged_part_bytes(int D_v, int BM) {
    return ((size_t)2 << kPagedTargetLog2) * BM * ((size_t)D_v + 2) * sizeof(float);
}

hipError_t launch_paged_f16_small(const PagedParams& p, hipStream_t stream);
hipError_t launch_paged_f16(const PagedParams& p, hipStream_t stream);
hipError_t launch_paged_f32_small(const PagedParams& p, hipStream_t stream);
hipError_t launch_paged_f32(const PagedParams& p, hipStream_t stream);

}  // namespace sdpa
