// sdpa_norm_rope.h -- arguments and launchers of the norm and rotation of
// queries and keys (sdpa_norm_rope.hip).
#pragma once

#include "sdpa_launch.h"
#include "sdpa_rope.h"

namespace sdpa {

// Queries (side 0) or keys (side 1): x in, y out; in the gradient x and dy in,
// dx (y, ys) and dw out.
struct NormRopeSide {
    const void* x;
    const void* dy;
    void* y;
    const void* w;  // [D] or null
    void* dw;       // [D] or null
    RowStrides xs, dys, ys;
    int H;
};

struct NormRopeParams {
    NormRopeSide side[2];
    RopeArgs r;
    const int32_t* positions;    // [S] or [B, S]; null: 0 .. S - 1
    long long positions_stride;  // between sequences (0: shared)
    float* part_dw;              // [workgroup][D]
    int B, S, D;
    int interleaved;  // pairs (2i, 2i + 1), else (i, i + R/2)
    int w32;          // weights are float, else T
    int vec;          // every row in whole aligned 16-byte chunks, pairs in them
};

// Workgroups that share a side's rows in the gradient, at most: the weight's
// gradient has one partial sum of each.  Forward and gradient of 4 x 4096 tokens, 32 +
// 32 heads of 128, fp16: 512 268 us, 1024 259, 2048 261; 2 x 2048, 16 + 16 heads, fp32: 62,
// 61, 67.
constexpr int kGradBlocks = 1024;
// Fewer waves than this of four rows per group of lanes: one row each.  32 + 8 heads of
// 128, fp16: 64 tokens (128 waves of four) 3.5 us with one row, 4.5 with four; 512 (1024)
// 4.7, 5.2; 1024 (2048) 6.7, 5.9; 2048 10.8, 9.3.
constexpr int kRopeFewWaves = 2048;

hipError_t launch_norm_rope(const NormRopeParams& p, DType dtype, hipStream_t stream);
hipError_t launch_norm_rope_grad(const NormRopeParams& p, DType dtype, hipStream_t stream);

}  // namespace sdpa
