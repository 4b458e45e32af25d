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
// gradient has one partial sum of each.
constexpr int kGradBlocks = 1024;
// Fewer waves than this of four rows per group of lanes: one row each.
constexpr int kRopeFewWaves = 2048;

hipError_t launch_norm_rope(const NormRopeParams& p, DType dtype, hipStream_t stream);
hipError_t launch_norm_rope_grad(const NormRopeParams& p, DType dtype, hipStream_t stream);

}  // namespace sdpa
