// sdpa_kv_append.hip -- the keys and values of new tokens into the pages of a
// cache, keys normed (where asked) and rotated on the way, and the queries of
// the same tokens rotated beside them, in one launch, for gfx950.
//
// Each row is read and written once, by lanes that hold it as in sdpa_rope.h.  Prompts
// wait for memory, generation for a chain of dependent loads (start, length, page, row).
//  A wave takes q, k or v heads of one
// token (of several where heads are few), one row per group of lanes; it finds its tokens' sequences by counting, a wave's width of
// q_starts at a time, those that begin at or before the token.
//
// 8643 tokens of 4 sequences, 32 + 8 + 8 heads of 128, fp16 (217 MB): 43 us, 5.1
// TB/s, where the rows lie in the last-level cache, 53 us, 4.1 TB/s, from HBM; up to four
// rows per group of lanes 45 and 53.  The forward of sdpa_norm_rope.hip, whose reads and
// writes are alike, reaches 5.9 with loads past the caches; here they have not been tried.
// By positions of the tokens' own, three axes in sections, 56 us from HBM (fp32 93, 434 MB), axes in turn 63.
// 64 single tokens: 4.6 us.
//
// A token of no sequence (behind the last), or of one that reaches past the T tokens,
// leaves everything as it was.  One
// whose place is outside the table's columns or the cache's pages is not
// appended, and its query row is NaN; a position outside the rotation tables
// makes the rotated rows NaN.
#include "sdpa_kv_append_device.h"

namespace sdpa {
namespace {

template <typename T, int EPC, int LPR, bool IN, bool AX, int KU>
__global__ __launch_bounds__(64 * kAppendWaves) void kv_append_kernel(const AppendParams p) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const PagedBatch& bt = p.batch;
    long long u = (long long)tile_id() * kAppendWaves + wave;
    AppendMap m = append_map<LPR, KU>(bt.T, p.H_q);
    int kind = 0;  // 0: q, 1: k, 2: v
    if (u >= m.units) {
        u -= m.units;
        m = append_map<LPR, KU>(bt.T, p.H_k);
        kind = 1;
        if (u >= m.units) {
            u -= m.units;
            m = append_map<LPR, KU>(bt.T, p.H_v);
            kind = 2;
            if (u >= m.units) return;
        }
    }
    append_rows<T, EPC, LPR, IN, AX, KU>(p, m, u, kind);
}

template <typename T, bool AX>
hipError_t launch_kv_append_t(const AppendParams& p, hipStream_t stream) {
    return with_append_row<T>(p, [&](auto epc, auto lpr, auto in) {
        constexpr int E = decltype(epc)::value, L = decltype(lpr)::value;
        constexpr bool IN = decltype(in)::value;
        const auto run = [&](auto ku) {
            constexpr int KU = decltype(ku)::value;
            const long long n = append_map<L, KU>(p.batch.T, p.H_q).units + append_map<L, KU>(p.batch.T, p.H_k).units +
                                append_map<L, KU>(p.batch.T, p.H_v).units;
            if (n == 0) return hipSuccess;
            return launch_kernel<kv_append_kernel<T, E, L, IN, AX, KU>>(tile_grid((n + kAppendWaves - 1) / kAppendWaves, 64 * kAppendWaves),
                                                                        64 * kAppendWaves, 0, stream, p);
        };
        // (queries alone, many of them: of the append in 4 bits)
        if (p.H_k == 0 && p.H_v == 0 && append_four_rows<L>(p.batch.T, p.H_q)) return run(std::integral_constant<int, 4>{});
        return run(std::integral_constant<int, 1>{});
    });
}

}  // namespace

hipError_t launch_kv_append(const AppendParams& p, DType dtype, hipStream_t stream) {
    return with_bool(p.axes.used != 0, [&](auto ax) {
        constexpr bool AX = decltype(ax)::value;
        return dtype == DType::F16 ? launch_kv_append_t<half_t, AX>(p, stream) : launch_kv_append_t<float, AX>(p, stream);
    });
}

}  // namespace sdpa
