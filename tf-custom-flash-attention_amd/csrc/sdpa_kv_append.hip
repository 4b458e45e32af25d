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
// 64 single tokens: 4.6 us.
//
// A token of no sequence (behind the last) leaves everything as it was.  One
// whose place is outside the table's columns or the cache's pages is not
// appended, and its query row is NaN; a position outside the rotation tables
// makes the rotated rows NaN.
#include <type_traits>

#include "sdpa_kv_append.h"

namespace sdpa {
namespace {

constexpr int kAppendWaves = 4;

// How the rows of q, k or v are dealt to waves.
struct AppendMap {
    int H, gpt, tpw, splits;
    long long units;
};
template <int LPR>
__host__ __device__ inline AppendMap append_map(int tokens, int H) {
    constexpr int RG = 64 / LPR;
    AppendMap m{H, 1, 1, 0, 0};
    if (H <= 0 || tokens <= 0) return m;
    while (m.gpt < H && m.gpt < RG) m.gpt *= 2;
    m.tpw = RG / m.gpt;
    m.splits = (H + m.gpt - 1) / m.gpt;
    m.units = ((long long)tokens + m.tpw - 1) / m.tpw * m.splits;
    return m;
}

template <typename T, int EPC, int LPR, bool IN>
__global__ __launch_bounds__(64 * kAppendWaves) void kv_append_kernel(const AppendParams p) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const PagedBatch& bt = p.batch;
    long long u = (long long)tile_id() * kAppendWaves + wave;
    AppendMap m = append_map<LPR>(bt.T, p.H_q);
    int kind = 0;  // 0: q, 1: k, 2: v
    if (u >= m.units) {
        u -= m.units;
        m = append_map<LPR>(bt.T, p.H_k);
        kind = 1;
        if (u >= m.units) {
            u -= m.units;
            m = append_map<LPR>(bt.T, p.H_v);
            kind = 2;
            if (u >= m.units) return;
        }
    }
    const unsigned uu = (unsigned)u, tg = uu / (unsigned)m.splits;
    const int group = lane / LPR, tok0 = (int)(tg * (unsigned)m.tpw), mine = group / m.gpt;
    const long long tok = (long long)tok0 + mine;
    const int h = (int)(uu - tg * (unsigned)m.splits) * m.gpt + group % m.gpt;
    const bool in_batch = tok < bt.T;

    // the row, before it is known where it goes
    const int D = kind == 2 ? p.D_v : p.D_qk;
    RowLane<EPC, IN> l;
    l.init(lane % LPR, D, kind == 2 ? 0 : p.r.R, p.interleaved != 0);
    const T* x = static_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v);
    const TokenStrides xs = kind == 0 ? p.qs : kind == 1 ? p.ks : p.vs;
    chunk_t<T, EPC> a, b;
    load_row<T, EPC, IN>(a, b, x + (in_batch ? tok : bt.T - 1) * xs.t + min(h, m.H - 1) * xs.h, l);

    // sequence of the token: the last that begins at or before it
    int count = 0;
    for (int n0 = 0; n0 < bt.N; n0 += 64) {
        const int n = n0 + lane;
        const int start = n < bt.N ? bt.q_starts[n] : 0x7FFFFFFF;
        for (int i = 0; i < m.tpw; ++i) {
            const int c = __popcll(__ballot((long long)start <= (long long)tok0 + i));
            if (i == mine) count += c;
        }
    }
    if (!in_batch || count == 0) return;
    const int s = count - 1, qs = bt.q_starts[s], qe = bt.q_starts[s + 1];
    if (tok < qs || tok >= qe) return;
    const long long pos = (long long)bt.kv_lens[s] - qe + tok;
    const long long pg = pos >> bt.page_log2;
    int page = -1;
    if (pos >= 0 && pg < bt.width) page = bt.page_table[s * bt.table_stride + pg];
    const bool placed = page >= 0 && page < bt.pages;

    RowTurn<EPC> t;
    if (kind != 2) t.load(p.r, l, pos);
    float wa[EPC], wb[EPC];
    load_weight<T, EPC, IN>(wa, wb, kind == 2 ? nullptr : kind == 0 ? p.q_weight : p.k_weight, p.w32 != 0, l);
    const long long slot = pos & ((1LL << bt.page_log2) - 1);
    if (kind != 0 && !placed) return;
    T* y;
    long long hs;
    if (kind == 0) {
        y = static_cast<T*>(p.q_out) + tok * p.qos.t;
        hs = p.qos.h;
    } else {
        hs = (long long)D << bt.page_log2;
        y = static_cast<T*>(kind == 1 ? p.k_cache : p.v_cache) + (long long)page * p.H_kv * hs + slot * D;
    }
    if (kind != 2) {
        RowFactors<EPC, IN> f;
        f.init(l, t, wa, wb);
        float r = p.r.norm ? row_rnorm<T, LPR, EPC, IN>(a, b, l, p.r) : 1.f;
        if (t.bad || !placed) r = __builtin_nanf("");
        f.template apply<T>(l, a, b, r);
    }
    store_row<T, EPC, IN>(y + h * hs, a, b, h < m.H, l);
}

// f<EPC, LPR, IN>() for the chunks these rows allow.
template <typename T, typename F>
hipError_t with_append_row(const AppendParams& p, F&& f) {
    constexpr int V = 16 / (int)sizeof(T);
    const int D = p.D_qk > p.D_v ? p.D_qk : p.D_v;
    const auto lpr = [&](auto epc, auto in) {
        constexpr int E = decltype(epc)::value;
        const int n = lanes_per_row(D, E);
        if constexpr (E == 1) {
            return f(epc, std::integral_constant<int, 64>{}, in);
        } else {
            if (n <= 4) return f(epc, std::integral_constant<int, 4>{}, in);
            if (E == 8 || n <= 8) return f(epc, std::integral_constant<int, 8>{}, in);
            return f(epc, std::integral_constant<int, E == 8 ? 8 : 16>{}, in);
        }
    };
    if (!p.vec) return lpr(std::integral_constant<int, 1>{}, std::false_type{});
    if (p.interleaved) return lpr(std::integral_constant<int, V>{}, std::true_type{});
    return lpr(std::integral_constant<int, V>{}, std::false_type{});
}

template <typename T>
hipError_t launch_kv_append_t(const AppendParams& p, hipStream_t stream) {
    return with_append_row<T>(p, [&](auto epc, auto lpr, auto in) {
        constexpr int E = decltype(epc)::value, L = decltype(lpr)::value;
        constexpr bool IN = decltype(in)::value;
        const long long n = append_map<L>(p.batch.T, p.H_q).units + append_map<L>(p.batch.T, p.H_k).units +
                            append_map<L>(p.batch.T, p.H_v).units;
        if (n == 0) return hipSuccess;
        return launch_kernel<kv_append_kernel<T, E, L, IN>>(tile_grid((n + kAppendWaves - 1) / kAppendWaves, 64 * kAppendWaves),
                                                            64 * kAppendWaves, 0, stream, p);
    });
}

}  // namespace

hipError_t launch_kv_append(const AppendParams& p, DType dtype, hipStream_t stream) {
    return dtype == DType::F16 ? launch_kv_append_t<half_t>(p, stream) : launch_kv_append_t<float>(p, stream);
}

}  // namespace sdpa
