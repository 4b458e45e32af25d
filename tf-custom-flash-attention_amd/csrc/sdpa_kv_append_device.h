// sdpa_kv_append_device.h -- one wave's rows of queries, keys or values of new tokens on
// their way to where they belong, shared by the appends (sdpa_kv_append.hip,
// sdpa_kv_fp4.hip).
#pragma once

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
// KU: rows of a group of lanes.
template <int LPR, int KU = 1>
__host__ __device__ inline AppendMap append_map(int tokens, int H) {
    constexpr int RG = 64 / LPR;
    AppendMap m{H, 1, 1, 0, 0};
    if (H <= 0 || tokens <= 0) return m;
    while (m.gpt < H && m.gpt < RG) m.gpt *= 2;
    m.tpw = RG / m.gpt;
    m.splits = (H + m.gpt * KU - 1) / (m.gpt * KU);
    m.units = ((long long)tokens + m.tpw - 1) / m.tpw * m.splits;
    return m;
}

// Whether queries alone go by four rows per group of lanes (sdpa_kv_append.h).
template <int LPR>
inline bool append_four_rows(int tokens, int H) {
    const AppendMap m = append_map<LPR, 4>(tokens, H);
    return m.units >= kAppendFewWaves && 8LL * H >= 7LL * 4 * m.gpt * m.splits;
}

// Unit u of the rows of q (kind 0), k (1) or v (2).
template <typename T, int EPC, int LPR, bool IN, bool AX, int KU = 1>
__device__ __forceinline__ void append_rows(const AppendParams& p, const AppendMap& m, long long u, int kind) {
    const int lane = threadIdx.x & 63;
    const PagedBatch& bt = p.batch;
    const unsigned uu = (unsigned)u, tg = uu / (unsigned)m.splits;
    const int group = lane / LPR, tok0 = (int)(tg * (unsigned)m.tpw), mine = group / m.gpt;
    const long long tok = (long long)tok0 + mine;
    const int h = (int)(uu - tg * (unsigned)m.splits) * m.gpt * KU + group % m.gpt;  // and further ones, gpt apart
    const bool in_batch = tok < bt.T;

    // the row, before it is known where it goes
    const int D = kind == 2 ? p.D_v : p.D_qk;
    RowLane<EPC, IN> l;
    l.init(lane % LPR, D, kind == 2 ? 0 : p.r.R, p.interleaved != 0);
    const T* x = static_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v);
    const TokenStrides xs = kind == 0 ? p.qs : kind == 1 ? p.ks : p.vs;
    chunk_t<T, EPC> a[KU], b[KU];
#pragma unroll
    for (int i = 0; i < KU; ++i)
        load_row<T, EPC, IN>(a[i], b[i], x + (in_batch ? tok : bt.T - 1) * xs.t + min(h + i * m.gpt, m.H - 1) * xs.h, l);
    RowTurn<EPC> t;
    if constexpr (AX)
        if (kind != 2) t.load_axes(p.r, p.axes, l, p.axes.positions + (in_batch ? tok : bt.T - 1));

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
    if (tok < qs || tok >= qe || qs < 0 || qe > bt.T) return;  // (as attention leaves them out)
    const long long pos = (long long)bt.kv_lens[s] - qe + tok;
    const long long pg = pos >> bt.page_log2;
    int page = -1;
    if (pos >= 0 && pg < bt.width) page = bt.page_table[s * bt.table_stride + pg];
    const bool placed = page >= 0 && page < bt.pages;

    if constexpr (!AX)
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
    // (several rows of a group of lanes are queries', and each is stored as it is done)
    if (KU > 1 || kind != 2) {
        RowFactors<EPC, IN> f;
        f.init(l, t, wa, wb);
#pragma unroll
        for (int i = 0; i < KU; ++i) {
            float r = p.r.norm ? row_rnorm<T, LPR, EPC, IN>(a[i], b[i], l, p.r) : 1.f;
            if (t.bad || !placed) r = __builtin_nanf("");
            f.template apply<T>(l, a[i], b[i], r);
            if constexpr (KU > 1) store_row<T, EPC, IN>(y + (h + i * m.gpt) * hs, a[i], b[i], h + i * m.gpt < m.H, l);
        }
    }
    if constexpr (KU == 1) store_row<T, EPC, IN>(y + h * hs, a[0], b[0], h < m.H, l);
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

}  // namespace
}  // namespace sdpa
