// sdpa_norm_rope.hip -- RMS norm of every head of the queries and keys with
// the rotation by position in the same pass, and its gradient, for gfx950.
//
//   r = 1 / sqrt(mean_d x^2 + eps),  n = w x r,  y = R(position) n
//   dn = R^T dy,  dw = sum over rows of dn x r,
//   dx = r (w dn - x r mean_d(w dn x r))
//
// Bound by memory: x is read and y written once (gradient: x and dy read, dx
// written); r is formed again in the gradient, which reads x anyway, rather
// than stored.  Rows are held as in sdpa_rope.h.  A wave takes neighbouring
// heads of one token (of several where heads are few), KU rows per group of
// lanes, whose loads all go out before the first is used and which share one
// read of the tables; strides let q and k be parts of a projection's output
// and the results be laid out [B H, S, D], as attention reads them, without a
// pass of their own.
//
// The weight's gradient is summed in registers over the rows of a workgroup,
// whose number is bounded (kGradBlocks), then over workgroups in order by a
// second kernel: no atomics, a call repeats to the bit.
#include <type_traits>

#include "sdpa_launch.h"
#include "sdpa_norm_rope.h"
#include "sdpa_rope.h"

namespace sdpa {
namespace {

constexpr int kRopeWaves = 4;

// How the rows of one side (q or k) are dealt to waves.
struct SideMap {
    int H, gpt, tpw;    // heads; groups of lanes per token; tokens per wave
    int splits;         // waves per token group
    long long units;    // waves in all
};
template <int LPR, int KU>
__host__ __device__ inline SideMap side_map(long long tokens, int H) {
    constexpr int RG = 64 / LPR;
    SideMap m{H, 1, 1, 0, 0};
    if (H <= 0 || tokens <= 0) return m;
    while (m.gpt < H && m.gpt < RG) m.gpt *= 2;
    m.tpw = RG / m.gpt;
    m.splits = (H + m.gpt * KU - 1) / (m.gpt * KU);
    m.units = (tokens + m.tpw - 1) / m.tpw * m.splits;
    return m;
}

// Token and first head of this lane's group in unit u; further rows of the
// group are gpt heads apart.
struct Place {
    long long tok;
    int b, s, h;
    bool live;
    __device__ __forceinline__ Place(const SideMap& m, long long u, int group, long long tokens, int S, int ku) {
        const unsigned uu = (unsigned)u, tg = uu / (unsigned)m.splits;
        tok = (long long)tg * m.tpw + group / m.gpt;
        h = (int)(uu - tg * (unsigned)m.splits) * m.gpt * ku + group % m.gpt;
        live = tok < tokens;
        b = (int)((unsigned)tok / (unsigned)S);
        s = (int)((unsigned)tok - (unsigned)b * (unsigned)S);
    }
};

__device__ __forceinline__ long long row_at(const RowStrides& st, const Place& at, int h) {
    return at.b * st.b + at.s * st.s + h * st.h;
}

__device__ __forceinline__ long long position_of(const NormRopeParams& p, const Place& at) {
    if (!p.positions || !at.live) return at.s;
    return p.positions[at.b * p.positions_stride + at.s];
}

template <typename T, int EPC, int LPR, bool IN, int KU>
__global__ __launch_bounds__(64 * kRopeWaves) void norm_rope_kernel(const NormRopeParams p) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long tokens = (long long)p.B * p.S;
    const SideMap mq = side_map<LPR, KU>(tokens, p.side[0].H), mk = side_map<LPR, KU>(tokens, p.side[1].H);
    long long u = (long long)tile_id() * kRopeWaves + wave;
    const int which = u < mq.units ? 0 : 1;
    const SideMap m = which ? mk : mq;
    if (which) u -= mq.units;
    if (u >= m.units) return;
    const NormRopeSide& sd = p.side[which];

    RowLane<EPC, IN> l;
    l.init(lane % LPR, p.D, p.r.R, p.interleaved != 0);
    const Place at(m, u, lane / LPR, tokens, p.S, KU);
    float a[KU][EPC], b[KU][EPC];
    const T* x = static_cast<const T*>(sd.x);
#pragma unroll
    for (int k = 0; k < KU; ++k) {
        const int h = at.h + k * m.gpt;
        load_row<T, EPC, IN>(a[k], b[k], x + row_at(sd.xs, at, h), at.live && h < m.H, l);
    }
    RowTurn<EPC> t;
    t.load(p.r, l, position_of(p, at));
    float wa[EPC], wb[EPC];
    load_weight<T, EPC, IN>(wa, wb, sd.w, p.w32 != 0, l);
    T* y = static_cast<T*>(sd.y);
#pragma unroll
    for (int k = 0; k < KU; ++k) {
        const int h = at.h + k * m.gpt;
        float r = p.r.norm ? row_rnorm<LPR, EPC>(a[k], b[k], p.D, p.r.eps) : 1.f;
        if (t.bad) r = __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < EPC; ++i) {
            a[k][i] = a[k][i] * r * wa[i];
            b[k][i] = b[k][i] * r * wb[i];
        }
        t.template apply<IN, false>(l, a[k], b[k]);
        store_row<T, EPC, IN>(y + row_at(sd.ys, at, h), a[k], b[k], at.live && h < m.H, l);
    }
}

// dx, and this workgroup's sum of dw (blocks of q before those of k).
template <typename T, int EPC, int LPR, bool IN, int KU>
__global__ __launch_bounds__(64 * kRopeWaves) void norm_rope_grad_kernel(const NormRopeParams p, const int blocks_q,
                                                                         const int blocks_k) {
    __shared__ float sums[kRopeWaves][2 * EPC * LPR];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long tokens = (long long)p.B * p.S;
    const int which = (int)blockIdx.x < blocks_q ? 0 : 1;
    const int block = which ? (int)blockIdx.x - blocks_q : (int)blockIdx.x, blocks = which ? blocks_k : blocks_q;
    const NormRopeSide& sd = p.side[which];
    const SideMap m = side_map<LPR, KU>(tokens, sd.H);

    RowLane<EPC, IN> l;
    l.init(lane % LPR, p.D, p.r.R, p.interleaved != 0);
    float wa[EPC], wb[EPC], da[EPC], db[EPC];
    load_weight<T, EPC, IN>(wa, wb, sd.w, p.w32 != 0, l);
#pragma unroll
    for (int i = 0; i < EPC; ++i) da[i] = db[i] = 0.f;
    const T* x = static_cast<const T*>(sd.x);
    const T* dy = static_cast<const T*>(sd.dy);
    T* dx = static_cast<T*>(sd.y);
    for (long long u = (long long)block * kRopeWaves + wave; u < m.units; u += (long long)blocks * kRopeWaves) {
        const Place at(m, u, lane / LPR, tokens, p.S, KU);
        float a[KU][EPC], b[KU][EPC], ga[KU][EPC], gb[KU][EPC];
#pragma unroll
        for (int k = 0; k < KU; ++k) {
            const int h = at.h + k * m.gpt;
            const bool live = at.live && h < m.H;
            load_row<T, EPC, IN>(a[k], b[k], x + row_at(sd.xs, at, h), live, l);
            load_row<T, EPC, IN>(ga[k], gb[k], dy + row_at(sd.dys, at, h), live, l);
        }
        RowTurn<EPC> t;
        t.load(p.r, l, position_of(p, at));
#pragma unroll
        for (int k = 0; k < KU; ++k) {
            const int h = at.h + k * m.gpt;
            const bool live = at.live && h < m.H;
            t.template apply<IN, true>(l, ga[k], gb[k]);
            if (t.bad)
#pragma unroll
                for (int i = 0; i < EPC; ++i) ga[k][i] = gb[k][i] = __builtin_nanf("");
            if (p.r.norm) {
                const float r = row_rnorm<LPR, EPC>(a[k], b[k], p.D, p.r.eps);
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < EPC; ++i) {
                    a[k][i] *= r;
                    b[k][i] *= r;
                    if (live) {
                        da[i] += ga[k][i] * a[k][i];
                        db[i] += gb[k][i] * b[k][i];
                    }
                    ga[k][i] *= wa[i];
                    gb[k][i] *= wb[i];
                    dot += ga[k][i] * a[k][i] + gb[k][i] * b[k][i];
                }
                dot = group_sum<LPR>(dot) / (float)p.D;
#pragma unroll
                for (int i = 0; i < EPC; ++i) {
                    ga[k][i] = r * (ga[k][i] - a[k][i] * dot);
                    gb[k][i] = r * (gb[k][i] - b[k][i] * dot);
                }
            }
            store_row<T, EPC, IN>(dx + row_at(sd.ys, at, h), ga[k], gb[k], live, l);
        }
    }
    if (!p.part_dw || !sd.dw) return;
    // over the groups of the wave, then over the waves
#pragma unroll
    for (int i = 0; i < EPC; ++i)
#pragma unroll
        for (int s = LPR; s < 64; s *= 2) {
            da[i] += __shfl_xor(da[i], s);
            db[i] += __shfl_xor(db[i], s);
        }
    if (lane < LPR)
#pragma unroll
        for (int i = 0; i < EPC; ++i) {
            sums[wave][2 * EPC * lane + i] = da[i];
            sums[wave][2 * EPC * lane + EPC + i] = db[i];
        }
    __syncthreads();
    if (wave == 0 && lane < LPR) {
        float* out = p.part_dw + (size_t)blockIdx.x * p.D;
#pragma unroll
        for (int i = 0; i < EPC; ++i) {
            float sa = 0.f, sb = 0.f;
#pragma unroll
            for (int w = 0; w < kRopeWaves; ++w) {
                sa += sums[w][2 * EPC * lane + i];
                sb += sums[w][2 * EPC * lane + EPC + i];
            }
            if (l.va) out[l.fa + i] = sa;
            if (l.vb) out[l.fb + i] = sb;
        }
    }
}

// dw[d] = sum over the workgroups of one side: one wave per feature.
template <typename T>
__global__ __launch_bounds__(256) void norm_rope_dw_kernel(const NormRopeParams p, const int blocks_q,
                                                           const int blocks_k) {
    const int lane = threadIdx.x & 63, c = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int which = c < p.D ? 0 : 1, d = which ? c - p.D : c;
    if (d >= p.D || !p.side[which].dw) return;
    const int n = which ? blocks_k : blocks_q;
    const float* src = p.part_dw + (size_t)(which ? blocks_q : 0) * p.D + d;
    float s = 0.f;
    for (int i = lane; i < n; i += 64) s += src[(size_t)i * p.D];
    s = group_sum<64>(s);
    if (lane != 0) return;
    if (p.w32) static_cast<float*>(p.side[which].dw)[d] = s;
    else static_cast<T*>(p.side[which].dw)[d] = (T)s;
}

// f<EPC, LPR, IN>() for the chunks these rows allow.
template <typename T, typename F>
hipError_t with_row(const NormRopeParams& p, F&& f) {
    constexpr int V = 16 / (int)sizeof(T);
    const auto lpr = [&](auto epc, auto in) {
        constexpr int E = decltype(epc)::value;
        const int n = lanes_per_row(p.D, E);
        if constexpr (E == 1) {
            if (n <= 16) return f(epc, std::integral_constant<int, 16>{}, in);
            return f(epc, std::integral_constant<int, 64>{}, in);
        } else {
            // 8 features a chunk: up to 8 lanes; 4 a chunk: up to 16
            if (n <= 2) return f(epc, std::integral_constant<int, 2>{}, in);
            if (n <= 4) return f(epc, std::integral_constant<int, 4>{}, in);
            if (E == 8 || n <= 8) return f(epc, std::integral_constant<int, 8>{}, in);
            return f(epc, std::integral_constant<int, E == 8 ? 8 : 16>{}, in);
        }
    };
    if (!p.vec) return lpr(std::integral_constant<int, 1>{}, std::false_type{});
    if (p.interleaved) return lpr(std::integral_constant<int, V>{}, std::true_type{});
    return lpr(std::integral_constant<int, V>{}, std::false_type{});
}

// Workgroups of one side in the gradient: as many as its rows need, at most
// kGradBlocks.
int grad_blocks(long long units) {
    const long long n = (units + kRopeWaves - 1) / kRopeWaves;
    return (int)(n < kGradBlocks ? n : kGradBlocks);
}

template <typename T>
hipError_t launch_norm_rope_t(const NormRopeParams& p, hipStream_t stream) {
    return with_row<T>(p, [&](auto epc, auto lpr, auto in) {
        constexpr int E = decltype(epc)::value, L = decltype(lpr)::value;
        constexpr bool IN = decltype(in)::value;
        const long long tokens = (long long)p.B * p.S;
        const auto run = [&](auto ku) {
            constexpr int KU = decltype(ku)::value;
            const long long n = side_map<L, KU>(tokens, p.side[0].H).units + side_map<L, KU>(tokens, p.side[1].H).units;
            if (n == 0) return hipSuccess;
            return launch_kernel<norm_rope_kernel<T, E, L, IN, KU>>(
                tile_grid((n + kRopeWaves - 1) / kRopeWaves, 64 * kRopeWaves), 64 * kRopeWaves, 0, stream, p);
        };
        const long long n4 = side_map<L, 4>(tokens, p.side[0].H).units + side_map<L, 4>(tokens, p.side[1].H).units;
        if (n4 >= kRopeFewWaves) return run(std::integral_constant<int, 4>{});
        return run(std::integral_constant<int, 1>{});
    });
}

template <typename T>
hipError_t launch_norm_rope_grad_t(const NormRopeParams& p, hipStream_t stream) {
    return with_row<T>(p, [&](auto epc, auto lpr, auto in) {
        constexpr int E = decltype(epc)::value, L = decltype(lpr)::value, KU = 2;
        constexpr bool IN = decltype(in)::value;
        const long long tokens = (long long)p.B * p.S;
        const int bq = grad_blocks(side_map<L, KU>(tokens, p.side[0].H).units);
        const int bk = grad_blocks(side_map<L, KU>(tokens, p.side[1].H).units);
        hipError_t e = hipSuccess;
        if (bq + bk > 0)
            e = launch_kernel<norm_rope_grad_kernel<T, E, L, IN, KU>>(dim3((unsigned)(bq + bk)), 64 * kRopeWaves, 0,
                                                                      stream, p, bq, bk);
        if (e != hipSuccess || (!p.side[0].dw && !p.side[1].dw)) return e;
        return launch_kernel<norm_rope_dw_kernel<T>>(dim3((unsigned)((2 * p.D + 3) / 4)), 256, 0, stream, p, bq, bk);
    });
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeParams& p, DType dtype, hipStream_t stream) {
    return dtype == DType::F16 ? launch_norm_rope_t<half_t>(p, stream) : launch_norm_rope_t<float>(p, stream);
}

hipError_t launch_norm_rope_grad(const NormRopeParams& p, DType dtype, hipStream_t stream) {
    return dtype == DType::F16 ? launch_norm_rope_grad_t<half_t>(p, stream)
                               : launch_norm_rope_grad_t<float>(p, stream);
}

}  // namespace sdpa
