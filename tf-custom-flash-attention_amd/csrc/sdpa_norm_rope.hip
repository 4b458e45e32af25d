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
// Rows stay halves until the fused multiply-adds, and a weight's products with cos and
// sin are formed once for a wave's rows: fp16 is bound by VALU work otherwise (910
// instructions per four rows 118 us, 740 now).  4 x 4096 tokens, 32 + 32 heads of
// 128, fp16: forward 91 us, 5.9 TB/s (a bare copy past the caches 5.95; two rows per
// group of lanes 97 us), gradient 146, 5.5 TB/s (one row 146, four 151).
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
    int b, s, h;
    int rows;  // per group, those that some group has (wave-uniform)
    bool live;
    __device__ __forceinline__ Place(const SideMap& m, long long u, int group, long long tokens, int S, int ku) {
        const unsigned uu = (unsigned)u, tg = uu / (unsigned)m.splits;
        long long tok = (long long)tg * m.tpw + group / m.gpt;
        const int h0 = (int)(uu - tg * (unsigned)m.splits) * m.gpt * ku;
        h = h0 + group % m.gpt;
        rows = min(ku, (m.H - h0 + m.gpt - 1) / m.gpt);
        live = tok < tokens;
        if (!live) tok = tokens - 1;  // (a row that exists is read in its place)
        b = (int)((unsigned)tok / (unsigned)S);
        s = (int)((unsigned)tok - (unsigned)b * (unsigned)S);
    }
};

__device__ __forceinline__ long long position_of(const NormRopeParams& p, const Place& at) {
    if (!p.positions) return at.s;
    return p.positions[at.b * p.positions_stride + at.s];
}

template <typename T, int EPC, int LPR, bool IN, int KU, bool NT>
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
    const NormRopeSide sd = which ? p.side[1] : p.side[0];

    RowLane<EPC, IN> l;
    l.init(lane % LPR, p.D, p.r.R, p.interleaved != 0);
    const Place at(m, u, lane / LPR, tokens, p.S, KU);
    chunk_t<T, EPC> a[KU], b[KU];
    const T* x = static_cast<const T*>(sd.x) + at.b * sd.xs.b + at.s * sd.xs.s;
#pragma unroll
    for (int k = 0; k < KU; ++k)
        if (k < at.rows) load_row<T, EPC, IN, NT>(a[k], b[k], x + min(at.h + k * m.gpt, m.H - 1) * sd.xs.h, l);
    RowTurn<EPC> t;
    t.load(p.r, l, position_of(p, at));
    float wa[EPC], wb[EPC];
    load_weight<T, EPC, IN>(wa, wb, sd.w, p.w32 != 0, l);
    RowFactors<EPC, IN> f;
    f.init(l, t, wa, wb);
    T* y = static_cast<T*>(sd.y) + at.b * sd.ys.b + at.s * sd.ys.s;
#pragma unroll
    for (int k = 0; k < KU; ++k) {
        if (k >= at.rows) break;
        const int h = at.h + k * m.gpt;
        float r = p.r.norm ? row_rnorm<T, LPR, EPC, IN>(a[k], b[k], l, p.r) : 1.f;
        if (t.bad) r = __builtin_nanf("");
        f.template apply<T>(l, a[k], b[k], r);
        store_row<T, EPC, IN>(y + h * sd.ys.h, a[k], b[k], at.live && h < m.H, l);
    }
}

// dx, and this workgroup's sum of dw (blocks of q before those of k).
template <typename T, int EPC, int LPR, bool IN, int KU, bool NT>
__global__ __launch_bounds__(64 * kRopeWaves) void norm_rope_grad_kernel(const NormRopeParams p, const int blocks_q,
                                                                         const int blocks_k) {
    __shared__ float sums[kRopeWaves][2 * EPC * LPR];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long tokens = (long long)p.B * p.S;
    const int which = (int)blockIdx.x < blocks_q ? 0 : 1;
    const int block = which ? (int)blockIdx.x - blocks_q : (int)blockIdx.x, blocks = which ? blocks_k : blocks_q;
    const NormRopeSide sd = which ? p.side[1] : p.side[0];
    const SideMap m = side_map<LPR, KU>(tokens, sd.H);

    RowLane<EPC, IN> l;
    l.init(lane % LPR, p.D, p.r.R, p.interleaved != 0);
    float wa[EPC], wb[EPC], da[EPC], db[EPC];
    load_weight<T, EPC, IN>(wa, wb, sd.w, p.w32 != 0, l);
#pragma unroll
    for (int i = 0; i < EPC; ++i) da[i] = db[i] = 0.f;
    for (long long u = (long long)block * kRopeWaves + wave; u < m.units; u += (long long)blocks * kRopeWaves) {
        const Place at(m, u, lane / LPR, tokens, p.S, KU);
        const T* x = static_cast<const T*>(sd.x) + at.b * sd.xs.b + at.s * sd.xs.s;
        const T* dy = static_cast<const T*>(sd.dy) + at.b * sd.dys.b + at.s * sd.dys.s;
        T* dx = static_cast<T*>(sd.y) + at.b * sd.ys.b + at.s * sd.ys.s;
        chunk_t<T, EPC> a[KU], b[KU], ya[KU], yb[KU];
#pragma unroll
        for (int k = 0; k < KU; ++k) {
            if (k >= at.rows) break;
            const int h = min(at.h + k * m.gpt, m.H - 1);
            load_row<T, EPC, IN, NT>(a[k], b[k], x + h * sd.xs.h, l);
            load_row<T, EPC, IN, NT>(ya[k], yb[k], dy + h * sd.dys.h, l);
        }
        RowTurn<EPC> t;
        t.load(p.r, l, position_of(p, at));
#pragma unroll
        for (int k = 0; k < KU; ++k) {
            if (k >= at.rows) break;
            const int h = at.h + k * m.gpt;
            const bool live = at.live && h < m.H;
            float ga[EPC], gb[EPC];
#pragma unroll
            for (int i = 0; i < EPC; ++i) {
                ga[i] = sdpa::at<T, EPC>(ya[k], i);
                gb[i] = sdpa::at<T, EPC>(yb[k], i);
            }
            t.back(l, ga, gb);
            float r = 1.f;
            if (p.r.norm) {
                r = row_rnorm<T, LPR, EPC, IN>(a[k], b[k], l, p.r);
                float xa[EPC], xb[EPC], sa = 0.f, sb = 0.f;
#pragma unroll
                for (int i = 0; i < EPC; ++i) {
                    xa[i] = sdpa::at<T, EPC>(a[k], i) * r;
                    xb[i] = sdpa::at<T, EPC>(b[k], i) * r;
                }
                if (live)
#pragma unroll
                    for (int i = 0; i < EPC; ++i) {
                        da[i] = __builtin_fmaf(ga[i], xa[i], da[i]);
                        db[i] = __builtin_fmaf(gb[i], xb[i], db[i]);
                    }
#pragma unroll
                for (int i = 0; i < EPC; ++i) {
                    ga[i] *= wa[i];
                    gb[i] *= wb[i];
                    sa = __builtin_fmaf(ga[i], xa[i], sa);
                    sb = __builtin_fmaf(gb[i], xb[i], sb);
                }
                const float mean = group_sum<LPR>((l.va ? sa : 0.f) + (l.vb ? sb : 0.f)) * p.r.inv_D;
#pragma unroll
                for (int i = 0; i < EPC; ++i) {
                    ga[i] = __builtin_fmaf(-xa[i], mean, ga[i]);
                    gb[i] = __builtin_fmaf(-xb[i], mean, gb[i]);
                }
            }
            if (t.bad) r = __builtin_nanf("");
#pragma unroll
            for (int i = 0; i < EPC; ++i) {
                ga[i] *= r;
                gb[i] *= r;
            }
            store_row<T, EPC, IN>(dx + h * sd.ys.h, chunk_of<T, EPC>(ga), chunk_of<T, EPC>(gb), live, l);
        }
        if (t.bad && at.live && at.h < m.H)
#pragma unroll
            for (int i = 0; i < EPC; ++i) da[i] = db[i] = __builtin_nanf("");
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

// dw[d] = sum over the workgroups of one side: 16 features a workgroup, whose 1024
// threads take every 64th partial sum each, then the 64 sums of a feature in order
// of halves.
template <typename T>
__global__ __launch_bounds__(1024) void norm_rope_dw_kernel(const NormRopeParams p, const int blocks_q,
                                                            const int blocks_k) {
    __shared__ double sums[64][17];
    const int which = (int)blockIdx.y, c = threadIdx.x & 15, g = threadIdx.x >> 4, d = (int)blockIdx.x * 16 + c;
    void* const dw = which ? p.side[1].dw : p.side[0].dw;
    if (!dw) return;
    const int n = which ? blocks_k : blocks_q;
    const float* src = p.part_dw + (size_t)(which ? blocks_q : 0) * p.D + d;
    double s = 0.;  // (the terms cancel: off by 0.9e-7 of 96000 rows, fp32 sums by 1.4e-7)
    if (d < p.D)
#pragma unroll 16
        for (int i = g; i < n; i += 64) s += src[(size_t)i * p.D];
    sums[g][c] = s;
    __syncthreads();
    for (int h = 32; h > 0; h /= 2) {
        if (g < h) sums[g][c] += sums[g + h][c];
        __syncthreads();
    }
    if (g != 0 || d >= p.D) return;
    if (p.w32) static_cast<float*>(dw)[d] = (float)sums[0][c];
    else static_cast<T*>(dw)[d] = (T)sums[0][c];
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

// Rows are read past the caches where q and k together outgrow what the 256 MB
// cache can hold of them beside the results.  Forward, fp16 and fp32 alike, called again
// and again: 268 MB of q and k plain 103 us, so 89; 134 MB 44 and 47; 67 MB 22 and 26.  Forward
// and gradient: 268 MB 274 and 262, 134 MB 143 and 127, 67 MB 63 and 71 (the gradient alone,
// which reads dy too, would gain from 134 MB on; one rule serves both).
template <typename T>
bool past_caches(const NormRopeParams& p) {
    return (long long)p.B * p.S * (p.side[0].H + p.side[1].H) * p.D * (long long)sizeof(T) > (128LL << 20);
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
            const dim3 grid = tile_grid((n + kRopeWaves - 1) / kRopeWaves, 64 * kRopeWaves);
            if constexpr (KU == 4) {
                if (past_caches<T>(p))
                    return launch_kernel<norm_rope_kernel<T, E, L, IN, KU, true>>(grid, 64 * kRopeWaves, 0, stream, p);
            }
            return launch_kernel<norm_rope_kernel<T, E, L, IN, KU, false>>(grid, 64 * kRopeWaves, 0, stream, p);
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
        const dim3 grid((unsigned)(bq + bk));
        if (bq + bk > 0)
            e = past_caches<T>(p) ? launch_kernel<norm_rope_grad_kernel<T, E, L, IN, KU, true>>(grid, 64 * kRopeWaves, 0,
                                                                                                 stream, p, bq, bk)
                                  : launch_kernel<norm_rope_grad_kernel<T, E, L, IN, KU, false>>(grid, 64 * kRopeWaves, 0,
                                                                                                  stream, p, bq, bk);
        if (e != hipSuccess || (!p.side[0].dw && !p.side[1].dw)) return e;
        return launch_kernel<norm_rope_dw_kernel<T>>(dim3((unsigned)((p.D + 15) / 16), 2), 1024, 0, stream, p, bq, bk);
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
