// sdpa_kv_fp4.hip -- keys and values of new tokens into the pages of a cache in 4 bits
// (sdpa_fp4.h), keys normed (where asked) and rotated on the way, the queries of the same
// tokens beside them in one launch; and tokens out of such pages again.  For gfx950.
//
// Queries go as in sdpa_kv_append.hip, where calls are large by its kernel (which
// needs half the registers, and waits for memory).  8 tokens of a head share the words of the
// values' codes, so a wave takes those new tokens of one head that lie in the same 8 places
// of a sequence; of a window of W packed tokens it takes each run of such that begins in it.
// The words of a run that does not fill its 8 places are read, and the other tokens' codes
// kept.
// 8643 tokens of 4 sequences, 32 + 8 + 8 heads of 128, fp16, three positions: keys and values 27 us
// (25 alone; 45 MB, 9 us at a copy's rate), queries 32 (142 MB, 4.4 TB/s) by a kernel of their own
// (one kernel for both 76 us where two took 68); fp32 34 (27 alone) and 58 (283 MB, 4.9 TB/s).  fp32 in place of
// the keys' fp64 takes 3.4 us off; by places and without norm they are 30 us, as 22 registers
// spill there (16 with fp32).  The rest is work that every wave does again for its head: the search for
// the run, the turn, the weights.  64 single tokens, without norm: 5.4 us, a chain of loads.  The read of 8643 tokens: 14
// us (45 MB; fp32 22, 80 MB), with the search for each head and for keys and values apart.
// Keys: norm and rotation in fp64, then rounded to fp32 and to 4 bits.  A code changes
// by a whole step where a value crosses a border, so with fp32 sums the codes of a token would go
// by the order of the additions, one in some 10^6 values; in fp64 they do not, in
// practice.  Keys pass from the lanes of the rotation to those of the codes, and codes of
// values from tokens to words, through LDS, a wave by itself.
#include "sdpa_fp4.h"
#include "sdpa_kv_append_device.h"
#include "sdpa_wave.h"

namespace sdpa {
namespace {

constexpr int kFp4Run = 8;  // tokens that share a word

// Tokens of a run: t .. t + n - 1 of the packed ones, places pos .. of sequence s, in one
// page (below 0: none; n is 1 then).
struct Fp4Run {
    int t, n, page;
    long long pos;
};

// work(run) for every run that begins in the window of W packed tokens from tok0 on.  The wave's
// lanes look for them together: lane i < W has token tok0 + i.  WHOLE: sequences that do not lie
// in the T tokens are left out, else those of their tokens that do are taken.
template <int W, bool WHOLE, typename F>
__device__ __forceinline__ void each_run(const PagedBatch& bt, int tok0, F&& work) {
    const int lane = threadIdx.x & 63;
    int count = 0;  // sequences that begin at or before the lane's token
    for (int n0 = 0; n0 < bt.N; n0 += 64) {
        const int n = n0 + lane, start = n < bt.N ? bt.q_starts[n] : 0x7FFFFFFF;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int c = __popcll(__ballot((long long)start <= (long long)tok0 + i));
            if (lane == i) count += c;
        }
    }
    const long long tok = (long long)tok0 + lane;
    int n = 0, page = -1;
    long long pos = 0;
    if (lane < W && tok < bt.T && count > 0) {
        const int s = count - 1, qs = bt.q_starts[s], qe = bt.q_starts[s + 1];
        if (tok >= qs && tok < qe && !(WHOLE && (qs < 0 || qe > bt.T))) {
            pos = (long long)bt.kv_lens[s] - qe + tok;
            const long long pg = pos >> bt.page_log2;
            if (pos >= 0 && pg < bt.width) page = bt.page_table[s * bt.table_stride + pg];
            if (page >= bt.pages) page = -1;
            const int at = (int)(pos & (kFp4Run - 1));
            const long long left = (qe < bt.T ? qe : bt.T) - tok;
            if (page < 0) n = 1;
            else if (tok == qs || at == 0) n = (int)(left < kFp4Run - at ? left : kFp4Run - at);
        }
    }
    for (uint64_t todo = __builtin_amdgcn_ballot_w64(n > 0); todo != 0; todo &= todo - 1) {
        const int l = __builtin_ctzll(todo);
        const auto get = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
        work(Fp4Run{tok0 + l, get(n), get(page), ((long long)get((int)(pos >> 32)) << 32) | (uint32_t)get((int)pos)});
    }
}

// LDS of a wave: rows of keys as fp32, or codes of values.
constexpr int kFp4RowStride = 128 + 8;
struct alignas(32) Fp4Lds {
    union {
        float keys[kFp4Run][kFp4RowStride];
        uint2v codes[kFp4Run][8 + 1];  // [place][16 features]
    };
};

__device__ __forceinline__ void store_byte(unsigned char* p, uint32_t x) { *p = (unsigned char)x; }

template <typename T, int EPC, int LPR, bool IN, bool AX>
__device__ __forceinline__ void append_keys(const AppendParams& p, const Fp4Run& run, int h, Fp4Lds& lds) {
    const int lane = threadIdx.x & 63, D = p.D_qk;
    constexpr int RG = 64 / LPR;
    RowLane<EPC, IN> l;
    l.init(lane % LPR, D, p.r.R, p.interleaved != 0);
    float wa[EPC], wb[EPC];
    load_weight<T, EPC, IN>(wa, wb, p.k_weight, p.w32 != 0, l);
#pragma unroll
    for (int r0 = 0; r0 < kFp4Run; r0 += RG) {
        const int r = r0 + lane / LPR, i = min(r, run.n - 1);
        if (r0 >= run.n) break;
        chunk_t<T, EPC> a, b;
        load_row<T, EPC, IN>(a, b, static_cast<const T*>(p.k) + (long long)(run.t + i) * p.ks.t + h * p.ks.h, l);
        RowTurn<EPC> t;
        if constexpr (AX) t.load_axes(p.r, p.axes, l, p.axes.positions + run.t + i);
        else t.load(p.r, l, run.pos + i);
        double rn = 1.;
        if (p.r.norm) {
            double sum = 0.;
#pragma unroll
            for (int e = 0; e < EPC; ++e) {
                const double x = at<T, EPC>(a, e), y = at<T, EPC>(b, e);
                if (l.va) sum = __builtin_fma(x, x, sum);
                if (l.vb) sum = __builtin_fma(y, y, sum);
            }
#pragma unroll
            for (int d = 1; d < LPR; d *= 2) sum += __shfl_xor(sum, d);
            rn = 1. / __builtin_sqrt(sum / D + (double)p.r.eps);
        }
        if (t.bad) rn = __builtin_nan("");
        float ya[EPC], yb[EPC];
        const auto turn = [&](float x, float y, float v, float w, int e, bool turned, float& u, float& z) {
            const double xv = (double)x * v, yw = (double)y * w;
            u = (float)((turned ? __builtin_fma(xv, (double)t.c[e], -yw * t.s[e]) : xv) * rn);
            z = (float)((turned ? __builtin_fma(yw, (double)t.c[e], xv * t.s[e]) : yw) * rn);
        };
        if constexpr (!IN) {
#pragma unroll
            for (int e = 0; e < EPC; ++e) turn(at<T, EPC>(a, e), at<T, EPC>(b, e), wa[e], wb[e], e, l.ra, ya[e], yb[e]);
        } else {
#pragma unroll
            for (int e = 0; e < EPC / 2; ++e) {
                turn(at<T, EPC>(a, 2 * e), at<T, EPC>(a, 2 * e + 1), wa[2 * e], wa[2 * e + 1], e, l.ra, ya[2 * e], ya[2 * e + 1]);
                turn(at<T, EPC>(b, 2 * e), at<T, EPC>(b, 2 * e + 1), wb[2 * e], wb[2 * e + 1], EPC / 2 + e, l.rb, yb[2 * e],
                     yb[2 * e + 1]);
            }
        }
        if (r < run.n) store_row<float, EPC, IN>(lds.keys[r], chunk_of<float, EPC>(ya), chunk_of<float, EPC>(yb), true, l);
    }
    lds_reads_done();
    const int r = lane / 8, f = lane % 8 * 16;
    if (r >= run.n || f >= D) return;
    float x[2][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const floatx4 v = *reinterpret_cast<const floatx4*>(&lds.keys[r][f + 4 * i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i / 2][4 * (i % 2) + e] = v[e];
    }
    uint32_t scale;
    const uint2v codes = fp4_half_group(x, scale);
    const int log2 = p.batch.page_log2;
    const long long slot = (run.pos & ((1 << log2) - 1)) + r;
    unsigned char* head = static_cast<unsigned char*>(p.k_cache) + ((long long)run.page * p.H_kv + h) * fp4_head_bytes(D, log2);
    *reinterpret_cast<uint2v*>(head + slot * (D / 2) + f / 2) = codes;
    if (f % 32 == 0) store_byte(head + fp4_scales_at(D, log2) + slot * (D / 32) + f / 32, scale);
}

// 16 features of a row as fp32.  VEC: in 16-byte chunks.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(float (&x)[2][8], const T* row) {
    if constexpr (VEC) {
        constexpr int E = 16 / (int)sizeof(T);
        typedef T chunk __attribute__((ext_vector_type(E)));
#pragma unroll
        for (int i = 0; i < 16; i += E) {
            const chunk c = *reinterpret_cast<const chunk*>(row + i);
#pragma unroll
            for (int e = 0; e < E; ++e) x[(i + e) / 8][(i + e) % 8] = (float)c[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i / 8][i % 8] = (float)row[i];
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void append_values(const AppendParams& p, const Fp4Run& run, int h, Fp4Lds& lds) {
    const int lane = threadIdx.x & 63, D = p.D_v, log2 = p.batch.page_log2;
    const int r = lane / 8, f = lane % 8 * 16, at = (int)(run.pos & (kFp4Run - 1));
    const long long block = (run.pos & ((1 << log2) - 1)) / kFp4Run;
    unsigned char* head = static_cast<unsigned char*>(p.v_cache) + ((long long)run.page * p.H_kv + h) * fp4_head_bytes(D, log2);
    uint2v* words = reinterpret_cast<uint2v*>(head + block * D * 4) + lane;  // of features 2 lane and 2 lane + 1
    uint2v old = {0, 0};
    if (run.n < kFp4Run && 2 * lane < D) old = *words;
    if (r < run.n && f < D) {
        float x[2][8];
        load16<T, VEC>(x, static_cast<const T*>(p.v) + (long long)(run.t + r) * p.vs.t + h * p.vs.h + f);
        uint32_t scale;
        lds.codes[at + r][f / 16] = fp4_half_group(x, scale);
        if (f % 32 == 0) store_byte(head + fp4_scales_at(D, log2) + (block * (D / 32) + f / 32) * 8 + at + r, scale);
    }
    lds_reads_done();
    if (2 * lane >= D) return;
    uint32_t w0 = 0, w1 = 0;
#pragma unroll
    for (int i = 0; i < kFp4Run; ++i) {
        const uint32_t b = reinterpret_cast<const unsigned char*>(lds.codes[i])[lane];
        w0 |= (b & 15u) << (4 * i);
        w1 |= (b >> 4) << (4 * i);
    }
    const uint32_t mask = (run.n < kFp4Run ? (1u << (4 * run.n)) - 1u : ~0u) << (4 * at);  // the run's tokens
    *words = (uint2v){(w0 & mask) | (old[0] & ~mask), (w1 & mask) | (old[1] & ~mask)};
}

// Windows of the keys or of the values.
template <int W>
__host__ __device__ inline long long fp4_units(int T, int H_kv) { return ((long long)T + W - 1) / W * H_kv; }

// QUERIES: those of the tokens too, behind the keys and values, which are the longer chains.
template <typename T, int EPC, int LPR, bool IN, bool AX, int W, bool QUERIES>
__global__ __launch_bounds__(64 * kAppendWaves, W > 1 ? 4 : 1) void kv_append_fp4_kernel(const AppendParams p) {
    __shared__ Fp4Lds lds[kAppendWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long n = fp4_units<W>(p.batch.T, p.H_kv);
    long long u = (long long)tile_id() * kAppendWaves + wave;
    constexpr int KINDS = W > 1 ? 1 : 2;  // keys and values by waves of their own, or by one after the other
    if (u >= KINDS * n) {
        if constexpr (QUERIES) {
            const AppendMap m = append_map<LPR>(p.batch.T, p.H_q);
            if (u - KINDS * n < m.units) append_rows<T, EPC, LPR, IN, AX>(p, m, u - KINDS * n, 0);
        }
        return;
    }
    const bool values = u >= n;
    if (values) u -= n;
    const int window = (int)(u / (unsigned)p.H_kv), h = (int)(u - (long long)window * p.H_kv);
    each_run<W, true>(p.batch, window * W, [&](const Fp4Run& run) __attribute__((always_inline)) {
        if (run.page < 0) return;
        if (KINDS == 1 || values) append_values<T, (EPC > 1)>(p, run, h, lds[wave]);
        if (KINDS == 1 || !values) append_keys<T, EPC, LPR, IN, AX>(p, run, h, lds[wave]);
    });
}

template <typename T, bool AX>
hipError_t launch_kv_append_fp4_t(const AppendParams& p, hipStream_t stream) {
    return with_append_row<T>(p, [&](auto epc, auto lpr, auto in) {
        constexpr int E = decltype(epc)::value, L = decltype(lpr)::value;
        constexpr bool IN = decltype(in)::value;
        const auto run = [&](auto w, auto queries) {
            constexpr int W = decltype(w)::value;
            constexpr bool Q = decltype(queries)::value;
            const long long n = (W > 1 ? 1 : 2) * fp4_units<W>(p.batch.T, p.H_kv) + (Q ? append_map<L>(p.batch.T, p.H_q).units : 0);
            if (n == 0) return hipSuccess;
            return launch_kernel<kv_append_fp4_kernel<T, E, L, IN, AX, W, Q>>(
                tile_grid((n + kAppendWaves - 1) / kAppendWaves, 64 * kAppendWaves), 64 * kAppendWaves, 0, stream, p);
        };
        if (fp4_units<kFp4Run>(p.batch.T, p.H_kv) < kFp4FewWindows) return run(std::integral_constant<int, 1>{}, std::true_type{});
        const hipError_t e = run(std::integral_constant<int, kFp4Run>{}, std::false_type{});
        if (e != hipSuccess || p.H_q == 0) return e;
        AppendParams q = p;
        q.H_k = q.H_v = 0;
        return launch_kv_append(q, sizeof(T) == 2 ? DType::F16 : DType::F32, stream);
    });
}

// ---- tokens out of the pages ---------------------------------------------------

template <typename T>
__device__ __forceinline__ void store16(T* row, const half2v (&x)[8]) {
    constexpr int E = 16 / (int)sizeof(T);
    typedef T chunk __attribute__((ext_vector_type(E)));
#pragma unroll
    for (int i = 0; i < 16; i += E) {
        chunk c;
#pragma unroll
        for (int e = 0; e < E; ++e) c[e] = (T)x[(i + e) / 2][(i + e) % 2];
        *reinterpret_cast<chunk*>(row + i) = c;
    }
}

template <typename T, int W>
__global__ __launch_bounds__(64 * kAppendWaves) void kv_read_fp4_kernel(const Fp4ReadParams p) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    long long u = (long long)tile_id() * kAppendWaves + wave;
    const long long n = fp4_units<W>(p.batch.T, p.H_kv);
    if (u >= 2 * n) return;
    const bool values = u >= n;
    if (values) u -= n;
    const int window = (int)(u / (unsigned)p.H_kv), h = (int)(u - (long long)window * p.H_kv);
    const int D = values ? p.D_v : p.D_qk, log2 = p.batch.page_log2;
    T* const out = static_cast<T*>(values ? p.v : p.k) + (long long)h * D;
    const long long token = (long long)p.H_kv * D;  // elements between tokens
    each_run<W, false>(p.batch, window * W, [&](const Fp4Run& run) __attribute__((always_inline)) {
        const bool none = run.page < 0;
        const unsigned char* head = static_cast<const unsigned char*>(values ? p.v_cache : p.k_cache) +
                                    ((long long)(none ? 0 : run.page) * p.H_kv + h) * fp4_head_bytes(D, log2);
        const long long slot = run.pos & ((1 << log2) - 1);
        if (none) {
            for (int d = lane; d < D; d += 64) out[run.t * token + d] = (T)__builtin_nanf("");
        } else if (!values) {
            const int r = lane / 8, f = lane % 8 * 16;
            if (r >= run.n || f >= D) return;
            const uint2v c = *reinterpret_cast<const uint2v*>(head + (slot + r) * (D / 2) + f / 2);
            const half2v s = fp4_scale2<0>(head[fp4_scales_at(D, log2) + (slot + r) * (D / 32) + f / 32]);
            const half2v x[8] = {fp4_pair<0>(c[0]) * s, fp4_pair<1>(c[0]) * s, fp4_pair<2>(c[0]) * s, fp4_pair<3>(c[0]) * s,
                                 fp4_pair<0>(c[1]) * s, fp4_pair<1>(c[1]) * s, fp4_pair<2>(c[1]) * s, fp4_pair<3>(c[1]) * s};
            store16(out + (long long)(run.t + r) * token + f, x);
        } else {
            // features 2 lane and 2 lane + 1 of the block's 8 tokens
            if (2 * lane >= D) return;
            const long long block = slot / kFp4Run;
            const int at = (int)(slot % kFp4Run);
            const uint2v c = reinterpret_cast<const uint2v*>(head + block * D * 4)[lane];
            const uint2v s = *reinterpret_cast<const uint2v*>(head + fp4_scales_at(D, log2) + (block * (D / 32) + lane / 16) * 8);
            const half2v s2[4] = {fp4_scales2<0>(s[0]), fp4_scales2<2>(s[0]), fp4_scales2<0>(s[1]), fp4_scales2<2>(s[1])};
            const half2v a[4] = {fp4_pair<0>(c[0]) * s2[0], fp4_pair<1>(c[0]) * s2[1], fp4_pair<2>(c[0]) * s2[2],
                                 fp4_pair<3>(c[0]) * s2[3]};
            const half2v b[4] = {fp4_pair<0>(c[1]) * s2[0], fp4_pair<1>(c[1]) * s2[1], fp4_pair<2>(c[1]) * s2[2],
                                 fp4_pair<3>(c[1]) * s2[3]};
            typedef T pair __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int i = 0; i < kFp4Run; ++i)
                if (i >= at && i < at + run.n)
                    *reinterpret_cast<pair*>(out + (long long)(run.t + i - at) * token + 2 * lane) =
                        (pair){(T)a[i / 2][i % 2], (T)b[i / 2][i % 2]};
        }
    });
}

template <typename T>
hipError_t launch_kv_read_fp4_t(const Fp4ReadParams& p, hipStream_t stream) {
    const auto run = [&](auto w) {
        constexpr int W = decltype(w)::value;
        const long long n = 2 * fp4_units<W>(p.batch.T, p.H_kv);
        if (n == 0) return hipSuccess;
        return launch_kernel<kv_read_fp4_kernel<T, W>>(tile_grid((n + kAppendWaves - 1) / kAppendWaves, 64 * kAppendWaves),
                                                       64 * kAppendWaves, 0, stream, p);
    };
    if (fp4_units<kFp4Run>(p.batch.T, p.H_kv) >= kFp4FewWindows) return run(std::integral_constant<int, kFp4Run>{});
    return run(std::integral_constant<int, 1>{});
}

}  // namespace

hipError_t launch_kv_append_fp4(const AppendParams& p, DType dtype, hipStream_t stream) {
    return with_bool(p.axes.used != 0, [&](auto ax) {
        constexpr bool AX = decltype(ax)::value;
        return dtype == DType::F16 ? launch_kv_append_fp4_t<half_t, AX>(p, stream) : launch_kv_append_fp4_t<float, AX>(p, stream);
    });
}

hipError_t launch_kv_read_fp4(const Fp4ReadParams& p, DType dtype, hipStream_t stream) {
    return dtype == DType::F16 ? launch_kv_read_fp4_t<half_t>(p, stream) : launch_kv_read_fp4_t<float>(p, stream);
}

}  // namespace sdpa
