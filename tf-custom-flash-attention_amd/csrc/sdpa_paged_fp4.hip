// sdpa_paged_fp4.hip -- attention of chunks of new tokens over a paged cache in 4 bits
// (sdpa_fp4.h), queries in fp16 or fp32, for gfx950: tiles of 128 rows (tokens times
// the query heads of a key head).
//
// As in sdpa_paged_f16.hip: per wave of 32 rows (lane = row), v_mfma_f32_32x32x16_f16,
//   S^T = K Q^T, online softmax over keys in the log2 domain,
//   O^T += V^T P^T with P straight from the S accumulator,
// four waves per workgroup, blocks of 64 keys.  A block's codes become fp16 once, for all four
// waves: a thread loads its words a block ahead, converts them (exactly) and writes each, 8
// values, where the lane of the MFMA operand that wants them reads it, 16 bytes a
// lane and the lanes side by side: K by the words of a key, V by those of a feature.  So
// neither is swizzled or transposed, but that the keys are dealt to the rows of the K operand in
// the order in which a lane holds 8 neighbouring scores (which meet 8 tokens of a V word), and K words are
// written 4 lanes apart by the part of the key (whose lanes would meet in a bank).
// fp32 queries are cut into three fp16 parts, and weights into two.  With fp16 queries weights are one
// part, 11 bits, and two only where few keys carry a row (kSplitLog2), the rule of every tile of
// 128 rows over fp16: 512 tokens over 16000, 32 heads on 8, D 128, 170 us, o off by 2.9e-4 of its norm
// (its own rounding is 2.1e-4 of that); two parts throughout 213 us and 2.1e-4.
//
// Bound by issue, as the kernel over fp16 pages is: 10 vector instructions a matrix instruction
// (there 7.3), matrix cores busy 36 %.  512 tokens over 16000, 32 heads on 8, D 128: 164 us a call, 806
// TFLOP/s (172 in another run; over fp16 pages 157 to 159; a product of 8192^3 1212), 12 of it the merge.  300 tokens over 2300
// and 3 single ones, 16 heads on 4, D 64, fp32: 24 and 7 us (over fp32 pages 33 and 7).
#include "sdpa_launch.h"
#include "sdpa_paged_fp4.h"
#include "sdpa_parts.h"

namespace sdpa {
namespace {

template <typename T, int DQK, int DV>
struct PagedFp4Cfg {
    static constexpr int NP = sizeof(T) == 2 ? 1 : 3;  // parts of a query
    static constexpr int NW = 4, NT = 64 * NW, BM = kPagedBM, BN = 64;
    static constexpr int KB = BN * DQK * 2, VB = BN * DV * 2, STAGE = KB + VB;
    static constexpr size_t LDS_BYTES = 2 * (size_t)STAGE;
    static constexpr int WPE = NP == 3 && DQK > 32 ? 1 : 2;
    static_assert(WPE * LDS_BYTES <= 160 * 1024, "gfx950 LDS");
};

template <typename T, int DQK, int DV>
__global__ __launch_bounds__((PagedFp4Cfg<T, DQK, DV>::NT))
__attribute__((amdgpu_waves_per_eu(PagedFp4Cfg<T, DQK, DV>::WPE, PagedFp4Cfg<T, DQK, DV>::WPE)))
void paged_fp4_kernel(const PagedParams p) {
    using Cfg = PagedFp4Cfg<T, DQK, DV>;
    constexpr int BM = Cfg::BM, BN = Cfg::BN, NP = Cfg::NP;
    constexpr int NKS = DQK / 16, NDT = DV / 32, KW = DQK / 32;
    constexpr int PER = DV == 96 ? 1 : NDT;  // a V word's feature: PER l32 + dt (96: 32 dt + l32)
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    PagedItem it;
    {
        PagedPlan<BM, BN> plan(p);
        const int at = xcd_item(tile_id(), plan.items);
        if (at < 0 || !plan.find(at, it) || !slot_ok(p, it)) return;
    }
    const int np = it.s.parts;
    const int kv_end = min(tile_keys(p, it, BM), it.s.len);
    const int in_tile = 32 * wave + l32;
    PagedRow row;
    row.init(p, it, it.tile * BM + in_tile);
    // keys seen by the wave's first row, the fewest of its live ones, and by its last
    const bool live = it.tile * BM + 32 * wave < it.s.n * p.G;
    const int see_min = __builtin_amdgcn_readfirstlane(row.see);
    PagedRow last;
    last.init(p, it, min(it.tile * BM + 32 * wave + 31, it.s.n * p.G - 1));
    const int see_max = min(__builtin_amdgcn_readfirstlane(last.see), it.s.len);
    const int see = row.see;

    // |scale| with negated queries for scale < 0; 1e-30 for 0 (sdpa_paged_f16.hip)
    const float sl2_raw = p.scale * kLog2e;
    const bool neg = sl2_raw < 0.f;
    float sl2 = (sl2_raw == 0.f) ? 1e-30f : fabsf(sl2_raw);
    half8 q[NKS][NP];
    {
        const T* qrow = static_cast<const T*>(p.q) + row.tok * p.qs.t + row.head * p.qs.h + 8 * hh;
        if constexpr (NP == 1) {
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                half8 v = half8{};
                if (row.live) v = *reinterpret_cast<const half8*>(qrow + 16 * ks);
                q[ks][0] = neg ? -v : v;
            }
        } else {
            float x[NKS][8], most = 0.f;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    floatx4 v = floatx4{};
                    if (row.live) v = *reinterpret_cast<const floatx4*>(qrow + 16 * ks + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[ks][4 * h + e] = v[e];
                        most = fmaxf(most, fabsf(v[e]));
                    }
                }
            float f;
            query_factor(xhalf_max(most), sl2_raw, f, sl2);
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[ks][e] *= f;
                cut_queries(q[ks], x[ks]);
            }
        }
    }

    // the steps [lo, nsteps) of this workgroup
    const int steps = (kv_end + BN - 1) / BN;
    const int lo = part_begin(steps, it.part, np), nsteps = part_begin(steps, it.part + 1, np);
    Fp4Pages K, V;
    K.init(p.k_cache, p.H_kv, it.h, DQK, p.batch.page_log2);
    V.init(p.v_cache, p.H_kv, it.h, DV, p.batch.page_log2);
    PageWindow pw{uniform_ptr(p.batch.page_table + it.seq * p.batch.table_stride), p.batch.pages,
                  (min(kv_end, nsteps * BN) + (1 << K.log2) - 1) >> K.log2};

    // This thread's words of a block: of key tid / 4 those from KW (tid % 4) on, and of the 8 tokens
    // tid / 32 NDT features.  A wave's 16 keys lie in one page.
    const int key = lane >> 2, part = lane & 3;  // of the wave's 16 keys
    Fp4Keys<KW> kr;
    uint32_t vr[NDT];
    uint2v vsr[PER == 1 ? NDT : 1];
    auto load_block = [&](int step) __attribute__((always_inline)) {
        const int kv0 = step * BN + 16 * wave;
        pw.need((step * BN) >> K.log2, lane);  // (a window holds whole blocks)
        const int page = pw.held(kv0 >> K.log2);
        const int slot = K.slot(kv0);
        const fp4_ptr codes = uniform(K.page(page) + slot * (DQK / 2));
        kr.load(codes + Fp4Keys<KW>::codes_at(key, part),
                codes + (K.scales_at() + slot * (KW - DQK / 2)) + Fp4Keys<KW>::scale_at(key, part), part);
        const fp4_ptr first = uniform(V.page(page) + slot * (DV / 2));
        const fp4_ptr words = first + (uint32_t)(hh * DV * 4);
        const fp4_ptr scales = first + (V.scales_at() + slot * (DV / 32 - DV / 2)) + (uint32_t)(hh * (DV / 4));
        if constexpr (PER == 4) {
            const uint4v x = fp4_load<uint4v>(words + 16 * l32);
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[e] = x[e];
            vsr[0] = fp4_load<uint2v>(scales + 8 * (l32 / 8));
        } else if constexpr (PER == 2) {
            const uint2v x = fp4_load<uint2v>(words + 8 * l32);
            vr[0] = x[0];
            vr[1] = x[1];
            vsr[0] = fp4_load<uint2v>(scales + 8 * (l32 / 16));
        } else {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                vr[dt] = fp4_load<uint32_t>(words + 4 * (32 * dt + l32));
                vsr[dt] = fp4_load<uint2v>(scales + 8 * dt);
            }
        }
    };
    // Where the words go in a stage: K chunk (32 keys s, step ks) holds lane 32 hh + m, m the row
    // of the operand that key 16 (m / 16) + 8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4 has
    const int k32 = 16 * (wave & 1) + key;  // of 32
    const int m_row = 16 * (k32 >> 4) + 4 * ((k32 >> 3) & 1) + 8 * ((k32 >> 2) & 1) + (k32 & 3);
    const uint32_t lds0 = lds_base();
    const uint32_t kst = lds0 + (uint32_t)((wave >> 1) * NKS * 1024);
    const uint32_t vst = lds0 + Cfg::KB + (uint32_t)(wave * NDT * 1024 + lane * 16);
    const auto put = [](uint32_t at, half8 x) __attribute__((always_inline)) {
        *reinterpret_cast<__attribute__((address_space(3))) half8*>((uintptr_t)at) = x;
    };
    auto store_keys = [&](uint32_t stage) __attribute__((always_inline)) {
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            const int wi = KW * part + w;
            put(kst + stage + (uint32_t)((wi >> 1) * 1024) + (uint32_t)((((wi & 1) * 32 + m_row) ^ (4 * part)) * 16), kr.word(w, part));
        }
    };
    auto store_values = [&](uint32_t stage, int step) __attribute__((always_inline)) {
        const int left = kv_end - (step * BN + 16 * wave + 8 * hh);  // what lies behind the last key is 0
        half2v s[4];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            if (dt == 0 || PER == 1) {
                uint2v x = vsr[PER == 1 ? dt : 0];
                if ((step + 1) * BN > kv_end) x = first_bytes(x, left);
                fp4_scales(s, x);
            }
            put(vst + stage + (uint32_t)(dt * 1024), fp4_word(vr[dt], s));
        }
    };

    pw.load((lo * BN) >> K.log2, lane);
    prologue_loads_landed();
    if (lo < nsteps) {
        load_block(lo);
        store_keys(0);
        store_values(0, lo);
        if (lo + 1 < nsteps) load_block(lo + 1);
    }
    floatx16 oacc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) oacc[dt] = floatx16{};
    float m_run = kMaxSentinel, l_run = 0.f;

    // Softmax of one 32-key sub-tile (raw scores; masked keys -inf): per-lane
    // lazy maximum, alpha, the sum and the fp16 B operands of the PV product; the
    // row maximum mxo (log2 units) and P in fp32 (pf, for the hi/lo split).
    auto softmax_sub = [&](const floatx16& sc, float& m_use, float& alpha, float& lsum, float& mxo, half8& pb0, half8& pb1,
                           float (&pf)[16]) {
        float mx = sc[0];
#pragma unroll
        for (int r = 1; r < 15; r += 2) mx = max3(mx, sc[r], sc[r + 1]);
        mx = __builtin_elementwise_maximum(mx, sc[15]);
        mx = xhalf_max(mx) * sl2;
        mxo = mx;
        m_use = (mx > m_run + kTauP) ? mx - kTopP : m_run;
        alpha = fast_exp2(m_run - m_use);
        const float nm = -m_use;
        uint32_t w[8];
        float lq[4];
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) pf[r + e] = fast_exp2(__builtin_fmaf(sc[r + e], sl2, nm));
            lq[r >> 2] = (pf[r] + pf[r + 1]) + (pf[r + 2] + pf[r + 3]);
            w[r >> 1] = pack_h2(pf[r], pf[r + 1]);
            w[(r >> 1) + 1] = pack_h2(pf[r + 2], pf[r + 3]);
        }
        lsum = (lq[0] + lq[1]) + (lq[2] + lq[3]);
        pb0 = half8_of(w[0], w[1], w[2], w[3]);
        pb1 = half8_of(w[4], w[5], w[6], w[7]);
    };
    // The lo part of a split sub-tile: O^T += V^T (P - fp16(P))^T.
    auto lo_pv = [&](const half8 (&av)[2][NDT], const half8& pb0, const half8& pb1, const float (&pf)[16]) {
        uint32_t wl[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            wl[i >> 1] = pack_h2(pf[i] - (float)pb0[i], pf[i + 1] - (float)pb0[i + 1]);
            wl[4 + (i >> 1)] = pack_h2(pf[8 + i] - (float)pb1[i], pf[9 + i] - (float)pb1[i + 1]);
        }
        const half8 l0 = half8_of(wl[0], wl[1], wl[2], wl[3]), l1 = half8_of(wl[4], wl[5], wl[6], wl[7]);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            oacc[dt] = mfma_f16(av[0][dt], l0, oacc[dt]);
            oacc[dt] = mfma_f16(av[1][dt], l1, oacc[dt]);
        }
    };
    // (register r of a lane: key 16 (r / 8) + 8 hh + r % 8 of the 32)
    auto mask_sub = [&](floatx16& sc, int key0) {
        const int left = see - key0 - 8 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (16 * (r >> 3) + (r & 7) >= left) sc[r] = -INFINITY;
    };
    // Rescale the output (rare, wave-uniform branch) and fold a sub-tile into
    // the running sum.
    auto commit_sub = [&](float m_use, float alpha, float lsum) {
        if (wave_any(alpha != 1.f)) {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) oacc[dt][r] *= alpha;
        }
        l_run = __builtin_fmaf(l_run, alpha, lsum);
        m_run = m_use;
    };

    // One step = 64 keys as two 32-key sub-tiles; the next block's words are converted between
    // their products (mid0, mid1).
    auto fwd_step = [&]<bool PART>(int kv0, uint32_t so, auto&& mid0, auto&& mid1) {
        const float thr = NP == 1 ? m_run + fast_log2(xhalf_sum(l_run)) + kSplitLog2 : 0.f;
        // (opaque lane terms keep the compiler from holding every address through the loop)
        uint32_t kl = (uint32_t)lane * 16, vl = lds0 + Cfg::KB + (uint32_t)lane * 16 + so;
        asm volatile("" : "+v"(kl), "+v"(vl));
        const auto key_operand = [&](int sub, int ks) __attribute__((always_inline)) {
            const int pt = KW % 2 == 0 ? 2 * ks / KW : (2 * ks + hh) / KW;
            return ld_b128((kl ^ (uint32_t)(64 * pt)) + lds0 + so + (uint32_t)((sub * NKS + ks) * 1024));
        };
        const auto value_operands = [&](half8 (&av)[2][NDT], int sub) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) av[j][dt] = ld_b128(vl + (uint32_t)(((2 * sub + j) * NDT + dt) * 1024));
        };
        half8 ak0[NKS], ak1[NKS];
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) ak0[ks] = key_operand(0, ks);
        floatx16 s0 = floatx16{}, s1 = floatx16{};
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
#pragma unroll
            for (int n = NP - 1; n >= 0; --n) s0 = mfma_f16(ak0[ks], q[ks][n], s0);
            ak1[ks] = key_operand(1, ks);
        }
        mid0();
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
            for (int n = NP - 1; n >= 0; --n) s1 = mfma_f16(ak1[ks], q[ks][n], s1);
        half8 av0[2][NDT], av1[2][NDT];
        value_operands(av0, 0);
        if (PART && kv0 + 32 > see_min) mask_sub(s0, kv0);
        float mu0, al0, ls0, mx0, pf0[16];
        half8 p00, p01;
        softmax_sub(s0, mu0, al0, ls0, mx0, p00, p01, pf0);
        commit_sub(mu0, al0, ls0);
        if (NP > 1 || wave_any(mx0 > thr)) lo_pv(av0, p00, p01, pf0);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            oacc[dt] = mfma_f16(av0[0][dt], p00, oacc[dt]);
            oacc[dt] = mfma_f16(av0[1][dt], p01, oacc[dt]);
        }
        mid1();
        value_operands(av1, 1);
        if (PART && kv0 + 64 > see_min) mask_sub(s1, kv0 + 32);
        float mu1, al1, ls1, mx1, pf1[16];
        half8 p10, p11;
        softmax_sub(s1, mu1, al1, ls1, mx1, p10, p11, pf1);
        commit_sub(mu1, al1, ls1);
        if (NP > 1 || wave_any(mx1 > thr)) lo_pv(av1, p10, p11, pf1);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            oacc[dt] = mfma_f16(av1[0][dt], p10, oacc[dt]);
            oacc[dt] = mfma_f16(av1[1][dt], p11, oacc[dt]);
        }
    };

    // Step `step`: its block is in LDS once every wave has written its words; the next one's go
    // to the other stage, which every wave has read by then.
    auto do_step = [&]<bool PART>(int step) {
        const uint32_t so = (uint32_t)(((step - lo) & 1) * Cfg::STAGE), other = (uint32_t)Cfg::STAGE - so;
        __syncthreads();
        const bool next = step + 1 < nsteps;
        const int kv0 = step * BN;
        auto mid0 = [&]() __attribute__((always_inline)) {
            if (next) store_keys(other);
        };
        auto mid1 = [&]() __attribute__((always_inline)) {
            if (next) store_values(other, step + 1);
            if (step + 2 < nsteps) load_block(step + 2);
        };
        if (!PART || (live && kv0 < see_max)) {
            fwd_step.template operator()<PART>(kv0, so, mid0, mid1);
        } else {
            mid0();
            mid1();
        }
    };
    const int n_full = live ? min(nsteps, see_min / BN) : 0;
    int step = lo;
    for (; step < n_full; ++step) do_step.template operator()<false>(step);
    for (; step < nsteps; ++step) do_step.template operator()<true>(step);

    // ---- epilogue
    const float l_tot = xhalf_sum(l_run);
    int* none = reinterpret_cast<int*>(smem);  // waves that met a page that is none
    __syncthreads();                           // (every block has been read)
    if (lane == 0) none[wave] = pw.bad || it.s.bad;
    __syncthreads();
    const bool bad = (none[0] | none[1] | none[2] | none[3]) != 0;
    put_paged_rows_by<T, DV, BM, true, PER>(p, it, wave, row, oacc, m_run, l_tot, bad, [&](const PagedRow& rr, int r) {
        const T* qr = static_cast<const T*>(p.q) + rr.tok * p.qs.t + rr.head * p.qs.h;
        put_care_row<T, BM>(p, it, rr, r, care_row_fp4<T>(p, pw.row, K, V, qr, lo * BN, min(nsteps * BN, min(rr.see, it.s.len))));
    });
}

}  // namespace

hipError_t launch_paged_fp4(const PagedParams& p, DType dtype, hipStream_t stream) {
    const auto run = [&](auto t) {
        using T = decltype(t);
        return with_fp4_dim(p.D_qk, [&](auto dqk) {
            return with_fp4_dim(p.D_v, [&](auto dv) {
                constexpr int DQK = decltype(dqk)::value, DV = decltype(dv)::value;
                using Cfg = PagedFp4Cfg<T, DQK, DV>;
                const PagedParams a = paged_parts(p, Cfg::BN, Cfg::WPE);
                const long long n = xcd_grid(paged_max_tiles(a, Cfg::BM) + (a.divide ? 1 << a.target_log2 : 0));
                hipError_t e = launch_kernel<paged_fp4_kernel<T, DQK, DV>>(tile_grid(n, Cfg::NT), Cfg::NT, Cfg::LDS_BYTES, stream, a);
                return e == hipSuccess && a.divide ? launch_paged_merge<T, Cfg::BM, Cfg::BN>(a, stream) : e;
            });
        });
    };
    return dtype == DType::F16 ? run(half_t{}) : run(float{});
}

}  // namespace sdpa
