// sdpa_paged_f16.hip -- attention of chunks of new tokens over a paged cache,
// fp16, for gfx950: tiles of 128 rows (tokens times the query heads of a key
// head).
//
// Per wave of 32 rows (lane = row), v_mfma_f32_32x32x16_f16:
//   S^T = K Q^T, online softmax over keys in the log2 domain,
//   O^T += V^T P^T with P straight from the S accumulator,
// four waves per workgroup, two workgroups per CU (three at D <= 64), blocks of 64 keys
// through an LDS ring filled by direct copies, one barrier per block, as in the
// dense forward (sdpa_f16_fwd.hip), whose step this is without the dropout.  Rows of
// several tokens and heads share a wave, so the mask is a number of keys per
// lane; steps that every row of the wave sees whole run without it.
//
// Pages: a wave's copy moves rows of one 16-row group, which lies in one page.
// Where a page holds whole blocks, one descriptor serves a block's copies;
// else each copy has its own.  A descriptor ends at the tile's last key.
//
// Bound by issue, as the dense forward is.  4 x 4096 tokens, 32 heads on 8, D 128: 618
// us a call, 890 TFLOP/s (a product of 8192^3 1159), pages of 16 instead of 64: 654; 512
// tokens over 16000 (four parts a tile) 159 us, 11 of it the merge.  A short call is a
// chain: 1.5 us for the plan, 0.9 for queries and page table, 0.5 for the first block,
// 1 for each block of a workgroup alone on its CU, 1 for the results.
#include "sdpa_launch.h"
#include "sdpa_paged_device.h"
#include "sdpa_parts.h"

namespace sdpa {
namespace {

template <int DQK, int DV>
struct PagedCfg {
    static constexpr int NW = 4, NT = 64 * NW, BM = kPagedBM, BN = 64;
    static constexpr int LK = lds_chunks(DQK), LV = lds_chunks(DV);
    static constexpr int KB = BN * LK * 16, VB = BN * LV * 16, STAGE = KB + VB;
    static constexpr int NSTAGE = 2 * 3 * STAGE <= 160 * 1024 ? 3 : 2;
    static constexpr size_t LDS_BYTES = NSTAGE * (size_t)STAGE;
    static_assert(2 * LDS_BYTES <= 160 * 1024, "two workgroups per CU in gfx950 LDS");
    static_assert(KB + VB <= 65536, "LDS immediates");
    static constexpr int WPE = (DQK <= 64 && DV <= 64 && 3 * LDS_BYTES <= 160 * 1024) ? 3 : 2;
};

// Copies of a 64-row tile of 16 L bytes a row by four waves: copy u of wave w
// fills 1 KB, rows (4 u + w) 64 / L and on.
template <int L, bool TR>
struct PagedTileCopy {
    static constexpr int NW = 4, PER_WAVE = L / NW, RPC = 64 / L;
    uint32_t voff;   // from the first row of the copy's 16-row group
    uint32_t voff64;  // from the first row of the tile's 16-row group of copy 0
    __device__ __forceinline__ static int group(int u, int wave) { return (NW * u + wave) * RPC / 16; }
    __device__ __forceinline__ void init(int wave, int lane, int row_bytes, int valid_chunks) {
        const int r = (wave * RPC) % 16 + lane / L;
        const int c = (lane % L) ^ (TR ? swz_tr<L>(r) : swz<L>(r));
        const bool ok = c < valid_chunks;
        voff = ok ? (uint32_t)(r * row_bytes + c * 16) : kOob;
        voff64 = ok ? (uint32_t)((r + 16 * group(0, wave)) * row_bytes + c * 16) : kOob;
    }
    // the tile lies in one page; rs covers its rows
    __device__ __forceinline__ void issue_whole(rsrc_t rs, uint32_t m0wave, int row_bytes) const {
#pragma unroll
        for (int u = 0; u < PER_WAVE; ++u)
            dma16_at(rs, m0wave + (uint32_t)(u * NW * 1024), voff64 + (uint32_t)(u * NW * RPC * row_bytes));
    }
};

// The sums of a wave's 32 rows over the keys [k0, k1) again, where some came out NaN
// (sdpa_paged_device.h): finite values weighted as before, by the final
// reference, then the infinite and NaN ones among each row's keys, counted by sign as
// products of ones.  Operands straight from the cache; a wave by itself.  4 x 4096
// tokens with an infinity in the first: 20 ms, where one row after the other took 208.
template <int NKS, int NDT>
__device__ __forceinline__ void care_wave(const PagedParams& p, const PagedRows& K, const PagedRows& V, const int32_t* table,
                                          const half8 (&q)[NKS], floatx16 (&oacc)[NDT], float m, float sl2, int see, int k0,
                                          int k1, int kv_end) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // (nothing of this is formed ahead of the kernel's loop)
    const int l32 = lane & 31, hh = lane >> 5;
    // V[key(j, i)][32 dt + l32], the key in the order of the scores' registers
    const auto value = [&](int at, int j, int dt, int i) {
        const int key = min(at + 16 * j + 8 * (i >> 2) + 4 * hh + (i & 3), kv_end - 1), d = 32 * dt + l32;
        return d < p.D_v ? reinterpret_cast<const half_t*>(V.at(table[key >> V.log2], key))[d] : (half_t)0.f;
    };
    const auto finite = [](half_t x) { return (__builtin_bit_cast(uint16_t, x) & 0x7C00) != 0x7C00; };
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) oacc[dt] = floatx16{};
    for (int at = k0; at < k1; at += 32) {
        const int key = min(at + l32, kv_end - 1);
        const half_t* k = reinterpret_cast<const half_t*>(K.at(table[key >> K.log2], key));
        floatx16 s = floatx16{};
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            const int d = 16 * ks + 8 * hh;
            half8 a = half8{};
            if (d < p.D_qk) a = *reinterpret_cast<const half8*>(k + d);
            s = mfma_f16(a, q[ks], s);
        }
#pragma unroll 1
        for (int j = 0; j < 2; ++j) {
            half8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = j == 0 ? s[i] : s[8 + i];
                const bool seen = at + 16 * j + 8 * (i >> 2) + 4 * hh + (i & 3) < see;
                const float w = seen ? fast_exp2(__builtin_fmaf(x, sl2, -m)) : 0.f;
                hi[i] = (half_t)w;
                lo[i] = (half_t)(w - (float)hi[i]);
            }
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                half8 v;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const half_t x = value(at, j, dt, i);
                    v[i] = finite(x) ? x : (half_t)0.f;
                }
                oacc[dt] = mfma_f16(v, lo, oacc[dt]);
                oacc[dt] = mfma_f16(v, hi, oacc[dt]);
            }
        }
    }
    // (an infinity and one of the other sign, or a NaN, which counts as both, make NaN)
#pragma unroll 1
    for (int sign = 0; sign < 2; ++sign) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            floatx16 n = floatx16{};
#pragma unroll 1
            for (int at = k0; at < k1; at += 16) {
                half8 seen, v;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    seen[i] = (half_t)(at + 8 * (i >> 2) + 4 * hh + (i & 3) < see ? 1.f : 0.f);
                    const half_t x = value(at, 0, dt, i);
                    const bool counts = !finite(x) && (x != x || (x < (half_t)0.f) == (sign != 0));
                    v[i] = (half_t)(counts ? 1.f : 0.f);
                }
                n = mfma_f16(v, seen, n);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (n[r] > 0.f) oacc[dt][r] += sign ? -INFINITY : INFINITY;
        }
    }
}

template <int DQK, int DV>
__global__ __launch_bounds__((PagedCfg<DQK, DV>::NT))
__attribute__((amdgpu_waves_per_eu(PagedCfg<DQK, DV>::WPE, PagedCfg<DQK, DV>::WPE)))
void paged_f16_kernel(const PagedParams p) {
    using Cfg = PagedCfg<DQK, DV>;
    constexpr int BM = Cfg::BM, BN = Cfg::BN, LK = Cfg::LK, LV = Cfg::LV, NSTAGE = Cfg::NSTAGE;
    constexpr int NKS = DQK / 16, NDT = DV / 32;
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    PagedItem it;
    {
        PagedPlan<BM, BN> plan(p);
        const int at = xcd_item(tile_id(), plan.items);
        if (at < 0 || !plan.find(at, it) || !slot_ok(p, it)) return;
    }
    const int D_qk = p.D_qk, D_v = p.D_v, np = it.s.parts;
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

    // |scale| with negated queries for scale < 0; 1e-30 for 0 (sdpa_f16_fwd.hip)
    const float sl2_raw = p.scale * kLog2e;
    const bool neg = sl2_raw < 0.f;
    const float sl2 = (sl2_raw == 0.f) ? 1e-30f : fabsf(sl2_raw);
    half8 qreg[NKS];
    {
        const half_t* qrow = static_cast<const half_t*>(p.q) + row.tok * p.qs.t + row.head * p.qs.h;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            const int d = 16 * ks + 8 * hh;
            half8 v = half8{};
            if (row.live && d < D_qk) v = *reinterpret_cast<const half8*>(qrow + d);
            qreg[ks] = neg ? -v : v;
        }
    }

    // the steps [lo, nsteps) of this workgroup
    const int steps = (kv_end + BN - 1) / BN;
    const int lo = part_begin(steps, it.part, np), nsteps = part_begin(steps, it.part + 1, np);
    PagedRows K, V;
    K.init(p.k_cache, p.H_kv, it.h, D_qk, 2, p.batch.page_log2);
    V.init(p.v_cache, p.H_kv, it.h, D_v, 2, p.batch.page_log2);
    PageWindow pw{uniform_ptr(p.batch.page_table + it.seq * p.batch.table_stride), p.batch.pages,
                  (min(kv_end, nsteps * BN) + (1 << K.log2) - 1) >> K.log2};
    PagedTileCopy<LK, false> kc;
    PagedTileCopy<LV, true> vc;  // V is read only transposed
    kc.init(wave, lane, D_qk * 2, D_qk / 8);
    vc.init(wave, lane, D_v * 2, D_v / 8);
    const uint32_t lds0 = lds_base();
    const uint32_t m0w = lds0 + 1024u * (uint32_t)wave;
    // copy of key block `step` into its ring slot (step % NSTAGE)
    auto issue = [&](int step) __attribute__((always_inline)) {
        const int kv0 = step * BN;
        const uint32_t mk = m0w + (uint32_t)((step % NSTAGE) * Cfg::STAGE), mv = mk + (uint32_t)Cfg::KB;
        pw.need(kv0 >> K.log2, lane);  // (a window holds whole blocks)
        if (K.log2 >= 6) {
            const int page = pw.held(kv0 >> K.log2);
            kc.issue_whole(K.rows(page, kv0, kv_end, BN), mk, K.row_bytes);
            vc.issue_whole(V.rows(page, kv0, kv_end, BN), mv, V.row_bytes);
        } else {
            const auto copy = [&](const PagedRows& m, const auto& c, uint32_t m0) __attribute__((always_inline)) {
                using C = std::decay_t<decltype(c)>;
#pragma unroll
                for (int u = 0; u < C::PER_WAVE; ++u) {
                    const int r0 = kv0 + 16 * C::group(u, wave);
                    dma16_at(m.rows(pw.held(r0 >> m.log2), r0, kv_end, 16), m0 + (uint32_t)(u * 4 * 1024), c.voff);
                }
            };
            copy(K, kc, mk);
            copy(V, vc, mv);
        }
    };
    // copies this wave issues per block (its vmcnt waits count only those)
    constexpr int CPB = PagedTileCopy<LK, false>::PER_WAVE + PagedTileCopy<LV, true>::PER_WAVE;
    pw.load((lo * BN) >> K.log2, lane);
    prologue_loads_landed();
#pragma unroll
    for (int i = 0; i < NSTAGE - 1; ++i)
        if (lo + i < nsteps) issue(lo + i);

    SwzLane<LK> swK;
    swK.init(lane);
    const uint32_t rkl = lds0 + swK.row;                          // K rows (^ 32 ks)
    const uint32_t tvl = lds0 + Cfg::KB + tr_lane_off<LV>(lane);  // V^T (^ 64 dt)
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
    auto mask_sub = [&](floatx16& sc, int key0) {
        const int left = see - key0 - 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + (r & 3) >= left) sc[r] = -INFINITY;
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

    // One step = 64 keys as two 32-key sub-tiles in software-pipeline order: each
    // MFMA group has independent work next to it (sdpa_f16_fwd.hip).
    auto fwd_step = [&]<bool PART>(int kv0, uint32_t so, auto&& mid) {
        const float thr = m_run + fast_log2(xhalf_sum(l_run)) + kSplitLog2;
        // read addresses of this step (opaque lane terms keep the compiler from
        // hoisting twelve of them into registers for the loop)
        uint32_t kl = rkl, vl = tvl;
        asm volatile("" : "+v"(kl), "+v"(vl));
        uint32_t rk[NKS], tv[NDT];
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) rk[ks] = (kl ^ (uint32_t)(32 * ks)) + so;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) tv[dt] = (vl ^ (uint32_t)(64 * dt)) + so;
        half8 ak0[NKS], ak1[NKS];
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) ak0[ks] = ld_b128(rk[ks]);
        floatx16 s0 = floatx16{}, s1 = floatx16{};
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            s0 = mfma_f16(ak0[ks], qreg[ks], s0);
            ak1[ks] = ld_b128(rk[ks] + 16 * LK * 32);
        }
        mid(1);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) s1 = mfma_f16(ak1[ks], qreg[ks], s1);
        half8 av0[2][NDT], av1[2][NDT];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
                av0[j][dt] = ld_tr8(tv[dt] + 16 * LV * 16 * j, tv[dt] + 16 * LV * (16 * j + 8));
        if (PART && kv0 + 32 > see_min) mask_sub(s0, kv0);
        float mu0, al0, ls0, mx0, pf0[16];
        half8 p00, p01;
        softmax_sub(s0, mu0, al0, ls0, mx0, p00, p01, pf0);
        commit_sub(mu0, al0, ls0);
        if (wave_any(mx0 > thr)) lo_pv(av0, p00, p01, pf0);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            oacc[dt] = mfma_f16(av0[0][dt], p00, oacc[dt]);
            oacc[dt] = mfma_f16(av0[1][dt], p01, oacc[dt]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
                av1[j][dt] = ld_tr8(tv[dt] + 16 * LV * (32 + 16 * j), tv[dt] + 16 * LV * (40 + 16 * j));
        if (PART && kv0 + 64 > see_min) mask_sub(s1, kv0 + 32);
        float mu1, al1, ls1, mx1, pf1[16];
        half8 p10, p11;
        softmax_sub(s1, mu1, al1, ls1, mx1, p10, p11, pf1);
        commit_sub(mu1, al1, ls1);
        if (wave_any(mx1 > thr)) lo_pv(av1, p10, p11, pf1);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            oacc[dt] = mfma_f16(av1[0][dt], p10, oacc[dt]);
            oacc[dt] = mfma_f16(av1[1][dt], p11, oacc[dt]);
        }
    };

    // Step `step`: wait for its block (the copies of the NSTAGE - 2 later blocks
    // may still fly; none at the tail), synchronise, multiply, and copy block
    // step + NSTAGE - 1 into the slot of block step - 1, which every wave has
    // read: waves 0 and 1 right after the barrier, waves 2 and 3 after the first
    // products, so that the four do not queue behind each other.
    auto do_step = [&]<bool PART>(int step) {
        const uint32_t so = (uint32_t)((step % NSTAGE) * Cfg::STAGE);
        if (step + NSTAGE - 2 < nsteps) wait_vm_n<(NSTAGE - 2) * CPB>();
        else wait_vm();
        __syncthreads();
        const bool cp = step + NSTAGE - 1 < nsteps, late = wave >= 2;
        if (cp && !late) issue(step + NSTAGE - 1);
        const int kv0 = step * BN;
        auto mid = [&](int) __attribute__((always_inline)) {
            if (cp && late) issue(step + NSTAGE - 1);
        };
        if (!PART || (live && kv0 < see_max)) fwd_step.template operator()<PART>(kv0, so, mid);
        else if (cp && late) issue(step + NSTAGE - 1);
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
    if (!bad && wave_any(row.live && l_tot == l_tot && any_nonfinite<NDT>(oacc)))
        care_wave<NKS, NDT>(p, K, V, pw.row, qreg, oacc, m_run, sl2, see, lo * BN, min(nsteps * BN, see_max), kv_end);
    put_paged_rows<half_t, DV, BM, false>(p, it, wave, row, oacc, m_run, l_tot, bad, pw.row, K, V, lo * BN, nsteps * BN);
}

}  // namespace

hipError_t launch_paged_f16(const PagedParams& p, hipStream_t stream) {
    return with_paged_dim(p.D_qk, [&](auto dqk) {
        return with_paged_dim(p.D_v, [&](auto dv) {
            constexpr int DQK = decltype(dqk)::value, DV = decltype(dv)::value;
            using Cfg = PagedCfg<DQK, DV>;
            const PagedParams a = paged_parts(p, Cfg::BN, 2);
            const long long n = xcd_grid(paged_max_tiles(a, Cfg::BM) + (a.divide ? 1 << a.target_log2 : 0));
            hipError_t e = launch_kernel<paged_f16_kernel<DQK, DV>>(tile_grid(n, Cfg::NT), Cfg::NT, Cfg::LDS_BYTES, stream, a);
            return e == hipSuccess && a.divide ? launch_paged_merge<half_t, Cfg::BM, Cfg::BN>(a, stream) : e;
        });
    });
}

}  // namespace sdpa
