// sdpa_paged_f16_small.hip -- attention of few new tokens per sequence
// (generation, short drafts) over a paged cache, fp16, for gfx950.
//
// A workgroup owns a tile of 32 rows (tokens times the query heads of a key
// head) and a part of its keys; its four waves take the 32-key blocks in turn,
// each with running statistics and sums of its own, which are merged through
// LDS in wave order at the end.  Each wave streams its blocks through a
// two-stage LDS ring of its own by direct copies (sdpa_dma.h), without a
// barrier in the loop: 32 KB of K and V per wave at D = 128, half of it in
// flight while the other half is multiplied.
//   S^T = K Q^T, online softmax in the log2 domain, O^T += V^T P^T
// with P taken from the S accumulators straight into the MFMA operand, as one
// fp16 part, two where few keys carry a row (sdpa_device.h, kSplitLog2).
//
// Pages: a copy moves whole rows of one 16-row group, which lies in one page;
// the page numbers of 64 columns are held in the lanes of a register, and the
// descriptor of a group ends at its last key, so that what a page holds behind
// a sequence is never read.
//
// Bound by memory: the cache is read once per key head.
#include "sdpa_launch.h"
#include "sdpa_paged_device.h"
#include "sdpa_parts.h"
#include "sdpa_wave.h"

namespace sdpa {
namespace {

constexpr float kTauP = 8.0f;  // lazy-rescale threshold (log2 units)

template <int DQK, int DV>
struct PagedSmallCfg {
    static constexpr int NW = 4, NT = 64 * NW, BM = kPagedSmallBM, BN = 32, PLAN = BN * NW;
    static constexpr int LK = DQK / 8, LV = DV / 8;
    static constexpr int KB = BN * DQK * 2, VB = BN * DV * 2, STAGE = KB + VB, RING = 2 * STAGE;
    // merge area (after the loop): O of every wave, m and l, flags of rows and waves
    static constexpr int OS = acc_stride(DV), MERGE = NW * BM * OS * 4 + NW * BM * 8 + (BM + NW) * 4;
    static constexpr size_t LDS_BYTES = NW * RING > MERGE ? NW * RING : MERGE;
    static_assert(LDS_BYTES <= 160 * 1024, "gfx950 LDS");
    static constexpr int WPE = 2 * LDS_BYTES <= 160 * 1024 ? 2 : 1;
    static constexpr int COPIES = LK / 2 + LV / 2;
};

// Copies of a 16-row group of a tile of 16 L bytes a row by one wave.
template <int L, bool TR>
struct GroupCopy {
    static constexpr int LOADS = L / 4, RPC = 64 / L;
    uint32_t voff[LOADS];
    __device__ __forceinline__ void init(int lane, int row_bytes, int valid_chunks) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int r = RPC * u + lane / L;
            const int c = (lane % L) ^ (TR ? swz_tr<L>(r) : swz<L>(r));
            voff[u] = c < valid_chunks ? (uint32_t)(r * row_bytes + c * 16) : kOob;
        }
    }
    __device__ __forceinline__ void issue(rsrc_t rs, uint32_t m0) const {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) dma16_at(rs, m0 + 1024u * u, voff[u]);
    }
};

template <int DQK, int DV>
__global__ __launch_bounds__((PagedSmallCfg<DQK, DV>::NT))
__attribute__((amdgpu_waves_per_eu(PagedSmallCfg<DQK, DV>::WPE, PagedSmallCfg<DQK, DV>::WPE)))
void paged_f16_small_kernel(const PagedParams p) {
    using Cfg = PagedSmallCfg<DQK, DV>;
    constexpr int BM = Cfg::BM, BN = Cfg::BN, LK = Cfg::LK, LV = Cfg::LV, NW = Cfg::NW;
    constexpr int NKS = DQK / 16, NDT = DV / 32;
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    PagedPlan<BM, Cfg::PLAN> plan(p);
    PagedItem it;
    {
        const int at = xcd_item(tile_id(), plan.template items<false>());
        if (at < 0 || !plan.template find<false>(at, it) || !slot_ok(p, it)) return;
    }
    const int D_qk = p.D_qk, D_v = p.D_v, np = it.s.parts;
    const int kv_end = min(tile_keys(p, it, BM), it.s.len);
    PagedRow row;
    row.init(p, it, it.tile * BM + l32);

    // |scale| with negated queries for scale < 0; 1e-30 for 0: the running
    // maximum is taken on raw scores, which needs a positive factor
    const float sl2_raw = p.scale * kLog2e;
    const bool neg = sl2_raw < 0.f;
    const float sl2 = (sl2_raw == 0.f) ? 1e-30f : fabsf(sl2_raw);
    half8 qreg[NKS];
    const half_t* qrow = static_cast<const half_t*>(p.q) + row.tok * p.qs.t + row.head * p.qs.h;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
        const int d = 16 * ks + 8 * hh;
        half8 v = half8{};
        if (row.live && d < D_qk) v = *reinterpret_cast<const half8*>(qrow + d);
        qreg[ks] = neg ? -v : v;
    }

    // this wave's blocks: lo + wave, lo + wave + NW, ... below hi
    const int nblk = (kv_end + BN - 1) / BN;
    const int lo = part_begin(nblk, it.part, np), hi = part_begin(nblk, it.part + 1, np);
    const uint32_t ring = lds_base() + (uint32_t)(wave * Cfg::RING);
    PagedRows K, V;
    K.init(p.k_cache, p.H_kv, it.h, D_qk, 2, p.batch.page_log2);
    V.init(p.v_cache, p.H_kv, it.h, D_v, 2, p.batch.page_log2);
    PageWindow pw{uniform_ptr(p.batch.page_table + it.seq * p.batch.table_stride), p.batch.pages,
                  (min(kv_end, hi * BN) + (1 << K.log2) - 1) >> K.log2};
    GroupCopy<LK, false> kc;
    GroupCopy<LV, true> vc;
    kc.init(lane, D_qk * 2, D_qk / 8);
    vc.init(lane, D_v * 2, D_v / 8);
    auto issue = [&](int blk, uint32_t so) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int r0 = blk * BN + 16 * g;
            const int page = r0 < kv_end ? pw.page(r0 >> K.log2, lane) : -1;
            kc.issue(K.rows(page, r0, kv_end, 16), ring + so + (uint32_t)(256 * LK * g));
            vc.issue(V.rows(page, r0, kv_end, 16), ring + so + (uint32_t)(Cfg::KB + 256 * LV * g));
        }
    };
    prologue_loads_landed();
    if (lo + wave < hi) issue(lo + wave, 0);

    SwzLane<LK> swK;
    swK.init(lane);
    const uint32_t rkl = ring + swK.row;                          // K rows (^ 32 ks)
    const uint32_t tvl = ring + Cfg::KB + tr_lane_off<LV>(lane);  // V^T (^ 64 dt)
    floatx16 oacc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) oacc[dt] = floatx16{};
    float m_run = -INFINITY, l_run = 0.f;

    uint32_t so = 0;
    for (int blk = lo + wave; blk < hi; blk += NW, so ^= (uint32_t)Cfg::STAGE) {
        // the other stage's block has been read; the next block's copies go
        // out there, and this block's have landed once only those are in flight
        lds_reads_done();
        if (blk + NW < hi) {
            issue(blk + NW, so ^ (uint32_t)Cfg::STAGE);
            wait_copies<Cfg::COPIES>();
        } else {
            wait_copies<0>();
        }
        const int kv0 = blk * BN;
        const float split_thr = m_run + fast_log2(xhalf_sum(l_run)) + kSplitLog2;
        floatx16 s = floatx16{};
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) s = mfma_f16(ld_b128((rkl ^ (uint32_t)(32 * ks)) + so), qreg[ks], s);
        half8 av[2][NDT];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                const uint32_t a = (tvl ^ (uint32_t)(64 * dt)) + so + 16 * LV * 16 * j;
                av[j][dt] = ld_tr8(a, a + 16 * LV * 8);
            }
        if (wave_any(kv0 + BN > row.see)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = kv0 + 8 * (r >> 2) + 4 * hh + (r & 3);
                if (key >= row.see) s[r] = -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx = xhalf_max(mx) * sl2;
        const float m_use = (mx > m_run + kTauP) ? mx : m_run;
        const float alpha = m_use == m_run ? 1.f : fast_exp2(m_run - m_use);
        const float nm = m_use == -INFINITY ? 0.f : -m_use;
        float lq[4], pf[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
#pragma unroll
            for (int e = 0; e < 4; ++e) pf[4 * g + e] = fast_exp2(__builtin_fmaf(s[4 * g + e], sl2, nm));
            lq[g] = (pf[4 * g] + pf[4 * g + 1]) + (pf[4 * g + 2] + pf[4 * g + 3]);
        }
        if (wave_any(alpha != 1.f)) {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) oacc[dt][r] *= alpha;
        }
        l_run = __builtin_fmaf(l_run, alpha, (lq[0] + lq[1]) + (lq[2] + lq[3]));
        m_run = m_use;
        half8 pb[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
            pb[j] = half8_of(pack_h2(pf[8 * j], pf[8 * j + 1]), pack_h2(pf[8 * j + 2], pf[8 * j + 3]),
                             pack_h2(pf[8 * j + 4], pf[8 * j + 5]), pack_h2(pf[8 * j + 6], pf[8 * j + 7]));
        if (wave_any(mx > split_thr)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float lo8[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) lo8[i] = pf[8 * j + i] - (float)pb[j][i];
                const half8 pl = half8_of(pack_h2(lo8[0], lo8[1]), pack_h2(lo8[2], lo8[3]),
                                          pack_h2(lo8[4], lo8[5]), pack_h2(lo8[6], lo8[7]));
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) oacc[dt] = mfma_f16(av[j][dt], pl, oacc[dt]);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) oacc[dt] = mfma_f16(av[j][dt], pb[j], oacc[dt]);
    }

    // ---- merge the four waves: every ring has been read
    __syncthreads();
    merge_paged_waves<half_t, DV, NW, BM>(p, it, reinterpret_cast<float*>(smem), oacc, m_run, xhalf_sum(l_run),
                                          pw.bad || it.s.bad, pw.row, K, V, lo * BN, hi * BN);
}

}  // namespace

hipError_t launch_paged_f16_small(const PagedParams& p, hipStream_t stream) {
    return with_dim(p.D_qk, [&](auto dqk) {
        return with_dim(p.D_v, [&](auto dv) {
            constexpr int DQK = decltype(dqk)::value, DV = decltype(dv)::value;
            using Cfg = PagedSmallCfg<DQK, DV>;
            const bool divide = paged_may_divide(p, Cfg::PLAN);
            PagedParams a = p;
            if (!divide) a.target = 0;
            const long long n = xcd_grid(paged_max_tiles(a, Cfg::BM) + a.target);
            hipError_t e = launch_kernel<paged_f16_small_kernel<DQK, DV>>(tile_grid(n, Cfg::NT), Cfg::NT, Cfg::LDS_BYTES,
                                                                         stream, a);
            return e == hipSuccess && divide ? launch_paged_merge<half_t, Cfg::BM, Cfg::PLAN>(a, stream) : e;
        });
    });
}

}  // namespace sdpa
