// sdpa_paged_f16_small.hip -- attention of few new tokens per sequence
// (generation, short drafts) over a paged cache, fp16, for gfx950.
//
// A workgroup walks an equal share of the key blocks of all tiles of 32 rows
// (tokens times the query heads of a key head; sdpa_paged.h); its four waves take
// the 32-key blocks of a tile in turn, each with running statistics and sums of its
// own, which are merged through LDS in wave order at a tile's end.  Each wave copies
// its blocks into LDS of its own (sdpa_dma.h), without a barrier in the loop, and
// reads a block's operands into registers whole, so that the next block's copies fly
// while this one is worked on.
//   S^T = K Q^T, online softmax in the log2 domain, O^T += V^T P^T
// with P taken from the S accumulators straight into the MFMA operand, as one
// fp16 part, two where few keys carry a row (sdpa_device.h, kSplitLog2).
//
// Pages: a copy moves whole rows of one 16-row group, which lies in one page;
// the page numbers of 64 columns are held in the lanes of a register, and the
// descriptor of a group ends at its last key, so that what a page holds behind
// a sequence is never read.
//
// Bound by memory: the cache is read once per key head, with the non-temporal
// hint (plain loads: 6.0 TB/s where these reach 6.7; copies of 16 KB alone, in no order, 1 GB).
// 64 sequences of 5120 tokens, 8 key heads, D 128 (1342 MB): 214 us with the
// merge, 6.3 TB/s; of 600 to 16384 tokens (1328 MB) 219.  Two workgroups per CU hide
// each other's ends of tiles: 512 sequences of 640 tokens 242 us, where one and a
// two-stage ring took 325 against 257 (and 4 sequences of 4096, 16 heads, 31.2
// against 32.7; 30 now).  Parts of tiles (sdpa_paged.h) instead of shares: 1328 MB in 218 to
// 255 us, by the number of parts, against 232.
#include "sdpa_launch.h"
#include "sdpa_paged_device.h"
#include "sdpa_parts.h"
#include "sdpa_wave.h"

namespace sdpa {
namespace {

template <int DQK, int DV>
struct PagedSmallCfg {
    static constexpr int NW = 4, NT = 64 * NW, BM = kPagedSmallBM, BN = 32, PLAN = BN * NW;
    static constexpr int LK = lds_chunks(DQK), LV = lds_chunks(DV);
    static constexpr int KB = BN * LK * 16, VB = BN * LV * 16, STAGE = KB + VB;
    // merge area (after the loop): O of every wave, m and l, flags of rows and waves
    static constexpr int OS = acc_stride(DV), MERGE = NW * BM * OS * 4 + NW * BM * 8 + (BM + NW) * 4;
    static constexpr int PLAN_AT = NW * STAGE > MERGE ? NW * STAGE : (MERGE + 15) / 16 * 16;  // the plan, behind them
    static constexpr size_t LDS_BYTES = PLAN_AT + PagedShares<BM, PLAN>::LDS_BYTES;
    static constexpr int WPE = 2;
    static_assert(WPE * LDS_BYTES <= 160 * 1024, "gfx950 LDS");
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
        for (int u = 0; u < LOADS; ++u) dma16_at_nt(rs, m0 + 1024u * u, voff[u]);
    }
};

template <int DQK, int DV>
__global__ __launch_bounds__((PagedSmallCfg<DQK, DV>::NT))
__attribute__((amdgpu_waves_per_eu(PagedSmallCfg<DQK, DV>::WPE, PagedSmallCfg<DQK, DV>::WPE)))
void paged_f16_small_kernel(const PagedParams p) {
    using Cfg = PagedSmallCfg<DQK, DV>;
    constexpr int BM = Cfg::BM, BN = Cfg::BN, LK = Cfg::LK, LV = Cfg::LV, NW = Cfg::NW;
    constexpr int NKS = DQK / 16, NDT = DV / 32;
    const int D_qk = p.D_qk, D_v = p.D_v;
    const PagedShares<BM, Cfg::PLAN> plan(p, smem + Cfg::PLAN_AT);
    plan.each(tile_id(), [&](const PagedItem& it) __attribute__((always_inline)) {
        int tid = threadIdx.x;  // (opaque: lane terms are formed for each tile, not held across them)
        asm volatile("" : "+v"(tid));
        const int lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
        const int lo = min(NW * it.u0, nblk), hi = min(NW * it.u1, nblk);
        const uint32_t ring = lds_base() + (uint32_t)(wave * Cfg::STAGE);
        PagedRows K, V;
        K.init(p.k_cache, p.H_kv, it.h, D_qk, 2, p.batch.page_log2);
        V.init(p.v_cache, p.H_kv, it.h, D_v, 2, p.batch.page_log2);
        PageWindow pw{uniform_ptr(p.batch.page_table + it.seq * p.batch.table_stride), p.batch.pages,
                      (min(kv_end, hi * BN) + (1 << K.log2) - 1) >> K.log2};
        GroupCopy<LK, false> kc;
        GroupCopy<LV, true> vc;
        kc.init(lane, D_qk * 2, D_qk / 8);
        vc.init(lane, D_v * 2, D_v / 8);
        auto issue = [&](int blk) __attribute__((always_inline)) {
            pw.need((blk * BN) >> K.log2, lane);  // (a window holds whole blocks)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int r0 = blk * BN + 16 * g, page = pw.held(r0 >> K.log2);
                kc.issue(K.rows(page, r0, kv_end, 16), ring + (uint32_t)(256 * LK * g));
                vc.issue(V.rows(page, r0, kv_end, 16), ring + (uint32_t)(Cfg::KB + 256 * LV * g));
            }
        };
        pw.load((lo * BN) >> K.log2, lane);
        prologue_loads_landed();
        if (lo + wave < hi) issue(lo + wave);

        SwzLane<LK> swK;
        swK.init(lane);
        const uint32_t rkl = ring + swK.row;                          // K rows (^ 32 ks)
        const uint32_t tvl = ring + Cfg::KB + tr_lane_off<LV>(lane);  // V^T (^ 64 dt)
        floatx16 oacc[NDT];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) oacc[dt] = floatx16{};
        float m_run = -INFINITY, l_run = 0.f;

        for (int blk = lo + wave; blk < hi; blk += NW) {
            wait_copies<0>();
            const int kv0 = blk * BN;
            const float split_thr = m_run + fast_log2(xhalf_sum(l_run)) + kSplitLog2;
            // (opaque lane terms: their offsets are formed here, not held)
            uint32_t kl = rkl, vl = tvl;
            asm volatile("" : "+v"(kl), "+v"(vl));
            floatx16 s = floatx16{};
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) s = mfma_f16(ld_b128(kl ^ (uint32_t)(32 * ks)), qreg[ks], s);
            half8 av[2][NDT];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
                    const uint32_t a = (vl ^ (uint32_t)(64 * dt)) + 16 * LV * 16 * j;
                    av[j][dt] = ld_tr8(a, a + 16 * LV * 8);
                }
            // the block is in registers: the next one's copies fly while this one is
            // worked on
            lds_reads_done();
            if (blk + NW < hi) issue(blk + NW);
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
            const float m_use = (mx > m_run + kTauP) ? mx - kTopP : m_run;
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
        __syncthreads();
    });
}

}  // namespace

hipError_t launch_paged_f16_small(const PagedParams& p, hipStream_t stream) {
    return with_paged_dim(p.D_qk, [&](auto dqk) {
        return with_paged_dim(p.D_v, [&](auto dv) {
            constexpr int DQK = decltype(dqk)::value, DV = decltype(dv)::value;
            using Cfg = PagedSmallCfg<DQK, DV>;
            hipError_t e = launch_kernel<paged_f16_small_kernel<DQK, DV>>(dim3(1u << p.target_log2), Cfg::NT, Cfg::LDS_BYTES,
                                                                         stream, p);
            return e == hipSuccess && paged_shares_divide(p, Cfg::PLAN)
                       ? launch_paged_share_merge<half_t, Cfg::BM, Cfg::PLAN>(p, stream)
                       : e;
        });
    });
}

}  // namespace sdpa
