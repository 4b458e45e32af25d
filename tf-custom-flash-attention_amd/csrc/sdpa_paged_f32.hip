// sdpa_paged_f32.hip -- attention of chunks of new tokens over a paged cache, fp32,
// for gfx950: tiles of 128 rows, the products on the bf16 matrix cores
// (sdpa_bf3.h), as in the dense fp32 forward (sdpa_f32_fwd.hip).
//
// Four groups of 32 rows, their parts in registers; NWK waves share each group's
// keys, 32 of a block's each.  K/V blocks pass through registers into LDS, where
// they arrive as three bf16 parts that all groups use:
//   S^T = K Q^T, online softmax, O^T += V^T P^T  (P cut in registers).
// A wave's loads move whole rows of one 16-row group, which lies in one page; the
// descriptor of a group ends at the tile's last key.
//
// An infinity among the operands leaves NaN in the sums; those rows are done again
// by themselves (sdpa_paged_device.h).
//
// What bounds it: VALU work beside the MFMAs, as in the dense forward.  2048 tokens
// over 4096, 16 heads on 4, D 128: 425 us, 121 TFLOP/s; 512 over 8192, D 64: 102 us,
// 163 TFLOP/s (32-row tiles on v_mfma_f32_32x32x2_f32, as for generation: 647 and 175).
#include "sdpa_bf3.h"
#include "sdpa_launch.h"
#include "sdpa_paged_device.h"
#include "sdpa_parts.h"

namespace sdpa {
namespace {

constexpr float kTauP32 = 8.0f;  // lazy-rescale threshold (log2 units)

template <int DQK, int DV>
struct PagedF32Cfg {
    static constexpr int LK = lds_chunks(DQK), LV = lds_chunks(DV);
    static constexpr int NWK = LK == 16 && LV == 16 ? 1 : 2, NT = 256 * NWK, BM = kPagedBM, BN = 32 * NWK;
    using KT = Bf3Tile<BN, LK>;
    using VT = Bf3Tile<BN, LV>;
    static constexpr int STAGE = KT::BYTES + VT::BYTES;
    static constexpr int OS = DV + 4, MERGE = NWK > 1 ? (BM * OS + BM * 2) * 4 : 0;  // after the loop
    static constexpr size_t LDS_BYTES = 2 * STAGE > MERGE ? 2 * STAGE : MERGE;
    static_assert(LDS_BYTES <= 160 * 1024, "gfx950 LDS");
};

// A block's rows of one matrix, staged by all threads through registers.
template <int ROWS, int COLS, int NT>
struct PagedBf3Stage {
    static constexpr int CPR = COLS / 4, PER = ROWS * CPR / NT;  // 16-byte chunks of a row, of a thread
    static_assert(ROWS * CPR % NT == 0 && 16 * CPR % 64 == 0, "a wave's chunks lie in one 16-row group");
    floatx4 r[PER];
    __device__ __forceinline__ void load(const PagedRows& m, const PageWindow& pw, int kv0, int kv_end, int ncols, int tid,
                                         int wave) {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int g = (wave * 64 + u * NT) / (16 * CPR), r0 = kv0 + 16 * g;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<unsigned char*>(uniform_ptr(m.at(pw.held(r0 >> m.log2), r0))), (short)0,
                __builtin_amdgcn_readfirstlane(max(0, min(16, kv_end - r0)) * m.row_bytes), 0x00020000);
            const int c = tid + u * NT, col = c % CPR * 4;
            const uint32_t off = col < ncols ? (uint32_t)(c / CPR % 16 * m.row_bytes + 4 * col) : kOob;
            r[u] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
        }
    }
    __device__ __forceinline__ void store(unsigned char* tile, int tid) const {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int c = tid + u * NT;
            Bf3Tile<ROWS, lds_chunks(COLS)>::template store4<false>(tile, c / CPR, c % CPR * 4, r[u]);
        }
    }
};

template <int DQK, int DV>
__global__ __launch_bounds__((PagedF32Cfg<DQK, DV>::NT))
__attribute__((amdgpu_waves_per_eu(PagedF32Cfg<DQK, DV>::NWK, PagedF32Cfg<DQK, DV>::NWK)))
void paged_f32_kernel(const PagedParams p) {
    using Cfg = PagedF32Cfg<DQK, DV>;
    using KT = typename Cfg::KT;
    using VT = typename Cfg::VT;
    constexpr int BM = Cfg::BM, BN = Cfg::BN, LK = Cfg::LK, LV = Cfg::LV, NDT = DV / 32;
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wq = wave & 3, wk = wave >> 2;

    PagedItem it;
    {
        PagedPlan<BM, BN> plan(p);
        const int at = xcd_item(tile_id(), plan.items);
        if (at < 0 || !plan.find(at, it) || !slot_ok(p, it)) return;
    }
    const int D_qk = p.D_qk, D_v = p.D_v;
    const int kv_end = min(tile_keys(p, it, BM), it.s.len);
    PagedRow row;
    row.init(p, it, it.tile * BM + 32 * wq + l32);
    // keys seen by the group's first row, the fewest of its live ones, and by its last
    const bool live = it.tile * BM + 32 * wq < it.s.n * p.G;
    const int see_min = __builtin_amdgcn_readfirstlane(row.see);
    PagedRow last;
    last.init(p, it, min(it.tile * BM + 32 * wq + 31, it.s.n * p.G - 1));
    const int see_max = live ? min(__builtin_amdgcn_readfirstlane(last.see), it.s.len) : 0;

    // the factor goes into the queries: scores come out in the log2 domain
    const float sl2 = p.scale * kLog2e;
    Bf3 q[DQK / 16];
    {
        const float* qrow = static_cast<const float*>(p.q) + row.tok * p.qs.t + row.head * p.qs.h;
#pragma unroll
        for (int ks = 0; ks < DQK / 16; ++ks) {
            const int d = 16 * ks + 8 * hh;
            floatx4 x = floatx4{}, y = floatx4{};
            if (row.live && d < D_qk) x = *reinterpret_cast<const floatx4*>(qrow + d) * sl2;
            if (row.live && d + 4 < D_qk) y = *reinterpret_cast<const floatx4*>(qrow + d + 4) * sl2;
            q[ks] = cut8([&](int i) { return i < 4 ? x[i] : y[i - 4]; });
        }
    }

    const int nblk = (kv_end + BN - 1) / BN;
    const int lo = part_begin(nblk, it.part, it.s.parts), hi = part_begin(nblk, it.part + 1, it.s.parts);
    PagedRows K, V;
    K.init(p.k_cache, p.H_kv, it.h, D_qk, 4, p.batch.page_log2);
    V.init(p.v_cache, p.H_kv, it.h, D_v, 4, p.batch.page_log2);
    PageWindow pw{uniform_ptr(p.batch.page_table + it.seq * p.batch.table_stride), p.batch.pages,
                  (min(kv_end, hi * BN) + (1 << K.log2) - 1) >> K.log2};
    pw.load((lo * BN) >> K.log2, lane);
    prologue_loads_landed();

    PagedBf3Stage<BN, DQK, Cfg::NT> kst;
    PagedBf3Stage<BN, DV, Cfg::NT> vst;
    auto load_block = [&](int blk) __attribute__((always_inline)) {
        pw.need((blk * BN) >> K.log2, lane);  // (a window holds whole blocks)
        kst.load(K, pw, blk * BN, kv_end, D_qk, tid, wave);
        vst.load(V, pw, blk * BN, kv_end, D_v, tid, wave);
    };
    auto store_block = [&](int blk) __attribute__((always_inline)) {
        unsigned char* n = smem + ((blk - lo) & 1) * Cfg::STAGE;
        kst.store(n, tid);
        vst.store(n + KT::BYTES, tid);
    };
    SwzLane<LK> swK;
    SwzLane<LV> swV;
    swK.init(lane);
    swV.init(lane);
    floatx16 oacc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) oacc[dt] = floatx16{};
    float m_run = -INFINITY, l_run = 0.f;
    if (lo < hi) {
        load_block(lo);
        store_block(lo);
        if (lo + 1 < hi) load_block(lo + 1);
    }
    __syncthreads();

    // The registers hold block blk + 1; it goes to LDS, and block blk + 2 into the
    // registers, at the end of the step.
    for (int blk = lo; blk < hi; ++blk) {
        const int kv0 = blk * BN + 32 * wk;
        const uint32_t ks0 = (uint32_t)(((blk - lo) & 1) * Cfg::STAGE), vs0 = ks0 + (uint32_t)KT::BYTES;
        if (kv0 < see_max) {
            floatx16 s = floatx16{};
#pragma unroll
            for (int ks = 0; ks < DQK / 16; ++ks) s = mfma_bf3(KT::row(ks0 + swK.row, ks, 32 * wk), q[ks], s);
            if (kv0 + 32 > see_min) {
                const int left = row.see - kv0 - 4 * hh;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (8 * (r >> 2) + (r & 3) >= left) s[r] = -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int r = 1; r < 15; r += 2) mx = max3(mx, s[r], s[r + 1]);
            mx = xhalf_max(__builtin_elementwise_maximum(mx, s[15]));
            const float m_use = mx > m_run + kTauP32 ? mx : m_run;
            const float alpha = m_use == m_run ? 1.f : fast_exp2(m_run - m_use);
            if (wave_any(alpha != 1.f)) {
                l_run *= alpha;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) oacc[dt][r] *= alpha;
            }
            m_run = m_use;
            const float m0 = m_use == -INFINITY ? 0.f : m_use;
            float lsum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = fast_exp2(s[r] - m0);
                lsum += s[r];
            }
            l_run += lsum;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const Bf3 pb = cut8([&](int i) { return s[8 * j + i]; });
                Bf3 va[NDT];
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) va[dt] = VT::tr(vs0 + swV.tr0, vs0 + swV.tr1, dt, 32 * wk + 16 * j);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 6; ++i)
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt) {
                        constexpr int ia[6] = {2, 0, 1, 1, 0, 0}, ib[6] = {0, 2, 1, 0, 1, 0};
                        oacc[dt] = mfma_bf16(va[dt].p[ia[i]], pb.p[ib[i]], oacc[dt]);
                    }
            }
        }
        if (blk + 1 < hi) {
            store_block(blk + 1);
            if (blk + 2 < hi) load_block(blk + 2);
        }
        __syncthreads();
    }

    float l_tot = xhalf_sum(l_run);
    if constexpr (Cfg::NWK == 2) {
        // O, m and l of the second wave of each group through LDS
        float* mo = reinterpret_cast<float*>(smem);
        float* ml = mo + BM * Cfg::OS;
        const int r = 32 * wq + l32;
        if (wk == 1) {
            store_rows_f32<DV, true>(mo + r * Cfg::OS, oacc, 1.f, hh, DV);
            if (hh == 0) {
                ml[2 * r] = m_run;
                ml[2 * r + 1] = l_tot;
            }
        }
        __syncthreads();
        if (wk == 0) {
            const float m1 = ml[2 * r], M = fmaxf(m_run, m1), a0 = part_weight(m_run, M), a1 = part_weight(m1, M);
            l_tot = l_tot * a0 + ml[2 * r + 1] * a1;
            m_run = M;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const floatx4 x = *reinterpret_cast<const floatx4*>(mo + r * Cfg::OS + 32 * dt + 8 * g + 4 * hh);
#pragma unroll
                    for (int e = 0; e < 4; ++e) oacc[dt][4 * g + e] = oacc[dt][4 * g + e] * a0 + x[e] * a1;
                }
        }
        __syncthreads();
    }
    int* none = reinterpret_cast<int*>(smem);  // waves that met a page that is none
    if (lane == 0) none[wave] = pw.bad || it.s.bad;
    __syncthreads();
    if (wk == 1) return;
    bool bad = false;
#pragma unroll
    for (int w = 0; w < 4 * Cfg::NWK; ++w) bad = bad || none[w] != 0;
    put_paged_rows<float, DV, BM, true>(p, it, wq, row, oacc, m_run, l_tot, bad, pw.row, K, V, lo * BN, hi * BN);
}

}  // namespace

hipError_t launch_paged_f32(const PagedParams& p, hipStream_t stream) {
    return with_paged_dim(p.D_qk, [&](auto dqk) {
        return with_paged_dim(p.D_v, [&](auto dv) {
            constexpr int DQK = decltype(dqk)::value, DV = decltype(dv)::value;
            using Cfg = PagedF32Cfg<DQK, DV>;
            const PagedParams a = paged_parts(p, Cfg::BN, 1);
            const long long n = xcd_grid(paged_max_tiles(a, Cfg::BM) + (a.divide ? 1 << a.target_log2 : 0));
            hipError_t e = launch_kernel<paged_f32_kernel<DQK, DV>>(tile_grid(n, Cfg::NT), Cfg::NT, Cfg::LDS_BYTES, stream, a);
            return e == hipSuccess && a.divide ? launch_paged_merge<float, Cfg::BM, Cfg::BN>(a, stream) : e;
        });
    });
}

}  // namespace sdpa
