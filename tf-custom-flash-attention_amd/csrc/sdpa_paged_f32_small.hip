// sdpa_paged_f32_small.hip -- attention of few new tokens per sequence over a paged
// cache, fp32, for gfx950, on v_mfma_f32_32x32x2_f32.
//
// Tiles, shares and waves as in sdpa_paged_f16_small.hip.  The operands go from
// the cache straight into registers, without LDS.  A lane of the K operand is
// one key's row, of which it loads whole 16-byte chunks (the order of the
// features in the sum is free; Q is held in the same); a lane of the V operand
// is a feature, whose 32 columns make a row's load a whole 128 bytes.  The P
// operand is the S accumulator as it stands: step r multiplies the keys that
// register r holds, 8 (r / 4) + 4 h + r % 4 in lane half h.
// K of the next block is loaded while P V of this one is formed, V while S is.
//
// Bound by memory and, at 128 features, the matrix instruction beside it: 32
// sequences of 4096 tokens, 16 heads on 4, D 128 (537 MB) 117 us, 4.6 TB/s.
#include "sdpa_launch.h"
#include "sdpa_paged_device.h"

namespace sdpa {
namespace {

// Cache policy of the V loads (nt).  32 sequences of 4096, D 128: 117 us, plain 127; 64 of
// 2048, D 64: 105 and 116.  K rows are read 32 bytes at a time, their lines again and again:
// with the hint 132 us there.
constexpr int kNonTemporal = 2;

template <int DQK, int DV>
struct PagedF32SmallCfg {
    static constexpr int WPE = DQK + DV > 128 ? 1 : 2;
    static constexpr int NW = 4, NT = 64 * NW, BM = kPagedSmallBM, BN = 32, PLAN = BN * NW;
    static constexpr int PLAN_AT = NW * BM * acc_stride(DV) * 4 + NW * BM * 8 + (BM + NW) * 4;
    static_assert(PLAN_AT % 16 == 0, "the plan, behind the sums");
    static constexpr size_t LDS_BYTES = PLAN_AT + PagedShares<BM, PLAN>::LDS_BYTES;
};

template <int DQK, int DV>
__global__ __launch_bounds__((PagedF32SmallCfg<DQK, DV>::NT))
__attribute__((amdgpu_waves_per_eu(PagedF32SmallCfg<DQK, DV>::WPE, PagedF32SmallCfg<DQK, DV>::WPE)))
void paged_f32_small_kernel(const PagedParams p) {
    using Cfg = PagedF32SmallCfg<DQK, DV>;
    constexpr int BM = Cfg::BM, BN = Cfg::BN, NW = Cfg::NW, NKC = DQK / 8, NDT = DV / 32;
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

        // the factor goes into the queries: scores come out in the log2 domain
        const float sl2 = p.scale * kLog2e;
        floatx4 q[NKC];
        const float* qrow = static_cast<const float*>(p.q) + row.tok * p.qs.t + row.head * p.qs.h;
#pragma unroll
        for (int c = 0; c < NKC; ++c) {
            const int d = 8 * c + 4 * hh;
            q[c] = floatx4{};
            if (row.live && d < D_qk) q[c] = *reinterpret_cast<const floatx4*>(qrow + d) * sl2;
        }

        const int nblk = (kv_end + BN - 1) / BN;
        const int lo = min(NW * it.u0, nblk), hi = min(NW * it.u1, nblk);
        PagedRows K, V;
        K.init(p.k_cache, p.H_kv, it.h, D_qk, 4, p.batch.page_log2);
        V.init(p.v_cache, p.H_kv, it.h, D_v, 4, p.batch.page_log2);
        PageWindow pw{uniform_ptr(p.batch.page_table + it.seq * p.batch.table_stride), p.batch.pages,
                      (min(kv_end, hi * BN) + (1 << K.log2) - 1) >> K.log2};
        floatx4 k[NKC];
        float v[16][NDT];
        // K rows of a block: keys past the last are read as the last (and masked)
        auto load_k = [&](int blk) {
            const int key = min(blk * BN + l32, kv_end - 1), column = key >> K.log2;
            pw.need((blk * BN) >> K.log2, lane);  // (a window holds whole blocks)
            const float* src = reinterpret_cast<const float*>(K.at(__shfl(pw.id, column - pw.first), key));
#pragma unroll
            for (int c = 0; c < NKC; ++c) {
                const int d = 8 * c + 4 * hh;
                k[c] = *reinterpret_cast<const floatx4*>(src + (d < D_qk ? d : 0));
                if (D_qk < DQK) k[c] = d < D_qk ? k[c] : floatx4{};
            }
        };
        // V rows of a block, zero past the last
        auto load_v = [&](int blk) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int r0 = blk * BN + 16 * g;
                const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                    const_cast<unsigned char*>(uniform_ptr(V.at(pw.held(r0 >> K.log2), r0))), (short)0,
                    __builtin_amdgcn_readfirstlane(max(0, min(16, kv_end - r0)) * V.row_bytes), 0x00020000);
#pragma unroll
                for (int r = 0; r < 8; ++r)
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt) {
                        const int d = 32 * dt + l32;
                        const uint32_t off = d < D_v ? (uint32_t)((8 * (r >> 2) + 4 * hh + (r & 3)) * V.row_bytes + 4 * d) : kOob;
                        v[8 * g + r][dt] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, kNonTemporal));
                    }
            }
        };
        pw.load((lo * BN) >> K.log2, lane);
        if (lo + wave < hi) load_k(lo + wave);

        floatx16 oacc[NDT];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) oacc[dt] = floatx16{};
        float m_run = -INFINITY, l_run = 0.f;
        for (int blk = lo + wave; blk < hi; blk += NW) {
            const int kv0 = blk * BN;
            load_v(blk);
            floatx16 s = floatx16{};
#pragma unroll
            for (int c = 0; c < NKC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) s = mfma_f32(k[c][e], q[c][e], s);
            if (blk + NW < hi) load_k(blk + NW);
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
            const float m_use = fmaxf(m_run, xhalf_max(mx));
            const float alpha = m_use == m_run ? 1.f : fast_exp2(m_run - m_use);
            const float m0 = m_use == -INFINITY ? 0.f : m_use;
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = fast_exp2(s[r] - m0);
                sum += s[r];
            }
            if (wave_any(alpha != 1.f)) {
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) oacc[dt][r] *= alpha;
            }
            l_run = __builtin_fmaf(l_run, alpha, sum);
            m_run = m_use;
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) oacc[dt] = mfma_f32(v[r][dt], s[r], oacc[dt]);
        }
        merge_paged_waves<float, DV, NW, BM>(p, it, reinterpret_cast<float*>(smem), oacc, m_run, xhalf_sum(l_run),
                                             pw.bad || it.s.bad, pw.row, K, V, lo * BN, hi * BN);
        __syncthreads();
    });
}

}  // namespace

hipError_t launch_paged_f32_small(const PagedParams& p, hipStream_t stream) {
    return with_paged_dim(p.D_qk, [&](auto dqk) {
        return with_paged_dim(p.D_v, [&](auto dv) {
            constexpr int DQK = decltype(dqk)::value, DV = decltype(dv)::value;
            using Cfg = PagedF32SmallCfg<DQK, DV>;
            PagedParams a = p;
            a.target_log2 = kPagedTargetLog2 - (Cfg::WPE == 1);  // one workgroup per CU, or two
            hipError_t e = launch_kernel<paged_f32_small_kernel<DQK, DV>>(dim3(1u << a.target_log2), Cfg::NT, Cfg::LDS_BYTES,
                                                                         stream, a);
            return e == hipSuccess && paged_shares_divide(a, Cfg::PLAN)
                       ? launch_paged_share_merge<float, Cfg::BM, Cfg::PLAN>(a, stream)
                       : e;
        });
    });
}

}  // namespace sdpa
