// sdpa_paged_fp4_small.hip -- attention of few new tokens per sequence (generation, short
// drafts) over a paged cache in 4 bits (sdpa_fp4.h), queries in fp16 or fp32, for gfx950.
//
// Tiles of 16 rows (tokens times the query heads of a key head) by equal shares of the key
// blocks (sdpa_paged.h); the four waves of a workgroup take a tile's blocks of 64
// keys in turn, each with sums of its own, merged through LDS at the tile's end.
//   S^T = K Q^T, online softmax in the log2 domain, O^T += V^T P^T
// on v_mfma_f32_16x16x32_f16, without LDS in the loop: a lane of the K operand is a key, 8
// of whose features are one word of codes; a lane of the V operand is a feature, 8 keys of
// which are one word; and the keys of a block are dealt to the rows of two K operands so
// that a lane holds the scores of 8 keys in a row, which is the P operand as it stands.
// A word becomes 8 fp16 values by four conversions (v_cvt_scalef32_pk_f16_fp4) and four
// packed products with the scale, exactly.
// P enters as two fp16 parts (22 bits): the matrix cores are idle beside the conversions.
// A wave loads its next block's words as soon as this one's are used up.
// fp32 queries are cut into three parts (33 bits), after a row's largest has been brought to
// 2^14 by a power of two.
//
// Bound by memory between a start and an end that do not read: 64 sequences of 600 to 16384 tokens, 32
// heads on 8, D 128 (298 MB): 69 us and the merge 4.6, 4.3 TB/s, some 6 in the loop (over fp16 pages 217
// and 9).  11 vector instructions a matrix instruction, matrix cores busy 13 %.  4 sequences of
// 4096, 16 heads (36 MB): 13.9 and 3.9, mostly a chain: plan, page table, queries, first block, merge.
// Four workgroups a CU with blocks of 32 keys: 71 and 17 us; two blocks ahead: no change.
#include "sdpa_launch.h"
#include "sdpa_paged_fp4.h"

namespace sdpa {
namespace {

template <typename T, int DQK, int DV>
struct PagedFp4SmallCfg {
    static constexpr int NP = sizeof(T) == 2 ? 1 : 3;  // parts of a query
    static constexpr int NW = 4, NT = 64 * NW, BM = kPagedFp4SmallBM, BN = 64, PLAN = BN * NW;
    static constexpr int OS = acc_stride(DV), MERGE = NW * BM * OS * 4 + NW * BM * 8 + (BM + NW) * 4;
    static constexpr int PLAN_AT = (MERGE + 15) / 16 * 16;
    static constexpr size_t LDS_BYTES = PLAN_AT + PagedShares<BM, PLAN>::LDS_BYTES;
    static constexpr int WPE = 2;
    static_assert(WPE * LDS_BYTES <= 160 * 1024, "gfx950 LDS");
};

// A lane's words of 32 keys, as they lie in the cache.
template <int DQK, int DV>
struct Fp4Block {
    static constexpr int KW = DQK / 32;              // words of a lane's key
    static constexpr int V4 = DV / 64, V2 = DV / 32 % 2;  // pieces of 64 features, and one of 32
    static constexpr int NV = V4 + V2;
    Fp4Keys<KW> k[2];
    uint32_t v[4 * V4 + 2 * V2];
    uint2v vs[NV];

    // Of the block from key kv0 on, in page `a` or, where pages hold 16 tokens, its second half in
    // page b.  Addresses are a page's in scalar registers and a lane's offset.
    template <bool HALVES>
    __device__ __forceinline__ void load_keys(const Fp4Pages& K, int a, int b, int kv0, int lane) {
        const int m = lane & 15, kb = lane >> 4, r = 8 * (HALVES ? (m >> 2) & 1 : m >> 2) + (m & 3);
        const int slot = HALVES ? 0 : K.slot(kv0);
        fp4_ptr codes = uniform(K.page(a) + slot * (DQK / 2)), scales = codes + (K.scales_at() + slot * (KW - DQK / 2));
        if constexpr (HALVES) {
            const fp4_ptr second = uniform(K.page(b));
            codes = m >= 8 ? second : codes;
            scales = codes + K.scales_at();
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
            k[t].load(codes + Fp4Keys<KW>::codes_at(r + 4 * t, kb), scales + Fp4Keys<KW>::scale_at(r + 4 * t, kb), kb);
    }
    template <bool HALVES>
    __device__ __forceinline__ void load_values(const Fp4Pages& V, int a, int b, int kv0, int lane) {
        const int i = lane & 15, kb = lane >> 4, block = HALVES ? kb & 1 : kb, first = HALVES ? 0 : V.slot(kv0) / 8;
        fp4_ptr words = uniform(V.page(a) + first * (DV * 4)), scales = words + (V.scales_at() + first * (DV / 4 - DV * 4));
        if constexpr (HALVES) {
            const fp4_ptr second = uniform(V.page(b));
            words = kb >= 2 ? second : words;
            scales = words + V.scales_at();
        }
        const uint32_t w0 = (uint32_t)(block * DV * 4), s0 = (uint32_t)(block * (DV / 4));
#pragma unroll
        for (int c = 0; c < V4; ++c) {
            const uint4v x = fp4_load_nt<uint4v>(words + (w0 + 256 * c + 16 * i));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * c + e] = x[e];
            vs[c] = fp4_load<uint2v>(scales + (s0 + 16 * c + 8 * (i >> 3)));
        }
        if constexpr (V2) {
            const uint2v x = fp4_load_nt<uint2v>(words + (w0 + 256 * V4 + 8 * i));
            v[4 * V4] = x[0];
            v[4 * V4 + 1] = x[1];
            vs[V4] = fp4_load<uint2v>(scales + (s0 + 16 * V4));
        }
    }
};

// HALVES: pages of 16 tokens, two to a block of keys.
template <typename T, int DQK, int DV, bool HALVES>
__global__ __launch_bounds__((PagedFp4SmallCfg<T, DQK, DV>::NT))
__attribute__((amdgpu_waves_per_eu(PagedFp4SmallCfg<T, DQK, DV>::WPE, PagedFp4SmallCfg<T, DQK, DV>::WPE)))
void paged_fp4_small_kernel(const PagedParams p) {
    using Cfg = PagedFp4SmallCfg<T, DQK, DV>;
    using Block = Fp4Block<DQK, DV>;
    constexpr int BM = Cfg::BM, BN = Cfg::BN, NW = Cfg::NW, NP = Cfg::NP, KW = Block::KW, NDT = DV / 16;
    const PagedShares<BM, Cfg::PLAN> plan(p, smem + Cfg::PLAN_AT);
    const int w = (int)blockIdx.x;
    if (p.cut && threadIdx.x == 0) p.cut[w].np = 0;
    plan.each(w, [&](const PagedItem& it) __attribute__((always_inline)) {
        int tid = threadIdx.x;  // (opaque: lane terms are formed for each tile, not held across them)
        asm volatile("" : "+v"(tid));
        const int lane = tid & 63, i16 = lane & 15, kb = lane >> 4;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int kv_end = min(tile_keys(p, it, BM), it.s.len);
        PagedRow row;
        row.init(p, it, it.tile * BM + i16);
        const int see = row.live ? row.see : 0x7FFFFFFF;  // (rows that are none need no mask)

        // the queries, before it is known where the keys are
        half8 q[KW][NP];
        typedef T t8 __attribute__((ext_vector_type(8)));
        typedef T t4 __attribute__((ext_vector_type(16 / sizeof(T))));
        t8 raw[KW];
        {
            const T* qrow = static_cast<const T*>(p.q) + row.tok * p.qs.t + row.head * p.qs.h + 8 * KW * kb;
#pragma unroll
            for (int w8 = 0; w8 < KW; ++w8) {
                raw[w8] = t8{};
                if (row.live)
#pragma unroll
                    for (int e = 0; e < 8; e += 16 / (int)sizeof(T)) {
                        const t4 x = *reinterpret_cast<const t4*>(qrow + 8 * w8 + e);
#pragma unroll
                        for (int i = 0; i < 16 / (int)sizeof(T); ++i) raw[w8][e + i] = x[i];
                    }
            }
        }

        // this wave's blocks: lo + wave, lo + wave + NW, ... below hi
        const int nblk = (kv_end + BN - 1) / BN;
        const int lo = min(NW * it.u0, nblk), hi = min(NW * it.u1, nblk);
        Fp4Pages K, V;
        K.init(p.k_cache, p.H_kv, it.h, DQK, p.batch.page_log2);
        V.init(p.v_cache, p.H_kv, it.h, DV, p.batch.page_log2);
        PageWindow pw{uniform_ptr(p.batch.page_table + it.seq * p.batch.table_stride), p.batch.pages,
                      (min(kv_end, hi * BN) + (1 << K.log2) - 1) >> K.log2};
        // A block's 64 keys in two halves, whose sums do not wait for each other's.
        Block half[2];
        int page[2][2];  // of a half (HALVES: of 16 keys each)
        const auto load_keys = [&](int blk) __attribute__((always_inline)) {
            pw.need((blk * BN) >> K.log2, lane);  // (a window holds whole blocks)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int kv0 = blk * BN + 32 * h, c = kv0 >> K.log2;
                page[h][0] = pw.held(c);
                page[h][1] = HALVES ? pw.held(c + 1) : 0;
                half[h].template load_keys<HALVES>(K, page[h][0], page[h][1], kv0, lane);
            }
        };
        const auto load_values = [&](int blk) __attribute__((always_inline)) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                half[h].template load_values<HALVES>(V, page[h][0], page[h][1], blk * BN + 32 * h, lane);
        };
        pw.load((lo * BN) >> K.log2, lane);
        if (lo + wave < hi) {
            load_keys(lo + wave);
            load_values(lo + wave);
        }
        // |scale| with negated queries for scale < 0; 1e-30 for 0: the running
        // maximum is taken on raw scores, which needs a positive factor
        const float sl2_raw = p.scale * kLog2e;
        float sl2 = (sl2_raw == 0.f) ? 1e-30f : fabsf(sl2_raw);
        if constexpr (NP == 1) {
#pragma unroll
            for (int w8 = 0; w8 < KW; ++w8) q[w8][0] = sl2_raw < 0.f ? -raw[w8] : raw[w8];
        } else {
            float most = 0.f;
#pragma unroll
            for (int w8 = 0; w8 < KW; ++w8)
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf((float)raw[w8][e]));
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            float f;
            query_factor(most, sl2_raw, f, sl2);
#pragma unroll
            for (int w8 = 0; w8 < KW; ++w8) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (float)raw[w8][e] * f;
                cut_queries(q[w8], x);
            }
        }
        // a tile that goes on in the next share: what the merge has to know
        if (p.cut && tid == 0 && it.divided && it.u0 == 0) {
            const long long first = share_begin(plan.total, w + 1, plan.n, p.target_log2) - it.u1;  // of the tile's blocks
            p.cut[w] = CutTile{share_owner(plan.total, first + it.s.blocks - 1, plan.n, p.target_log2) - w + 1,
                               min(BM, it.s.n * p.G - it.tile * BM), it.tile * BM, it.s.q0, it.h, {0, 0, 0}};
        }
        floatx4 oacc[NDT];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) oacc[dt] = floatx4{};
        float m_run = -INFINITY, l_run = 0.f;

        for (int blk = lo + wave; blk < hi; blk += NW) {
            const int kv0 = blk * BN;
            const bool more = blk + NW < hi;
            floatx4 s[2][2] = {};  // [half][tile]
#pragma unroll
            for (int w8 = 0; w8 < KW; ++w8)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const half8 k = half[h].k[t].word(w8, kb);
#pragma unroll
                        for (int n = NP - 1; n >= 0; --n) s[h][t] = mfma16_f16(k, q[w8][n], s[h][t]);
                    }
            if (more) load_keys(blk + NW);
            const int key0 = kv0 + 8 * kb;  // of this lane's 8 scores of each half
            if (wave_any(kv0 + BN > see)) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (key0 + 32 * h + 4 * t + r >= see) s[h][t][r] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < 2; ++t) mx = max3(mx, max3(s[h][t][0], s[h][t][1], s[h][t][2]), s[h][t][3]);
            {
                const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
                mx = __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
                const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
                mx = __builtin_elementwise_maximum(__uint_as_float(h[0]), __uint_as_float(h[1])) * sl2;
            }
            const float m_use = (mx > m_run + kTauP) ? mx - kTopP : m_run;
            const float alpha = m_use == m_run ? 1.f : fast_exp2(m_run - m_use);
            const float nm = m_use == -INFINITY ? 0.f : -m_use;
            if (wave_any(alpha != 1.f)) {
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) oacc[dt][r] *= alpha;
            }
            m_run = m_use;
            l_run *= alpha;
            half8 part[2][2];  // [half][part]
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float pf[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) pf[j] = fast_exp2(__builtin_fmaf(s[h][j / 4][j % 4], sl2, nm));
                l_run += ((pf[0] + pf[1]) + (pf[2] + pf[3])) + ((pf[4] + pf[5]) + (pf[6] + pf[7]));
                cut_queries(part[h], pf);
            }
            if (kv0 + BN > kv_end)  // what lies behind the last key, whatever it is, is 0
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < Block::NV; ++c) half[h].vs[c] = first_bytes(half[h].vs[c], kv_end - key0 - 32 * h);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < Block::NV; ++c) {
                    half2v vs[4];
                    fp4_scales(vs, half[h].vs[c]);
#pragma unroll
                    for (int e = 0; e < (c < Block::V4 ? 4 : 2); ++e) {
                        const half8 v = fp4_word(half[h].v[4 * c + e], vs);
#pragma unroll
                        for (int n = 1; n >= 0; --n) oacc[4 * c + e] = mfma16_f16(v, part[h][n], oacc[4 * c + e]);
                    }
                }
            if (more) load_values(blk + NW);
        }

        // ---- merge the four waves.  Lane (row i16, kb): features 64 c + 16 kb + 4 r + e, of a
        // piece of 32 features 64 c + 8 kb + 2 r + e
        {
            const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
            l_run = xhalf_sum(__uint_as_float(h[0]) + __uint_as_float(h[1]));
        }
        float* lds = reinterpret_cast<float*>(smem);
        // (opaque: what is formed from it stays out of the loop, whose registers it would take)
        int end_tid = threadIdx.x;
        asm volatile("" : "+v"(end_tid));
        const int end_lane = end_tid & 63, er = end_lane & 15, ek = end_lane >> 4;
        float* mml = lds + NW * BM * Cfg::OS;
        int* again = reinterpret_cast<int*>(mml + 2 * NW * BM);
        int* none = again + BM;
        const int at = wave * BM + er;
        if (ek == 0) {
            mml[2 * at] = m_run;
            mml[2 * at + 1] = l_run;
        }
        if (end_tid < BM) again[end_tid] = 0;
        if (end_lane == 0) none[wave] = pw.bad || it.s.bad;
#pragma unroll
        for (int c = 0; c < Block::V4; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<floatx4*>(lds + at * Cfg::OS + 64 * c + 16 * ek + 4 * r) =
                    (floatx4){oacc[4 * c][r], oacc[4 * c + 1][r], oacc[4 * c + 2][r], oacc[4 * c + 3][r]};
        if constexpr (Block::V2) {
            constexpr int c = Block::V4;
#pragma unroll
            for (int r = 0; r < 4; r += 2)
                *reinterpret_cast<floatx4*>(lds + at * Cfg::OS + 64 * c + 8 * ek + 2 * r) =
                    (floatx4){oacc[4 * c][r], oacc[4 * c + 1][r], oacc[4 * c][r + 1], oacc[4 * c + 1][r + 1]};
        }
        reduce_paged_waves<T, DV, NW, BM>(p, it, lds, end_tid, [&](int r) {
            PagedRow rr;
            rr.init(p, it, it.tile * BM + r);
            const T* qr = static_cast<const T*>(p.q) + rr.tok * p.qs.t + rr.head * p.qs.h;
            put_care_row<T, BM>(p, it, rr, r, care_row_fp4<T>(p, pw.row, K, V, qr, lo * BN, min(hi * BN, min(rr.see, it.s.len))));
        });
        __syncthreads();
    });
}

// Merge of the tiles that shares cut, a workgroup a share: four columns of a row a thread, and where
// a tile has fewer of them than there are threads its parts dealt over groups of
// threads, whose sums meet in LDS.
template <typename T>
__global__ __launch_bounds__(256) void paged_fp4_merge_kernel(const PagedParams p) {
    __shared__ MergeLds lds;
    constexpr int BM = kPagedFp4SmallBM, U = 4;
    const int w = (int)blockIdx.x, tid = (int)threadIdx.x;
    const CutTile cut = p.cut[w];
    const int np = cut.np;
    if (np == 0) return;
    const int cpr = p.D_v / 4, items = cut.rows * cpr;
    const int groups = items >= 256 ? 1 : 256 / items;
    for (int i0 = 0; i0 < items; i0 += 256) {
        const int group = groups > 1 ? tid / items : 0, i = groups > 1 ? tid - group * items : i0 + tid;
        const int r = i / cpr, c = 4 * (i - r * cpr);
        const bool mine = i < items && group < groups;
        MergedRow x;
        if (mine)
            for (int k0 = group; k0 < np; k0 += U * groups) {
                floatx2 ml[U];
                floatx4 o[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const size_t row = (size_t)share_slot(w, min(k0 + u * groups, np - 1)) * BM + r;
                    ml[u] = *reinterpret_cast<const floatx2*>(p.part_ml + 2 * row);
                    o[u] = *reinterpret_cast<const floatx4*>(p.part_o + row * p.D_v + c);
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (k0 + u * groups < np) x.add(ml[u][0], ml[u][1], o[u]);
            }
        if (groups > 1) {
            lds.sum[tid] = x.acc;
            lds.ml[tid] = (floatx2){x.M, x.L};
            __syncthreads();
            if (!mine || group != 0) return;
            for (int g = 1; g < min(groups, np); ++g) x.add(lds.ml[g * items + i][0], lds.ml[g * items + i][1], lds.sum[g * items + i]);
        }
        if (!mine) continue;
        const int row = cut.row0 + r, t = (int)((unsigned)row / (unsigned)p.G);
        const int tok = cut.q0 + t, head = cut.h * p.G + (row - t * p.G);
        x.write(p, static_cast<T*>(p.o) + tok * p.os.t + head * p.os.h + c, c == 0 ? p.stats + (size_t)tok * p.H_kv * p.G + head : nullptr);
    }
}

}  // namespace

hipError_t launch_paged_fp4_small(const PagedParams& p, DType dtype, hipStream_t stream) {
    const auto run = [&](auto t) {
        using T = decltype(t);
        return with_fp4_dim(p.D_qk, [&](auto dqk) {
            return with_fp4_dim(p.D_v, [&](auto dv) {
                return with_bool(p.batch.page_log2 == 4, [&](auto halves) {
                    constexpr int DQK = decltype(dqk)::value, DV = decltype(dv)::value;
                    using Cfg = PagedFp4SmallCfg<T, DQK, DV>;
                    hipError_t e = launch_kernel<paged_fp4_small_kernel<T, DQK, DV, decltype(halves)::value>>(
                        dim3(1u << p.target_log2), Cfg::NT, Cfg::LDS_BYTES, stream, p);
                    return e == hipSuccess && paged_shares_divide(p, Cfg::PLAN)
                               ? launch_kernel<paged_fp4_merge_kernel<T>>(dim3((1u << p.target_log2) - 1), 256, 0, stream, p)
                               : e;
                });
            });
        });
    };
    return dtype == DType::F16 ? run(half_t{}) : run(float{});
}

}  // namespace sdpa
