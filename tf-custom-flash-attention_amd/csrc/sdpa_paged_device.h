// sdpa_paged_device.h -- what the kernels of attention over a paged cache
// share: a workgroup's place in the plan, the pages of its keys, rows done
// again with care, and the merge of divided tiles.
#pragma once

#include <algorithm>

#include "sdpa_dma.h"
#include "sdpa_launch.h"
#include "sdpa_paged.h"
#include "sdpa_scan.h"
#include "sdpa_wave.h"

namespace sdpa {
namespace {

__device__ __forceinline__ float max3(float a, float b, float c) {  // v_maximum3_f32: a NaN comes out
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// Weights of the fp16 kernels are 2^(s - m), s in log2 units.  The reference m is taken 7
// below a row's maximum, and again where the maximum has come 15 above it: weights up to
// 2^15, the largest of a row at least 2^7, so that fp16 loses those below 2^-32 of the largest
// (2^-25 with m at the maximum: 400000 keys of 2^-25.25 beside one of 1, a hundredth of
// the result, vanished).
constexpr float kTauP = 15.0f, kTopP = 7.0f;

// Padded feature widths: 32, 64, 96 and 128.  The LDS rows of 96 (80, 88) features are
// those of 128, as the swizzles want, but only three quarters of the products are formed: 3
// sequences of 2000 tokens over 6000, 16 heads on 8, D 96 321 -> 285 us; fp32, 1500 over
// 3000 649 -> 497.
template <typename F>
hipError_t with_paged_dim(int d, F&& f) {
    if (d > 64 && d <= 96) return f(std::integral_constant<int, 96>{});
    return with_dim(d, f);
}
// 16-byte chunks of fp16 (or bf16) in an LDS row of D features.
constexpr int lds_chunks(int D) { return D == 96 ? 16 : D / 8; }

// One workgroup's work, the same in every lane: a tile, or a part of its keys.
struct PagedItem {
    SeqPlan s;
    int seq, h, tile;
    bool divided;
    int slot;    // of this part in the workspace, where the tile is divided
    int part;    // (parts) of s.parts
    int u0, u1;  // (shares) blocks of the tile
};

// The plan by parts.  MERGE: its items are the divided tiles.
template <int BM, int BN, bool MERGE = false>
struct PagedPlan {
    const PagedParams& p;
    const int lane;
    int chunk = 0;
    // of sequence n0 + lane: q_starts, kv_lens; the items and slots up to it
    int q0, q1, len, end, slot;
    int items = 0;  // in all

    __device__ __forceinline__ SeqPlan seq() const {
        return seq_plan(q0, q1, len, p.batch, p.G, p.causal != 0, BM, BN, chunk);
    }
    __device__ __forceinline__ static int count(const SeqPlan& s) {
        return MERGE ? (s.parts > 1 ? s.tiles : 0) : s.tiles * s.parts;
    }
    __device__ __forceinline__ static int slots(const SeqPlan& s) { return s.parts > 1 ? s.tiles * s.parts : 0; }
    __device__ __forceinline__ void read(int n0) {
        const int s = n0 + lane;
        q0 = q1 = len = 0;
        if (s < p.batch.N) {
            q0 = p.batch.q_starts[s];
            q1 = p.batch.q_starts[s + 1];
            len = p.batch.kv_lens[s];
        }
    }
    __device__ __forceinline__ void scan(int items_before, int slots_before) {
        const SeqPlan s = seq();
        end = wave_scan(count(s) * p.H_kv) + items_before;
        slot = wave_scan(slots(s) * p.H_kv) + slots_before;
    }
    __device__ __forceinline__ PagedPlan(const PagedParams& p_) : p(p_), lane(threadIdx.x & 63) {
        read(0);
        if (p.divide) {
            long long cost = 0;
            for (int n0 = 0; n0 < p.batch.N; n0 += 64) {
                if (n0 > 0) read(n0);
                const SeqPlan s = seq();
                cost += (long long)s.tiles * s.blocks;
            }
            chunk = plan_chunk(readlane64(wave_scan(cost), 63) * p.H_kv, p.target_log2, p.min_chunk,
                               p.one_per_cu);
            if (p.batch.N > 64) read(0);
        }
        scan(0, 0);
        items = __builtin_amdgcn_readlane(end, 63);
        for (int n0 = 64; n0 < p.batch.N; n0 += 64) {
            read(n0);
            items += __builtin_amdgcn_readlane(wave_scan(count(seq()) * p.H_kv), 63);
        }
    }
    // Item `at` in the order sequence, key head, tile (last first: under the
    // causal mask it has the most keys), part.
    __device__ __forceinline__ bool find(int at, PagedItem& it) {
        int base = 0, slots_before = 0;
        for (int n0 = 0; n0 < p.batch.N; n0 += 64) {
            if (p.batch.N > 64) {
                read(n0);
                scan(base, slots_before);
            }
            const uint64_t over = __builtin_amdgcn_ballot_w64(end > at);
            if (over != 0) {
                const int l = __builtin_ctzll(over);
                const auto get = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
                const SeqPlan s = seq();
                it.s = SeqPlan{get(s.q0), get(s.n), get(s.len), get(s.tiles), get(s.blocks), get(s.parts), get(s.bad) != 0};
                it.seq = n0 + l;
                int i = at - (get(end) - count(it.s) * p.H_kv);
                const int per_tile = MERGE ? 1 : it.s.parts, per_head = it.s.tiles * per_tile;
                it.h = i / per_head;
                i -= it.h * per_head;
                const int t = i / per_tile;
                it.tile = it.s.tiles - 1 - t;
                it.part = i - t * per_tile;
                it.slot = get(slot) - slots(it.s) * p.H_kv + (it.h * it.s.tiles + it.tile) * it.s.parts + it.part;
                it.divided = it.s.parts > 1;
                return true;
            }
            base = __builtin_amdgcn_readlane(end, 63);
            slots_before = __builtin_amdgcn_readlane(slot, 63);
        }
        return false;
    }
};

// The plan by shares: the blocks of all tiles in the order sequence, key head, tile.
// Where there are up to 64 sequences their lanes' part of it is kept in LDS (each
// wave writes the same), as registers are short in the kernels' loops.
template <int BM, int BN>
struct PagedShares {
    struct Lane {
        SeqPlan s;
        long long first, last;  // blocks
    };
    static constexpr int LDS_BYTES = 64 * (int)sizeof(Lane);
    const PagedParams& p;
    Lane* const kept;
    long long total = 0;
    int n = 0;  // workgroups

    // sequences n0 + lane; base: the blocks before them
    __device__ __forceinline__ Lane form(int n0, long long base) const {
        const int lane = threadIdx.x & 63, i = n0 + lane;
        int q0 = 0, q1 = 0, len = 0;
        if (i < p.batch.N) {
            q0 = p.batch.q_starts[i];
            q1 = p.batch.q_starts[i + 1];
            len = p.batch.kv_lens[i];
        }
        Lane x;
        // (all tiles of a sequence count as its last one)
        x.s = seq_plan(q0, q1, len, p.batch, p.G, false, BM, BN, 0);
        const long long mine = (long long)x.s.tiles * x.s.blocks * p.H_kv;
        x.last = wave_scan(mine) + base;
        x.first = x.last - mine;
        return x;
    }
    __device__ __forceinline__ PagedShares(const PagedParams& p_, void* lds) : p(p_), kept(static_cast<Lane*>(lds)) {
        for (int n0 = 0; n0 < p.batch.N; n0 += 64) {
            const Lane x = form(n0, total);
            total = readlane64(x.last, 63);
            if (p.batch.N <= 64) kept[threadIdx.x & 63] = x;
        }
        n = (int)(total < (1LL << p.target_log2) ? total : 1LL << p.target_log2);
    }
    // The tile that holds block `at` < total, and its first block.
    __device__ __forceinline__ long long tile(long long at, PagedItem& it) const {
        long long base = 0;
        for (int n0 = 0; n0 < p.batch.N; n0 += 64) {
            const Lane x = p.batch.N <= 64 ? kept[threadIdx.x & 63] : form(n0, base);
            const uint64_t over = __builtin_amdgcn_ballot_w64(x.last > at);
            base = readlane64(x.last, 63);
            if (over == 0) continue;
            const int l = __builtin_ctzll(over);
            const auto get = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            it.s = SeqPlan{get(x.s.q0), get(x.s.n), get(x.s.len), get(x.s.tiles), get(x.s.blocks), 1, get(x.s.bad) != 0};
            it.seq = n0 + l;
            const long long begin = readlane64(x.first, l);
            const int t = div_small(at - begin, it.s.blocks);
            it.h = t / it.s.tiles;
            it.tile = t - it.h * it.s.tiles;
            return begin + (long long)t * it.s.blocks;
        }
        // (not reached, unless the lengths change under the call: nothing, up to the share's end)
        it.s = SeqPlan{0, 0, 0, 0, 0x7FFFFFFF, 1, false};
        it.seq = it.h = it.tile = 0;
        return at;
    }
    // work(item) for every tile, or part of one, of workgroup w's share.  Without a
    // workspace the tiles that begin in the share, whole.
    template <typename F>
    __device__ __forceinline__ void each(int w, F&& work) const {
        if (w >= n) return;
        const long long end = share_begin(total, w + 1, n, p.target_log2);
        for (long long at = share_begin(total, w, n, p.target_log2); at < end;) {
            PagedItem it;
            const long long t0 = tile(at, it), t1 = t0 + it.s.blocks;
            const ShareStep step = share_step(at, end, t0, t1, w, p.part_o != nullptr);
            it.u0 = step.u0;
            it.u1 = step.u1;
            it.divided = step.divided;
            it.slot = step.slot;
            it.part = 0;
            at = step.stop;
            if (!step.skip && it.s.n > 0) work(it);
        }
    }
};

// A divided tile's part has room in the workspace.  (It always has, but for
// q_starts that go back and forth, whose sums may pass 32 bits.)
__device__ __forceinline__ bool slot_ok(const PagedParams& p, const PagedItem& it) {
    return !it.divided || (it.slot >= 0 && it.slot + it.s.parts <= (2 << p.target_log2) + it.part);
}

// Workgroup id -> item, XCD-major: XCD x takes the items [x n / 8, (x + 1) n / 8),
// so that the tiles of a sequence's key head, which read the same pages, share an L2.
__host__ __device__ __forceinline__ int xcd_item(int id, int n) {
    const int x = id & 7, i = id >> 3;
    const int lo = (int)((long long)n * x / 8), hi = (int)((long long)n * (x + 1) / 8);
    return lo + i < hi ? lo + i : -1;
}
// Workgroups of a launch of up to n items under that map.
inline long long xcd_grid(long long n) { return (n + 7) / 8 * 8; }

// A window of 64 columns of a sequence's row of the page table, one in each lane.
// A page that is none counts as page 0 and makes the rows NaN in the end (bad).
struct PageWindow {
    const int32_t* row;
    int pages, columns;  // columns that hold keys of this workgroup
    int first = -64, id = 0;  // (nothing is held yet)
    bool bad = false;
    __device__ __forceinline__ void load(int column, int lane) {
        first = column;
        const bool in = column + lane < columns;
        id = in ? row[column + lane] : 0;
        const bool none = in && (id < 0 || id >= pages);
        bad = bad || __builtin_amdgcn_ballot_w64(none) != 0;
        if (none) id = 0;
    }
    // the window holds `column` (wave-uniform; the blocks of a wave ascend)
    __device__ __forceinline__ void need(int column, int lane) {
        if (column >= first + 64) load(column, lane);
    }
    __device__ __forceinline__ int held(int column) const { return __builtin_amdgcn_readlane(id, column - first); }
};

// One head's matrices of a cache.  rows(): a descriptor over the rows [row,
// min(row + most, end)), which share a page: `most` is 16, or more where pages are
// larger, and row a multiple of it.
struct PagedRows {
    const unsigned char* base;  // the cache, from this head's matrix of page 0 on
    long long page_bytes;
    int row_bytes, log2;
    __device__ __forceinline__ void init(const void* cache, int H_kv, int h, int D, int esize, int page_log2) {
        row_bytes = D * esize;
        log2 = page_log2;
        const long long m = (long long)row_bytes << page_log2;
        page_bytes = m * H_kv;
        base = uniform_ptr(static_cast<const unsigned char*>(cache) + m * h);
    }
    __device__ __forceinline__ const unsigned char* at(int page, int row) const {
        return base + page * page_bytes + (row & ((1 << log2) - 1)) * row_bytes;
    }
    __device__ __forceinline__ rsrc_t rows(int page, int row, int end, int most) const {
        const uint64_t a = reinterpret_cast<uint64_t>(at(page, row));
        return (rsrc_t){__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
                        __builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xFFFFu)),
                        __builtin_amdgcn_readfirstlane(max(0, min(end - row, most)) * row_bytes), 0x00020000};
    }
};

// The queries of this lane's row of a tile, and how many keys they see.
struct PagedRow {
    int tok, head;  // of the T tokens and H_q heads
    int see;        // keys [0, see)
    bool live;
    __device__ __forceinline__ void init(const PagedParams& p, const PagedItem& it, int row) {
        live = row < it.s.n * p.G;
        const int i = live ? (int)((unsigned)row / (unsigned)p.G) : 0;
        tok = it.s.q0 + i;
        head = it.h * p.G + (live ? row - i * p.G : 0);
        const int v = p.causal ? it.s.len - it.s.n + i + 1 : it.s.len;
        see = live ? (v < 0 ? 0 : v) : 0;
    }
};
// Keys that the last row of a tile sees.
__device__ __forceinline__ int tile_keys(const PagedParams& p, const PagedItem& it, int BM) {
    if (!p.causal) return it.s.len;
    const int rows = it.s.n * p.G, last = min((it.tile + 1) * BM, rows) - 1;
    return max(0, it.s.len - it.s.n + (int)((unsigned)last / (unsigned)p.G) + 1);
}

// ---- rows done again ---------------------------------------------------------
// A product of a masked weight, 0, with an infinite or NaN value is NaN, and
// tiles are multiplied whole.  A row whose sums come out NaN, though the sum of its
// weights is none, is therefore done again (fp16 chunks: sdpa_paged_f16.hip) by one wave, key by key over the keys [lo, hi) it sees: finite values
// weighted, others added as they are, so that one among the row's own keys makes
// the result infinite or NaN and one behind the mask nothing.  Lane l returns
// columns l and l + 64 of the unnormalised sums; m in log2 units.
struct CareRow {
    float m, l, o[2], extra[2];
};
// none: the query holds a NaN; dot(page, key): its product with a key; value(page, key,
// column).
template <typename D, typename V>
__device__ __forceinline__ CareRow care_row_of(const PagedParams& p, const int32_t* table, int log2, bool none, int lo, int hi,
                                            D&& dot, V&& value) {
    const int lane = threadIdx.x & 63;
    CareRow r{-INFINITY, 0.f, {0.f, 0.f}, {0.f, 0.f}};
    const float sl2 = p.scale * kLog2e;
    // (of a NaN query all that sees a key is NaN)
    if (lo < hi && __builtin_amdgcn_ballot_w64(none) != 0) {
        r.l = __builtin_nanf("");
        return r;
    }
    for (int j0 = lo; j0 < hi; j0 += 64) {
        const int j = j0 + lane;
        float s = -INFINITY;
        int page = 0;
        if (j < hi) {
            page = table[j >> log2];
            s = dot(page, j) * sl2;
        }
        float mx = s;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
        const float m = fmaxf(r.m, mx), a = m == r.m ? 1.f : fast_exp2(r.m - m);
        float w = j < hi ? (m == -INFINITY ? (s == s ? 0.f : s) : fast_exp2(s - m)) : 0.f;
        float sum = w;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
        r.l = __builtin_fmaf(r.l, a, sum);
        r.m = m;
        r.o[0] *= a;
        r.o[1] *= a;
        for (int i = 0; i < 64 && j0 + i < hi; ++i) {
            const float wi = __shfl(w, i);
            const int pg = __shfl(page, i);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int d = lane + 64 * c;
                if (d >= p.D_v) continue;
                const float x = value(pg, j0 + i, d);
                if (__builtin_fabsf(x) < INFINITY) r.o[c] = __builtin_fmaf(wi, x, r.o[c]);
                else r.extra[c] += x;
            }
        }
    }
    r.o[0] += r.extra[0];
    r.o[1] += r.extra[1];
    return r;
}
template <typename T>
__device__ __forceinline__ CareRow care_row(const PagedParams& p, const int32_t* table, const PagedRows& K, const PagedRows& V,
                                         const T* q, int lo, int hi) {
    const int lane = threadIdx.x & 63;
    const bool none = (lane < p.D_qk && q[lane] != q[lane]) || (lane + 64 < p.D_qk && q[lane + 64] != q[lane + 64]);
    return care_row_of(
        p, table, K.log2, none, lo, hi,
        [&](int page, int j) {
            typedef T chunk __attribute__((ext_vector_type(16 / sizeof(T))));
            const chunk *k = reinterpret_cast<const chunk*>(K.at(page, j)), *qc = reinterpret_cast<const chunk*>(q);
            constexpr int EPC = 16 / (int)sizeof(T);
            float dot = 0.f;
            for (int d = 0; d < p.D_qk / EPC; ++d)
#pragma unroll
                for (int e = 0; e < EPC; ++e) dot = __builtin_fmaf((float)qc[d][e], (float)k[d][e], dot);
            return dot;
        },
        [&](int page, int j, int d) { return (float)reinterpret_cast<const T*>(V.at(page, j))[d]; });
}

// One row's results of one wave, column d at a time: to o and stats, or (the
// tile is divided) to the workspace.
template <typename T, int BM>
__device__ __forceinline__ void put_care_row(const PagedParams& p, const PagedItem& it, const PagedRow& row, int in_tile,
                                             const CareRow& r) {
    const int lane = threadIdx.x & 63;
    if (it.divided) {
        const size_t at = (size_t)it.slot * BM + in_tile;
        if (lane == 0) {
            p.part_ml[2 * at] = r.m;
            p.part_ml[2 * at + 1] = r.l;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
            if (lane + 64 * c < p.D_v) p.part_o[at * p.D_v + lane + 64 * c] = r.o[c];
        return;
    }
    const float inv = r.l == 0.f ? 0.f : 1.f / r.l;
    T* o = static_cast<T*>(p.o) + row.tok * p.os.t + row.head * p.os.h;
#pragma unroll
    for (int c = 0; c < 2; ++c)
        if (lane + 64 * c < p.D_v) o[lane + 64 * c] = (T)(r.o[c] * inv);
    if (lane == 0) p.stats[(size_t)row.tok * p.H_kv * p.G + row.head] = r.m * kLn2 + logf(r.l);
}

// Whether an accumulator of this lane holds a NaN or an infinity.
template <int N>
__device__ __forceinline__ bool any_nonfinite(const floatx16 (&acc)[N]) {
    float z = 0.f;
#pragma unroll
    for (int dt = 0; dt < N; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) z = __builtin_fmaf(acc[dt][r], 0.f, z);
    return z != z;
}

// Results of a wave of 32 rows (lane l32: row; accumulator tiles over features) of a
// kernel of 128-row tiles: to o and stats, or to the workspace.  PER: features of one tile are
// PER apart (tile dt: features PER m + dt; 1: 32 dt + m).  CARE: rows whose sums
// hold a NaN or an infinity, or whose scores do, again with care: care(item's row, row in the tile).
template <typename T, int DV, int BM, bool CARE, int PER, typename F>
__device__ __forceinline__ void put_paged_rows_by(const PagedParams& p, const PagedItem& it, int wave, const PagedRow& row,
                                                  const floatx16 (&oacc)[DV / 32], float m_run, float l_tot, bool bad, F&& care) {
    const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5, in_tile = 32 * wave + l32, D_v = p.D_v;
    uint32_t again = 0;
    if constexpr (CARE) {
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(row.live && !bad && (l_tot != l_tot || any_nonfinite<DV / 32>(oacc)));
        again = (uint32_t)lanes | (uint32_t)(lanes >> 32);
    }
    if (row.live && !((again >> l32) & 1)) {
        const float m = l_tot == 0.f ? -INFINITY : m_run, l = bad ? __builtin_nanf("") : l_tot;
        const float f = it.divided ? 1.f : (l == 0.f ? 0.f : 1.f / l);
        const size_t at = (size_t)it.slot * BM + in_tile;
        if (hh == 0) {
            if (it.divided) {
                p.part_ml[2 * at] = m;
                p.part_ml[2 * at + 1] = l;
            } else {
                p.stats[(size_t)row.tok * p.H_kv * p.G + row.head] = m * kLn2 + logf(l);
            }
        }
        typedef T t4 __attribute__((ext_vector_type(4)));
        T* o = static_cast<T*>(p.o) + row.tok * p.os.t + row.head * p.os.h;
        static_assert(PER == 1 || PER == DV / 32, "the tiles' features in turn, or each its own");
#pragma unroll
        for (int dt = 0; dt < DV / 32; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                // four neighbouring features: of one tile, or of PER tiles and 4 / PER registers
                const int i = PER == 4 ? 4 * dt + g : PER == 2 ? 8 * dt + 2 * g : 4 * g;
                const int d0 = PER == 1 ? 32 * dt + 8 * g + 4 * hh : PER * (8 * (i >> 2) + 4 * hh + (i & 3));
                if (d0 >= D_v) continue;
                floatx4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = PER == 1 ? oacc[dt][i + e] : oacc[e % PER][i + e / PER];
                if (it.divided) {
                    *reinterpret_cast<floatx4*>(p.part_o + at * D_v + d0) = x;
                } else {
                    t4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = (T)(x[e] * f);
                    *reinterpret_cast<t4*>(o + d0) = v;
                }
            }
    }
    if constexpr (!CARE) return;
    for (uint32_t todo = again; todo != 0; todo &= todo - 1) {
        const int r = 32 * wave + __builtin_ctz(todo);
        PagedRow rr;
        rr.init(p, it, it.tile * BM + r);
        care(rr, r);
    }
}

// The same with the features in order, over a cache of T.  [k0, k1): this workgroup's keys.
template <typename T, int DV, int BM, bool CARE>
__device__ __forceinline__ void put_paged_rows(const PagedParams& p, const PagedItem& it, int wave, const PagedRow& row,
                                               const floatx16 (&oacc)[DV / 32], float m_run, float l_tot, bool bad,
                                               const int32_t* table, const PagedRows& K, const PagedRows& V, int k0,
                                               int k1) {
    put_paged_rows_by<T, DV, BM, CARE, 1>(p, it, wave, row, oacc, m_run, l_tot, bad, [&](const PagedRow& rr, int r) {
        const T* q = static_cast<const T*>(p.q) + rr.tok * p.qs.t + rr.head * p.qs.h;
        put_care_row<T, BM>(p, it, rr, r, care_row<T>(p, table, K, V, q, k0, min(k1, min(rr.see, it.s.len))));
    });
}

// Weight 2^(m - M) of a part (0 where both are -inf: nothing was seen).
__device__ __forceinline__ float part_weight(float m, float M) { return m == -INFINITY ? 0.f : fast_exp2(m - M); }
// acc + x w, an infinite or NaN x as it is (w may have vanished)
__device__ __forceinline__ float add_part(float acc, float x, float w) {
    return __builtin_fabsf(x) < INFINITY ? __builtin_fmaf(x, w, acc) : acc + x;
}

// The sums of NW waves' accumulators in LDS ([wave][row][acc_stride(DV)], then their statistics, flags of
// rows and of waves), in wave order: to o and stats, or to the workspace.  The
// callers have written accumulators, statistics and `none`, and cleared `again`.
// care(row in the tile): a wave does a row again.
template <typename T, int DV, int NW, int BM, typename F>
__device__ __forceinline__ void reduce_paged_waves(const PagedParams& p, const PagedItem& it, float* lds, int tid, F&& care) {
    constexpr int OS = acc_stride(DV), NT = 64 * NW, ITER = (BM * (DV / 4) + NT - 1) / NT;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    float* mml = lds + NW * BM * OS;
    int* again = reinterpret_cast<int*>(mml + 2 * NW * BM);
    int* none = again + BM;
    __syncthreads();
    bool bad = false;
#pragma unroll
    for (int w = 0; w < NW; ++w) bad = bad || none[w] != 0;
    // one thread per four columns of a row
    const int rows = min(BM, it.s.n * p.G - it.tile * BM);
    floatx4 acc[ITER];
    float M[ITER], L[ITER];
#pragma unroll
    for (int u = 0; u < ITER; ++u) {
        const int i = u * NT + tid, r = i / (DV / 4), c = 4 * (i % (DV / 4));
        M[u] = -INFINITY;
        L[u] = 0.f;
        acc[u] = floatx4{};
        if (r >= rows || c >= p.D_v) continue;
        float mw[NW];
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            mw[w] = mml[(w * BM + r) * 2];
            M[u] = fmaxf(M[u], mw[w]);
        }
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = part_weight(mw[w], M[u]);
            L[u] = __builtin_fmaf(mml[(w * BM + r) * 2 + 1], f, L[u]);
            const floatx4 x = *reinterpret_cast<const floatx4*>(lds + (w * BM + r) * OS + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[u][e] = __builtin_fmaf(x[e], f, acc[u][e]);
        }
        if (bad) {
            L[u] = __builtin_nanf("");
            acc[u] = (floatx4){L[u], L[u], L[u], L[u]};
        } else {
            bool nan = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) nan = nan || acc[u][e] != acc[u][e];
            if (nan && L[u] == L[u]) again[r] = 1;
        }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ITER; ++u) {
        const int i = u * NT + tid, r = i / (DV / 4), c = 4 * (i % (DV / 4));
        if (r >= rows || c >= p.D_v || again[r]) continue;
        if (it.divided) {
            const size_t at = (size_t)it.slot * BM + r;
            if (c == 0) {
                p.part_ml[2 * at] = M[u];
                p.part_ml[2 * at + 1] = L[u];
            }
            *reinterpret_cast<floatx4*>(p.part_o + at * p.D_v + c) = acc[u];
        } else {
            PagedRow row;
            row.init(p, it, it.tile * BM + r);
            const float inv = L[u] == 0.f ? 0.f : 1.f / L[u];
            typedef T t4 __attribute__((ext_vector_type(4)));
            t4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)(acc[u][e] * inv);
            *reinterpret_cast<t4*>(static_cast<T*>(p.o) + row.tok * p.os.t + row.head * p.os.h + c) = v;
            if (c == 0) p.stats[(size_t)row.tok * p.H_kv * p.G + row.head] = M[u] * kLn2 + logf(L[u]);
        }
    }
    for (int r = wave; r < rows; r += NW)
        if (__builtin_amdgcn_readfirstlane(again[r])) care(r);
}

// The sums of the NW waves of a workgroup, whose 32 rows and lanes are those of
// an MFMA accumulator (lane l32: row; features 32 dt + 8 g + 4 hh + e), through
// LDS in wave order: to o and stats, or to the workspace.  bad: a page of some
// wave's keys is none; the rows are NaN.  [k0, k1): this workgroup's keys.
template <typename T, int DV, int NW, int BM>
__device__ __forceinline__ void merge_paged_waves(const PagedParams& p, const PagedItem& it, float* lds,
                                                  const floatx16 (&oacc)[DV / 32], float m_run, float l_tot, bool bad,
                                                  const int32_t* table, const PagedRows& K, const PagedRows& V, int k0,
                                                  int k1) {
    constexpr int OS = acc_stride(DV);
    static_assert(BM == 32, "one accumulator tile of rows");
    // (opaque: what is formed from it below stays out of the callers' loops, whose
    // registers it would take)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    float* mml = lds + NW * BM * OS;
    int* again = reinterpret_cast<int*>(mml + 2 * NW * BM);  // rows to do again
    int* none = again + BM;                                  // waves that met a page that is none
    if (hh == 0) {
        mml[(wave * BM + l32) * 2] = m_run;
        mml[(wave * BM + l32) * 2 + 1] = l_tot;
    }
    if (tid < BM) again[tid] = 0;
    if (lane == 0) none[wave] = bad;
    acc_to_lds<DV>(lds, wave * BM + l32, oacc, hh);
    reduce_paged_waves<T, DV, NW, BM>(p, it, lds, tid, [&](int r) {
        PagedRow row;
        row.init(p, it, it.tile * BM + r);
        const T* q = static_cast<const T*>(p.q) + row.tok * p.qs.t + row.head * p.qs.h;
        put_care_row<T, BM>(p, it, row, r, care_row<T>(p, table, K, V, q, k0, min(k1, min(row.see, it.s.len))));
    });
}

// The sums of a row's parts, four columns of them, as they come:
// o = sum_i O_i 2^(m_i - M) / L, stats = M ln 2 + log L.
struct MergedRow {
    float M = -INFINITY, L = 0.f;
    floatx4 acc = floatx4{};
    __device__ __forceinline__ void add(float m, float l, const floatx4& o) {
        const float Mn = fmaxf(M, m), a = M == Mn ? 1.f : part_weight(M, Mn), b = part_weight(m, Mn);
        // (a NaN sum has no maximum to weigh it by)
        L = l == l ? __builtin_fmaf(l, b, L * a) : l;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = add_part(add_part(0.f, acc[e], a), o[e], b);
        M = Mn;
    }
    // four columns to o, the statistics (null: another thread's) to stats
    template <typename T>
    __device__ __forceinline__ void write(const PagedParams& p, T* o, float* stats) const {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        typedef T t4 __attribute__((ext_vector_type(4)));
        t4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(acc[e] * inv);
        *reinterpret_cast<t4*>(o) = v;
        if (stats) *stats = M * kLn2 + logf(L);
    }
    // columns c .. c + 3 of row r of a tile
    template <typename T, int BM>
    __device__ __forceinline__ void put(const PagedParams& p, const PagedItem& it, int r, int c) const {
        PagedRow row;
        row.init(p, it, it.tile * BM + r);
        write(p, static_cast<T*>(p.o) + row.tok * p.os.t + row.head * p.os.h + c,
              c == 0 ? p.stats + (size_t)row.tok * p.H_kv * p.G + row.head : nullptr);
    }
};

// One row of a tile by a workgroup of 256 threads: its np parts, in slots slot(k), are
// dealt over groups of D_v / 4 threads (a thread: four columns), whose sums meet in
// LDS; four parts' loads go out together.
struct MergeLds {
    floatx4 sum[256];
    floatx2 ml[256];
};
template <typename T, int BM, typename F>
__device__ __forceinline__ void merge_row(const PagedParams& p, const PagedItem& it, int r, int np, MergeLds& lds, F&& slot) {
    const int tid = threadIdx.x, cpr = p.D_v / 4, groups = 256 / cpr, group = tid / cpr, c = 4 * (tid - group * cpr);
    MergedRow x;
    constexpr int U = 4;
    if (group < groups)
        for (int k0 = group; k0 < np; k0 += U * groups) {
            floatx2 ml[U];
            floatx4 o[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t row = (size_t)slot(min(k0 + u * groups, np - 1)) * BM + r;
                ml[u] = *reinterpret_cast<const floatx2*>(p.part_ml + 2 * row);
                o[u] = *reinterpret_cast<const floatx4*>(p.part_o + row * p.D_v + c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (k0 + u * groups < np) x.add(ml[u][0], ml[u][1], o[u]);
        }
    __syncthreads();  // (the row before has been read)
    lds.sum[tid] = x.acc;
    lds.ml[tid] = (floatx2){x.M, x.L};
    __syncthreads();
    if (group != 0) return;
    for (int g = 1; g < min(groups, np); ++g) x.add(lds.ml[g * cpr + tid][0], lds.ml[g * cpr + tid][1], lds.sum[g * cpr + tid]);
    x.put<T, BM>(p, it, r, c);
}

// Merge of the tiles that parts divide.  Many tiles: a workgroup takes 32 rows of a
// tile at a time, a thread four columns of a row; 128 tiles of four parts (512 tokens over
// 16000, 32 heads, D 128, 34 MB): 11 us.  Few tiles, which have many parts: a workgroup a
// row (merge_row).  The whole call of 16 tokens, 16 heads on 4, over 30000 (4 tiles): 106
// us by 32 rows, 26 by one; 128 tokens over 16000, 32 on 8 (32 tiles): 70 and 66; 256 (64
// tiles): 95 and 107.
constexpr int kMergeRows = 32, kMergeRowTiles = 32;
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedParams p) {
    __shared__ MergeLds lds;
    PagedPlan<BM, BN, true> plan(p);
    const bool by_row = plan.items <= kMergeRowTiles;
    const int per_tile = by_row ? BM : BM / kMergeRows;
    const int units = plan.items * per_tile, cpr = p.D_v / 4;
    for (int unit = (int)blockIdx.x; unit < units; unit += (int)gridDim.x) {
        PagedItem it;
        if (!plan.find(unit / per_tile, it) || !slot_ok(p, it)) return;
        const int np = it.s.parts, row0 = unit % per_tile * (BM / per_tile);
        const int rows = min(BM / per_tile, it.s.n * p.G - it.tile * BM - row0);
        if (by_row) {
            if (rows > 0) merge_row<T, BM>(p, it, row0, np, lds, [&](int k) { return it.slot + k; });
            continue;
        }
        for (int i = threadIdx.x; i < rows * cpr; i += 256) {
            const int r = row0 + i / cpr, c = 4 * (i % cpr);
            constexpr int U = 4;
            MergedRow x;
            for (int k0 = 0; k0 < np; k0 += U) {
                floatx2 ml[U];
                floatx4 o[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const size_t at = (size_t)(it.slot + min(k0 + u, np - 1)) * BM + r;
                    ml[u] = *reinterpret_cast<const floatx2*>(p.part_ml + 2 * at);
                    o[u] = *reinterpret_cast<const floatx4*>(p.part_o + at * p.D_v + c);
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (k0 + u < np) x.add(ml[u][0], ml[u][1], o[u]);
            }
            x.put<T, BM>(p, it, r, c);
        }
    }
}

// Merge of the tiles that shares divide.  Workgroup (w, y) looks at the boundary
// before share w + 1: it merges rows y, y + gridDim.y, ... of the tile that lies
// across it, if the tile lies across none before.  64 rows of eight parts: 4.6 us, most
// of it the plan and one trip to memory.  Rows y at most (the whole call of 8 tokens, 16 heads
// on 4, D 128, for 32 sequences of 4096 and for 4 of 2000): 4 69 and 34 us, 8 63 and 25.6,
// 16 66 and 23.9, 32 75 and 28.5, as workgroups without rows form the plan too.
constexpr int kShareMergeRows = 8;
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256) void paged_share_merge_kernel(const PagedParams p) {
    __shared__ MergeLds lds;
    __shared__ typename PagedShares<BM, BN>::Lane lanes[64];
    const PagedShares<BM, BN> plan(p, lanes);
    const int w = (int)blockIdx.x;
    if (w + 1 >= plan.n) return;
    const long long at = share_begin(plan.total, w + 1, plan.n, p.target_log2);
    PagedItem it;
    const long long t0 = plan.tile(at, it);
    if (it.s.n == 0) return;
    const int np = share_merge(plan.total, at, t0, it.s.blocks, w, plan.n, p.target_log2);
    if (np == 0) return;
    const int rows = min(BM, it.s.n * p.G - it.tile * BM);
    for (int r = (int)blockIdx.y; r < rows; r += (int)gridDim.y)
        merge_row<T, BM>(p, it, r, np, lds, [&](int k) { return share_slot(w, k); });
}

template <typename T, int BM, int BN>
hipError_t launch_paged_share_merge(const PagedParams& p, hipStream_t stream) {
    return launch_kernel<paged_share_merge_kernel<T, BM, BN>>(dim3((1u << p.target_log2) - 1, (unsigned)std::min(p.most_rows, kShareMergeRows)),
                                                             256, 0, stream, p);
}

template <typename T, int BM, int BN>
hipError_t launch_paged_merge(const PagedParams& p, hipStream_t stream) {
    return launch_kernel<paged_merge_kernel<T, BM, BN>>(dim3(1024), 256, 0, stream, p);
}

// The arguments of a launch by parts, for so many workgroups a CU: nothing is divided
// for want of a workspace, or where no tile walks more than min_chunk blocks.
inline PagedParams paged_parts(const PagedParams& p, int BN, int per_cu) {
    PagedParams a = p;
    a.min_chunk = kPagedMinChunk * 64 / BN;
    a.one_per_cu = per_cu > 1 ? kPagedOnePerCu : 0;
    a.target_log2 = per_cu > 1 ? kPagedTargetLog2 : kPagedTargetLog2 - 1;
    a.divide = p.part_o && ((long long)p.batch.width << p.batch.page_log2) > (long long)kPagedMinChunk * 64;
    return a;
}
// Whether a launch by shares may divide a tile.
inline bool paged_shares_divide(const PagedParams& p, int BN) {
    return p.part_o && ((long long)p.batch.width << p.batch.page_log2) > BN;
}

}  // namespace
}  // namespace sdpa
