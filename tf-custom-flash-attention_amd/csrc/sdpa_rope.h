// sdpa_rope.h -- one head of a query or key row: RMS norm, rotation by
// position and their gradient, by a group of lanes in registers; shared by the
// kernels of sdpa_norm_rope.hip and sdpa_kv_append.hip.
//
// A row of D features is cut into chunks of EPC (16 bytes each, or one
// feature where rows are not aligned).  Lane j of the row's LPR lanes holds
// two of them, chosen so that the two features of a rotated pair meet in one
// lane and no value crosses lanes but the sum of squares:
//   pairs (i, i + R/2): chunks j and j + R/(2 EPC) of the rotated part, and
//                       neighbouring chunks behind it;
//   pairs (2i, 2i + 1): chunks 2j and 2j + 1.
// All arithmetic is fp32; a result is rounded once, when it is stored.
#pragma once

#include <type_traits>

#include "sdpa_device.h"

namespace sdpa {

// Strides, in elements, of a [B, S, H, D] tensor whose features are dense.
struct RowStrides {
    long long b, s, h;
};

// Rotation tables [rows, R/2] and how a row is rotated and normed.
struct RopeArgs {
    const float* cos;
    const float* sin;
    int rows;  // of the tables: a position outside them makes the row NaN
    int R;     // rotated features (even; 0: none)
    int norm;  // x / sqrt(mean x^2 + eps), then the weight where there is one
    float eps, inv_D;
};

// Positions with several axes (time, height, width): pair i is turned by the row of the
// tables that the token's position on axis axis_of(i) names.
constexpr int kMaxAxes = 4;
struct AxesArgs {
    const int32_t* positions;  // axis a of a token: a * stride behind its axis 0
    long long stride;
    uint64_t lo, hi;  // bits 0 and 1 of the axis of every pair
    int used;         // bit a: some pair follows axis a (0: no axes)
};

namespace {

// Pow2-sized groups of lanes per row, for D features in chunks of epc.
__host__ __device__ inline int lanes_per_row(int D, int epc) {
    const int pairs = ((D + epc - 1) / epc + 1) / 2;
    int n = 1;
    while (n < pairs) n *= 2;
    return n;
}

// Sum over groups of LPR neighbouring lanes, in every lane.  Steps of 1, 2 and
// then mirrored halves of 8 and 16 lanes (whose quads hold equal values by
// then) are DPP moves; 16 and 32 are lane swaps.
template <int LPR>
__device__ __forceinline__ float group_sum(float x) {
    const auto dpp = [](float v, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    if constexpr (LPR >= 2) x += dpp(x, std::integral_constant<int, 0xB1>{});   // quad_perm 1,0,3,2
    if constexpr (LPR >= 4) x += dpp(x, std::integral_constant<int, 0x4E>{});   // quad_perm 2,3,0,1
    if constexpr (LPR >= 8) x += dpp(x, std::integral_constant<int, 0x141>{});  // row_half_mirror
    if constexpr (LPR >= 16) x += dpp(x, std::integral_constant<int, 0x140>{}); // row_mirror
    if constexpr (LPR >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (LPR >= 64) x = xhalf_sum(x);
    return x;
}

template <typename T, int EPC>
struct Chunk {
    typedef T vec __attribute__((ext_vector_type(EPC)));
};
template <typename T>
struct Chunk<T, 1> {
    typedef T vec;
};

template <typename T, int EPC>
using chunk_t = typename Chunk<T, EPC>::vec;

// Value i of a chunk as fp32 (an operand that the fused multiply-adds read as it is).
template <typename T, int EPC>
__device__ __forceinline__ float at(const chunk_t<T, EPC>& v, int i) {
    if constexpr (EPC == 1) return (float)v;
    else return (float)v[i];
}
template <typename T, int EPC>
__device__ __forceinline__ chunk_t<T, EPC> chunk_of(const float (&x)[EPC]) {
    chunk_t<T, EPC> v;
    if constexpr (EPC == 1) v = (T)x[0];
    else
#pragma unroll
        for (int i = 0; i < EPC; ++i) v[i] = (T)x[i];
    return v;
}
// EPC values of a table.
template <int EPC>
__device__ __forceinline__ void load_table(float (&x)[EPC], const float* p) {
    const chunk_t<float, EPC> v = *reinterpret_cast<const chunk_t<float, EPC>*>(p);
#pragma unroll
    for (int i = 0; i < EPC; ++i) x[i] = at<float, EPC>(v, i);
}

// What lane j of a row's lanes holds: features fa .. + EPC and fb .. + EPC.
// IN: pairs of neighbouring features inside a chunk (EPC > 1).
template <int EPC, bool IN>
struct RowLane {
    int fa, fb;
    bool va, vb;  // inside the row
    bool ra, rb;  // rotated (the same unless IN)
    int t;        // first column of the tables
    __device__ __forceinline__ void init(int j, int D, int R, bool interleaved) {
        const int n = D / EPC, r = R / EPC;
        int a, b;
        if (IN || interleaved) {
            a = 2 * j;
            b = 2 * j + 1;
            t = IN ? EPC * j : j;
            ra = a < r;
            rb = b < r;
        } else {
            const int half = r / 2;
            ra = rb = j < half;
            a = ra ? j : r + 2 * (j - half);
            b = ra ? j + half : a + 1;
            t = EPC * j;
        }
        va = a < n;
        vb = b < n;
        fa = va ? a * EPC : 0;
        fb = vb ? b * EPC : 0;
    }
};

// cos and sin of a lane's pairs: column i belongs to pair i of (a, b), or (IN)
// the first half to the pairs inside a and the second to those inside b.
template <int EPC>
struct RowTurn {
    float c[EPC], s[EPC];
    bool bad;  // the position lies outside the tables
    template <bool IN>
    __device__ __forceinline__ void load(const RopeArgs& p, const RowLane<EPC, IN>& l, long long pos) {
        bad = p.R > 0 && (pos < 0 || pos >= p.rows);
        const long long row = (bad ? 0 : pos) * (p.R / 2);
#pragma unroll
        for (int i = 0; i < EPC; ++i) {
            c[i] = 1.f;
            s[i] = 0.f;
        }
        if constexpr (!IN) {
            if (l.ra && p.rows > 0) {
                load_table<EPC>(c, p.cos + row + l.t);
                load_table<EPC>(s, p.sin + row + l.t);
            }
        } else {
            constexpr int HP = EPC / 2;
            float h[HP];
            if (l.ra && p.rows > 0) {
                load_table<HP>(h, p.cos + row + l.t);
#pragma unroll
                for (int i = 0; i < HP; ++i) c[i] = h[i];
                load_table<HP>(h, p.sin + row + l.t);
#pragma unroll
                for (int i = 0; i < HP; ++i) s[i] = h[i];
            }
            if (l.rb && p.rows > 0) {
                load_table<HP>(h, p.cos + row + l.t + HP);
#pragma unroll
                for (int i = 0; i < HP; ++i) c[HP + i] = h[i];
                load_table<HP>(h, p.sin + row + l.t + HP);
#pragma unroll
                for (int i = 0; i < HP; ++i) s[HP + i] = h[i];
            }
        }
    }
    // The same by axes; `pos`: the token's position on axis 0.  A lane whose pairs all follow one
    // axis reads that row of the tables, as with one position; where some lane's do not, all
    // read the rows of every axis and choose pair by pair.
    template <bool IN>
    __device__ __forceinline__ void load_axes(const RopeArgs& p, const AxesArgs& ax, const RowLane<EPC, IN>& l,
                                              const int32_t* pos) {
        // pairs of this lane: t .. t + EPC (IN: the first half in a, the second in b)
        constexpr int HP = IN ? EPC / 2 : EPC;
        constexpr uint32_t kHalf = (1u << HP) - 1;
        const uint32_t mine = (l.ra ? kHalf : 0u) | (IN && l.rb ? kHalf << HP : 0u);
        const uint32_t lo = mine ? (uint32_t)(ax.lo >> l.t) & mine : 0u, hi = mine ? (uint32_t)(ax.hi >> l.t) & mine : 0u;
        int32_t row[kMaxAxes];
        const int any = __builtin_ctz((unsigned)ax.used);
#pragma unroll
        for (int a = 0; a < kMaxAxes; ++a) row[a] = pos[((ax.used >> a) & 1 ? a : any) * ax.stride];
        bad = false;
#pragma unroll
        for (int a = 0; a < kMaxAxes; ++a) bad = bad || (uint32_t)row[a] >= (uint32_t)p.rows;
#pragma unroll
        for (int i = 0; i < EPC; ++i) {
            c[i] = 1.f;
            s[i] = 0.f;
        }
        if (p.rows == 0) return;
        const auto load = [&](int32_t r, float (&x)[EPC], float (&y)[EPC]) __attribute__((always_inline)) {
            const long long at = (long long)(bad ? 0 : r) * (p.R / 2) + l.t;
#pragma unroll
            for (int h = 0; h < EPC; h += HP)
                if ((mine >> h) & 1) {
                    float u[HP], v[HP];
                    load_table<HP>(u, p.cos + at + h);
                    load_table<HP>(v, p.sin + at + h);
#pragma unroll
                    for (int i = 0; i < HP; ++i) {
                        x[h + i] = u[i];
                        y[h + i] = v[i];
                    }
                }
        };
        const bool mixed = (lo != 0 && lo != mine) || (hi != 0 && hi != mine);
        if (!wave_any(mixed)) {
            load(lo ? (hi ? row[3] : row[1]) : (hi ? row[2] : row[0]), c, s);
            return;
        }
#pragma unroll
        for (int a = 0; a < kMaxAxes; ++a) {
            if (!((ax.used >> a) & 1)) continue;
            float x[EPC] = {}, y[EPC] = {};
            load(row[a], x, y);
            const uint32_t on = mine & (a & 1 ? lo : ~lo) & (a & 2 ? hi : ~hi);
#pragma unroll
            for (int i = 0; i < EPC; ++i)
                if ((on >> i) & 1) {
                    c[i] = x[i];
                    s[i] = y[i];
                }
        }
    }
    // The pairs of (a, b) turned back by the angle.
    template <bool IN>
    __device__ __forceinline__ void back(const RowLane<EPC, IN>& l, float (&a)[EPC], float (&b)[EPC]) const {
        const auto turn = [&](float& x, float& y, int i) {
            const float u = __builtin_fmaf(y, s[i], x * c[i]), v = __builtin_fmaf(-x, s[i], y * c[i]);
            x = u;
            y = v;
        };
        if constexpr (!IN) {
            if (l.ra)
#pragma unroll
                for (int i = 0; i < EPC; ++i) turn(a[i], b[i], i);
        } else {
            if (l.ra)
#pragma unroll
                for (int i = 0; i < EPC / 2; ++i) turn(a[2 * i], a[2 * i + 1], i);
            if (l.rb)
#pragma unroll
                for (int i = 0; i < EPC / 2; ++i) turn(b[2 * i], b[2 * i + 1], EPC / 2 + i);
        }
    }
};

// The rotation of a weighted row: for each pair (x, y) of weights (v, w)
//   x v c - y w s,  y w c + x v s,
// its four factors formed once for the rows of a token.
template <int EPC, bool IN>
struct RowFactors {
    float xx[EPC], xy[EPC], yx[EPC], yy[EPC];  // pairs of (a, b); IN: of a, then of b
    __device__ __forceinline__ void pair(int i, float v, float w, const RowTurn<EPC>& t, bool turned) {
        xx[i] = turned ? v * t.c[i] : v;
        xy[i] = w * t.s[i];
        yx[i] = v * t.s[i];
        yy[i] = turned ? w * t.c[i] : w;
    }
    __device__ __forceinline__ void init(const RowLane<EPC, IN>& l, const RowTurn<EPC>& t, const float (&wa)[EPC],
                                         const float (&wb)[EPC]) {
        if constexpr (!IN) {
#pragma unroll
            for (int i = 0; i < EPC; ++i) pair(i, wa[i], wb[i], t, l.ra);
        } else {
#pragma unroll
            for (int i = 0; i < EPC / 2; ++i) {
                pair(i, wa[2 * i], wa[2 * i + 1], t, l.ra);
                pair(EPC / 2 + i, wb[2 * i], wb[2 * i + 1], t, l.rb);
            }
        }
    }
    // (a plain feature stays clear of its neighbour's infinities.  The products are
    // fused multiply-adds, which take halves as they are.)
    template <bool TURNED>
    __device__ __forceinline__ void one(int i, float x, float y, float r, float& u, float& v) const {
        if constexpr (TURNED) {
            u = __builtin_fmaf(x, xx[i], __builtin_fmaf(-y, xy[i], 0.f)) * r;
            v = __builtin_fmaf(y, yy[i], __builtin_fmaf(x, yx[i], 0.f)) * r;
        } else {
            u = __builtin_fmaf(x, xx[i], 0.f) * r;
            v = __builtin_fmaf(y, yy[i], 0.f) * r;
        }
    }
    // a and b: the row as it lies, the result in place, times r
    template <typename T>
    __device__ __forceinline__ void apply(const RowLane<EPC, IN>& l, chunk_t<T, EPC>& a, chunk_t<T, EPC>& b, float r) const {
        float u[EPC], v[EPC];
        if constexpr (!IN) {
            const auto all = [&](auto turned) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < EPC; ++i)
                    one<decltype(turned)::value>(i, at<T, EPC>(a, i), at<T, EPC>(b, i), r, u[i], v[i]);
            };
            if (l.ra) all(std::true_type{});
            else all(std::false_type{});
        } else {
            const auto all = [&](auto turned, const chunk_t<T, EPC>& x, float (&w)[EPC], int i0) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < EPC / 2; ++i)
                    one<decltype(turned)::value>(i0 + i, at<T, EPC>(x, 2 * i), at<T, EPC>(x, 2 * i + 1), r, w[2 * i],
                                                 w[2 * i + 1]);
            };
            if (l.ra) all(std::true_type{}, a, u, 0);
            else all(std::false_type{}, a, u, 0);
            if (l.rb) all(std::true_type{}, b, v, EPC / 2);
            else all(std::false_type{}, b, v, EPC / 2);
        }
        a = chunk_of<T, EPC>(u);
        b = chunk_of<T, EPC>(v);
    }
};

// A lane's part of the norm's weight (1 without one), which is of type T or float.
template <typename T, int EPC, bool IN>
__device__ __forceinline__ void load_weight(float (&wa)[EPC], float (&wb)[EPC], const void* w, bool w32,
                                            const RowLane<EPC, IN>& l) {
    typedef chunk_t<float, EPC> F;
    F a, b;
    if (w && w32) {
        a = *reinterpret_cast<const F*>(static_cast<const float*>(w) + l.fa);
        b = *reinterpret_cast<const F*>(static_cast<const float*>(w) + l.fb);
    } else if (w) {
        const chunk_t<T, EPC> ta = *reinterpret_cast<const chunk_t<T, EPC>*>(static_cast<const T*>(w) + l.fa);
        const chunk_t<T, EPC> tb = *reinterpret_cast<const chunk_t<T, EPC>*>(static_cast<const T*>(w) + l.fb);
        if constexpr (EPC == 1) {
            a = (float)ta;
            b = (float)tb;
        } else {
            a = __builtin_convertvector(ta, F);
            b = __builtin_convertvector(tb, F);
        }
    } else {
        a = b = F(1.f);
    }
#pragma unroll
    for (int i = 0; i < EPC; ++i) {
        wa[i] = at<float, EPC>(a, i);
        wb[i] = at<float, EPC>(b, i);
    }
}

// A lane's part of a row (outside of the row, its first chunk).  NT: past the caches.
template <typename T, int EPC, bool IN, bool NT = false>
__device__ __forceinline__ void load_row(chunk_t<T, EPC>& a, chunk_t<T, EPC>& b, const T* row, const RowLane<EPC, IN>& l) {
    typedef chunk_t<T, EPC> V;
    const V *pa = reinterpret_cast<const V*>(row + l.fa), *pb = reinterpret_cast<const V*>(row + l.fb);
    a = NT ? __builtin_nontemporal_load(pa) : *pa;
    b = NT ? __builtin_nontemporal_load(pb) : *pb;
}
template <typename T, int EPC, bool IN>
__device__ __forceinline__ void store_row(T* row, const chunk_t<T, EPC>& a, const chunk_t<T, EPC>& b, bool live,
                                          const RowLane<EPC, IN>& l) {
    typedef chunk_t<T, EPC> V;
    if (live && l.va) *reinterpret_cast<V*>(row + l.fa) = a;
    if (live && l.vb) *reinterpret_cast<V*>(row + l.fb) = b;
}

// 1 / sqrt(mean x^2 + eps) of a row held by LPR lanes.
template <typename T, int LPR, int EPC, bool IN>
__device__ __forceinline__ float row_rnorm(const chunk_t<T, EPC>& a, const chunk_t<T, EPC>& b, const RowLane<EPC, IN>& l,
                                           const RopeArgs& p) {
    float qa = 0.f, qb = 0.f;
#pragma unroll
    for (int i = 0; i < EPC; ++i) {
        qa = __builtin_fmaf(at<T, EPC>(a, i), at<T, EPC>(a, i), qa);
        qb = __builtin_fmaf(at<T, EPC>(b, i), at<T, EPC>(b, i), qb);
    }
    return rsqrtf(__builtin_fmaf(group_sum<LPR>((l.va ? qa : 0.f) + (l.vb ? qb : 0.f)), p.inv_D, p.eps));
}

}  // namespace
}  // namespace sdpa
