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
    float eps;
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

// EPC values of type T as fp32, and back.
template <typename T, int EPC>
__device__ __forceinline__ void load_chunk(float (&x)[EPC], const T* p) {
    const auto v = *reinterpret_cast<const typename Chunk<T, EPC>::vec*>(p);
    if constexpr (EPC == 1) x[0] = (float)v;
    else
#pragma unroll
        for (int i = 0; i < EPC; ++i) x[i] = (float)v[i];
}
template <typename T, int EPC>
__device__ __forceinline__ void store_chunk(T* p, const float (&x)[EPC]) {
    typename Chunk<T, EPC>::vec v;
    if constexpr (EPC == 1) v = (T)x[0];
    else
#pragma unroll
        for (int i = 0; i < EPC; ++i) v[i] = (T)x[i];
    *reinterpret_cast<typename Chunk<T, EPC>::vec*>(p) = v;
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
                load_chunk<float, EPC>(c, p.cos + row + l.t);
                load_chunk<float, EPC>(s, p.sin + row + l.t);
            }
        } else {
            constexpr int HP = EPC / 2;
            float h[HP];
            if (l.ra && p.rows > 0) {
                load_chunk<float, HP>(h, p.cos + row + l.t);
#pragma unroll
                for (int i = 0; i < HP; ++i) c[i] = h[i];
                load_chunk<float, HP>(h, p.sin + row + l.t);
#pragma unroll
                for (int i = 0; i < HP; ++i) s[i] = h[i];
            }
            if (l.rb && p.rows > 0) {
                load_chunk<float, HP>(h, p.cos + row + l.t + HP);
#pragma unroll
                for (int i = 0; i < HP; ++i) c[HP + i] = h[i];
                load_chunk<float, HP>(h, p.sin + row + l.t + HP);
#pragma unroll
                for (int i = 0; i < HP; ++i) s[HP + i] = h[i];
            }
        }
    }
    // (x, y) turned by the angle, INV: back
    template <bool INV>
    __device__ __forceinline__ void turn(float& x, float& y, int i) const {
        const float sn = INV ? -s[i] : s[i];
        const float u = x * c[i] - y * sn, v = y * c[i] + x * sn;
        x = u;
        y = v;
    }
    template <bool IN, bool INV>
    __device__ __forceinline__ void apply(const RowLane<EPC, IN>& l, float (&a)[EPC], float (&b)[EPC]) const {
        if constexpr (!IN) {
            if (l.ra)
#pragma unroll
                for (int i = 0; i < EPC; ++i) turn<INV>(a[i], b[i], i);
        } else {
            if (l.ra)
#pragma unroll
                for (int i = 0; i < EPC / 2; ++i) turn<INV>(a[2 * i], a[2 * i + 1], i);
            if (l.rb)
#pragma unroll
                for (int i = 0; i < EPC / 2; ++i) turn<INV>(b[2 * i], b[2 * i + 1], EPC / 2 + i);
        }
    }
};

// A lane's part of the norm's weight (1 without one), which is of type T or float.
template <typename T, int EPC, bool IN>
__device__ __forceinline__ void load_weight(float (&wa)[EPC], float (&wb)[EPC], const void* w, bool w32,
                                            const RowLane<EPC, IN>& l) {
#pragma unroll
    for (int i = 0; i < EPC; ++i) {
        wa[i] = wb[i] = 1.f;
        if (!w) continue;
        if (w32) {
            wa[i] = static_cast<const float*>(w)[l.fa + i];
            wb[i] = static_cast<const float*>(w)[l.fb + i];
        } else {
            wa[i] = (float)static_cast<const T*>(w)[l.fa + i];
            wb[i] = (float)static_cast<const T*>(w)[l.fb + i];
        }
    }
}

// A lane's part of a row (0 outside of it).
template <typename T, int EPC, bool IN>
__device__ __forceinline__ void load_row(float (&a)[EPC], float (&b)[EPC], const T* row, bool live,
                                         const RowLane<EPC, IN>& l) {
#pragma unroll
    for (int i = 0; i < EPC; ++i) a[i] = b[i] = 0.f;
    if (live && l.va) load_chunk<T, EPC>(a, row + l.fa);
    if (live && l.vb) load_chunk<T, EPC>(b, row + l.fb);
}
template <typename T, int EPC, bool IN>
__device__ __forceinline__ void store_row(T* row, const float (&a)[EPC], const float (&b)[EPC], bool live,
                                          const RowLane<EPC, IN>& l) {
    if (live && l.va) store_chunk<T, EPC>(row + l.fa, a);
    if (live && l.vb) store_chunk<T, EPC>(row + l.fb, b);
}

// 1 / sqrt(mean x^2 + eps) of a row held by LPR lanes.
template <int LPR, int EPC>
__device__ __forceinline__ float row_rnorm(const float (&a)[EPC], const float (&b)[EPC], int D, float eps) {
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < EPC; ++i) q += a[i] * a[i] + b[i] * b[i];
    return rsqrtf(group_sum<LPR>(q) / (float)D + eps);
}

}  // namespace
}  // namespace sdpa
