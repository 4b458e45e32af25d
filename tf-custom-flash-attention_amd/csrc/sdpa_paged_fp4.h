// sdpa_paged_fp4.h -- device side of attention over a cache in 4 bits (sdpa_fp4.h): its
// pages, single values, and queries as fp16 parts.
#pragma once

#include "sdpa_fp4.h"
#include "sdpa_paged_device.h"

namespace sdpa {
namespace {

__device__ __forceinline__ floatx4 mfma16_f16(const half8& a, const half8& b, const floatx4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <typename F>
hipError_t with_fp4_dim(int d, F&& f) {
    if (d == 96) return f(std::integral_constant<int, 96>{});
    return with_dim(d, f);
}

// An address that is the same in every lane, in scalar registers.
__device__ __forceinline__ fp4_ptr uniform(fp4_ptr p) {
    const uint64_t a = (uint64_t)p;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
    return (fp4_ptr)(((uint64_t)hi << 32) | lo);
}

// One head's bytes in the pages of a cache.
struct Fp4Pages {
    fp4_ptr base;      // of page 0
    long long stride;  // between pages
    int D, log2;
    __device__ __forceinline__ void init(const void* cache, int H_kv, int h, int D_, int page_log2) {
        D = D_;
        log2 = page_log2;
        const long long bytes = fp4_head_bytes(D, log2);
        stride = bytes * H_kv;
        base = (fp4_ptr)uniform_ptr(static_cast<const unsigned char*>(cache) + bytes * h);
    }
    __device__ __forceinline__ fp4_ptr page(int id) const { return base + id * stride; }
    __device__ __forceinline__ int slot(int key) const { return key & ((1 << log2) - 1); }
    __device__ __forceinline__ int scales_at() const { return (D / 2) << log2; }
};

__device__ __forceinline__ half8 half8_of2(half2v a, half2v b, half2v c, half2v d) {
    return (half8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The 8 values of a word, their scale in both halves of s.
__device__ __forceinline__ half8 fp4_word(uint32_t w, half2v s) {
    return half8_of2(fp4_pair<0>(w) * s, fp4_pair<1>(w) * s, fp4_pair<2>(w) * s, fp4_pair<3>(w) * s);
}
// The same with a scale of each (8 tokens of a feature).
__device__ __forceinline__ half8 fp4_word(uint32_t w, const half2v (&s)[4]) {
    return half8_of2(fp4_pair<0>(w) * s[0], fp4_pair<1>(w) * s[1], fp4_pair<2>(w) * s[2], fp4_pair<3>(w) * s[3]);
}
__device__ __forceinline__ void fp4_scales(half2v (&s)[4], uint2v x) {
    s[0] = fp4_scales2<0>(x[0]);
    s[1] = fp4_scales2<2>(x[0]);
    s[2] = fp4_scales2<0>(x[1]);
    s[3] = fp4_scales2<2>(x[1]);
}
// The first n of 8 bytes, the others 0 (n may be below 0 and above 8).
__device__ __forceinline__ uint2v first_bytes(uint2v x, int n) {
    x[0] &= n <= 0 ? 0u : (n >= 4 ? ~0u : (1u << (8 * n)) - 1u);
    x[1] &= n <= 4 ? 0u : (n >= 8 ? ~0u : (1u << (8 * (n - 4))) - 1u);
    return x;
}

// One row of queries done again with care (sdpa_paged_device.h).
template <typename T>
__device__ __forceinline__ CareRow care_row_fp4(const PagedParams& p, const int32_t* table, const Fp4Pages& K, const Fp4Pages& V,
                                             const T* q, int lo, int hi) {
    const int lane = threadIdx.x & 63;
    const bool none = (lane < p.D_qk && q[lane] != q[lane]) || (lane + 64 < p.D_qk && q[lane + 64] != q[lane + 64]);
    return care_row_of(
        p, table, K.log2, none, lo, hi,
        [&](int page, int j) {
            const fp4_ptr words = K.page(page) + (long long)K.slot(j) * (p.D_qk / 2);
            const fp4_ptr scales = K.page(page) + K.scales_at() + (long long)K.slot(j) * (p.D_qk / 32);
            float dot = 0.f;
            for (int w = 0; w < p.D_qk / 8; ++w) {
                const half8 k = fp4_word(fp4_load<uint32_t>(words + 4 * w), fp4_scale2<0>(scales[w / 4]));
#pragma unroll
                for (int e = 0; e < 8; ++e) dot = __builtin_fmaf((float)q[8 * w + e], (float)k[e], dot);
            }
            return dot;
        },
        [&](int page, int j, int d) {
            const fp4_ptr head = V.page(page);
            const int slot = V.slot(j), block = slot / 8, at = slot % 8;
            const uint32_t byte = head[((long long)block * p.D_v + d) * 4 + at / 2];
            const uint32_t scale = head[V.scales_at() + ((long long)block * (p.D_v / 32) + d / 32) * 8 + at];
            return (float)(fp4_pair<0>(at & 1 ? byte >> 4 : byte)[0] * fp4_scale2<0>(scale)[0]);
        });
}

// A lane's words of a K operand: KW = DQK / 32 neighbouring ones, those from KW part on, of a
// key's 4 KW, and their scales.
template <int KW>
struct Fp4Keys {
    uint32_t words[KW];
    uint32_t first, last;  // scales of the first and the last word
    __device__ __forceinline__ static int group(int part, int w) { return (KW * part + w) / 4; }
    // bytes from the page's (or a block's) codes and scales on: of key `slot`, from word KW part on
    __device__ __forceinline__ static uint32_t codes_at(int slot, int part) { return (uint32_t)(slot * (16 * KW) + 4 * KW * part); }
    __device__ __forceinline__ static uint32_t scale_at(int slot, int part) { return (uint32_t)(slot * KW + group(part, 0)); }
    __device__ __forceinline__ void load(fp4_ptr row, fp4_ptr scale, int part) {
        if constexpr (KW == 4) {
            const uint4v x = fp4_load_nt<uint4v>(row);
#pragma unroll
            for (int w = 0; w < 4; ++w) words[w] = x[w];
        } else if constexpr (KW == 2) {
            const uint2v x = fp4_load_nt<uint2v>(row);
            words[0] = x[0];
            words[1] = x[1];
        } else {
#pragma unroll
            for (int w = 0; w < KW; ++w) words[w] = fp4_load_nt<uint32_t>(row + 4 * w);
        }
        first = scale[0];
        if constexpr (KW == 3) last = scale[group(part, 2) - group(part, 0)];
    }
    __device__ __forceinline__ half8 word(int w, int part) const {
        uint32_t s = first;
        if constexpr (KW == 3) s = group(part, w) == group(part, 0) ? s : last;
        return fp4_word(words[w], fp4_scale2<0>(s));
    }
};

// 8 queries as N fp16 parts, the first the nearest fp16 and so on.
template <int N>
__device__ __forceinline__ void cut_queries(half8 (&part)[N], float (&x)[8]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            part[n][e] = (half_t)x[e];
            x[e] = __builtin_fmaf((float)part[n][e], -1.f, x[e]);  // (one instruction, on the half as it is)
        }
}

// The power of two that brings a row's largest |query| near 2^14 (within what a float holds; queries
// below 2^-100 lose bits), negated for a scale below 0, and the scale (log2 units) of the products of such
// queries.  That one stays a normal number, as 0 times the -inf of a masked score is NaN: the
// scores, below 2^14 128 61440 < 2^37, are 0 by 2^-126 as by what is less.  Scale 0: the queries are 0.
__device__ __forceinline__ void query_factor(float most, float sl2_raw, float& f, float& sl2) {
    const int up = min(max(14 - (int)(__float_as_uint(most) >> 23) + 127, -113), 114);
    f = __builtin_copysignf(__uint_as_float((uint32_t)(127 + up) << 23), sl2_raw);
    sl2 = fabsf(sl2_raw) * __uint_as_float((uint32_t)(127 - up) << 23);
    sl2 = sl2 < 0x1p-126f ? 0x1p-126f : sl2;  // (NaN stays)
    if (sl2_raw == 0.f) {
        f = 0.f;
        sl2 = 1.f;
    }
}

}  // namespace
}  // namespace sdpa
