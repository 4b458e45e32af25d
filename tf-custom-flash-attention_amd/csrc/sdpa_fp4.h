// sdpa_fp4.h -- the cache in 4 bits: where its bytes lie, and values to codes.
//
// A value is s c: c one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (e2m1, 4 bits), s a scale
// that 32 neighbouring features of a token and head share (e5m2, the upper byte of an
// fp16).  Products of 2 and 3 significant bits: exact in fp16, and in bf16.
//   s = max |x| / 6, rounded to nearest even and at most 10240 (6 s <= 61440);
//   c = x / s, rounded to nearest even, at most 6 in size.
// Of normal values a 32nd of whose groups' range is rounded so, the error is 0.103 of
// their deviation (with powers of two as scales 0.112, 0.126 without a value cut off).
// A group that holds an infinity or a NaN is NaN.
//
// The bytes of a page's head:
//   K  codes [page][D / 2], the feature before in the lower half of a byte, then scales
//      [page][D / 32]: a lane of the K operand is a key, whose features it reads in whole words;
//   V  codes [page / 8][D] words, the 8 tokens of a feature from the lowest bits on, then
//      scales [page / 8][D / 32][8]: a lane of the V operand is a feature, of
//      which it needs 8 keys.  So neither passes through LDS on its way to the matrix cores.
#pragma once

#include "sdpa_device.h"

namespace sdpa {

constexpr float kFp4Most = 10240.f;  // the largest scale

// Bytes of one head of a page, and where its scales begin.
__host__ __device__ inline long long fp4_head_bytes(int D, int page_log2) { return (long long)(17 * (D / 32)) << page_log2; }
__host__ __device__ inline long long fp4_scales_at(int D, int page_log2) { return (long long)(D / 2) << page_log2; }

namespace {

// A cache's bytes in device memory: pointers that went through scalar registers are
// taken for any memory otherwise, and loads from those wait for LDS too.
typedef __attribute__((address_space(1))) const unsigned char* fp4_ptr;
template <typename V>
__device__ __forceinline__ V fp4_load(fp4_ptr p) {
    return *reinterpret_cast<__attribute__((address_space(1))) const V*>(p);
}
template <typename V>  // past the caches
__device__ __forceinline__ V fp4_load_nt(fp4_ptr p) {
    return __builtin_nontemporal_load(reinterpret_cast<__attribute__((address_space(1))) const V*>(p));
}

typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

// The scale of a group whose largest |x| has these bits.  The quotient is rounded twice,
// to fp32 and then to 3 significant bits, but as 6 times a border between two scales is a
// number of few bits, none falls onto a border that is not one.
__device__ __forceinline__ uint32_t fp4_scale(uint32_t abs_bits) {
    if (abs_bits >= 0x7F800000u) return 0x7F;
    const float q = fminf(__uint_as_float(abs_bits) / 6.f, kFp4Most);
    if (q < 0x1p-14f) return (uint32_t)__builtin_rintf(q * 0x1p16f);  // (steps of 2^-16)
    const uint32_t b = __float_as_uint(q);
    return ((b + 0xFFFFFu + ((b >> 21) & 1u)) >> 21) - ((127 - 15) << 2);
}
// A scale's value (NaN from 0x7D on).
__device__ __forceinline__ float fp4_scale_value(uint32_t byte) {
    return (float)__builtin_bit_cast(half_t, (uint16_t)(byte << 8));
}
// Both halves a scale: byte k of x as an fp16.
template <int K>
__device__ __forceinline__ half2v fp4_scale2(uint32_t x) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0u, x, 0x000C000Cu | ((uint32_t)K << 24 | (uint32_t)K << 8)));
}
// Bytes k and k + 1.
template <int K>
__device__ __forceinline__ half2v fp4_scales2(uint32_t x) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0u, x, 0x000C000Cu | ((uint32_t)(K + 1) << 24 | (uint32_t)K << 8)));
}
// Codes 2 b and 2 b + 1 of a word as fp16.
template <int B>
__device__ __forceinline__ half2v fp4_pair(uint32_t word) {
    return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.f, B));
}

// Codes of 8 values, the first in the lowest bits.  x / s by a reciprocal and one
// correction, which leaves exact quotients exact: ties go where they belong, and no other
// quotient comes onto one (the quotients of neighbours are further apart than fp32's half step).
// Zeros keep the sign of x.
__device__ __forceinline__ uint32_t fp4_codes(const float (&x)[8], float s, float r) {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = x[i] * r;
        q[i] = __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-a, s, x[i]), r, a), x[i]);
    }
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[0], q[1], 1.f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[2], q[3], 1.f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[4], q[5], 1.f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[6], q[7], 1.f, 3);
    return w;
}

// 16 of a group's features, the lane beside (l ^ 1) holding the others: their codes
// and the group's scale.
__device__ __forceinline__ uint2v fp4_half_group(const float (&x)[2][8], uint32_t& scale) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(x[i][e]) & 0x7FFFFFFFu);
    most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0xB1, 0xF, 0xF, true));  // lanes 1, 0, 3, 2
    scale = fp4_scale(most);
    const float s = fp4_scale_value(scale), r = s > 0.f ? 1.f / s : 0.f;
    return (uint2v){fp4_codes(x[0], s, r), fp4_codes(x[1], s, r)};
}

}  // namespace
}  // namespace sdpa
