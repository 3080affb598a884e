// MXFP4: groups of 32 values along K share one power-of-two scale, each value
// is a 4-bit e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives).  Two
// codes a byte, even k in the low nibble; one E8M0 scale byte a group (2^(byte
// - 127), 255 = NaN).  Shared by the quantizers, the product and the experts
// layer for few tokens.
//
// Scale rule: with a the group's largest magnitude rounded to one mantissa bit
// (ties up), byte = exponent(a) - 2, so a / scale lies in {4, 6}: values above
// 6 scales are below 7, where 6 is the nearest code, and no value is off by
// more than half the spacing of the codes at the top of the range.  In bits:
// adding a quarter of the mantissa range carries into the exponent exactly for
// mantissas >= 1.75.  This is a choice: the OCP microscaling document's own
// conversion takes exponent(max) - 2 without the rounding, which clips magnitudes
// of 7 to 8 scales to 6; groups whose maximum has a mantissa of 1.75 and more get
// the next scale here, and so other codes than from a producer that goes by that
// rule.  Codes and scales of either are read alike.  At least 1 (2^-126, groups of zeros and of subnormal
// numbers), at most 253.  A group that holds an infinity or a NaN has no such
// scale: byte 255 and codes of 0, so it reads back as NaN.
#pragma once

#include "kbn_common.h"

namespace kbn {

enum MxIn : int { kMxBf16 = 0, kMxF16 = 1, kMxF32 = 2 };   // the C entries' dtype codes

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kMxGroup = 32;

// Scale byte of the largest magnitude's fp32 bits.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t abits) {
    const int e = (int)((abits + 0x200000u) >> 23) - 2;
    return abits >= 0x7F800000u ? 255u : (uint32_t)(e < 1 ? 1 : e);
}

// Largest magnitude of eight values, as fp32 bits (NaN above infinity).
template <int kIn>
__device__ __forceinline__ uint32_t mx_absmax8(const uint32_t (&w)[kIn == kMxF32 ? 8 : 4]) {
    if constexpr (kIn == kMxF32) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
        return m;
    } else if constexpr (kIn == kMxBf16) {
        return absmax8_bits(w);
    } else {   // fp16 magnitudes order like their bits too; the widening is exact
        auto mag = [](uint32_t x) { return __builtin_bit_cast(u16x2, x & 0x7FFF7FFFu); };
        const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(mag(w[0]), mag(w[1])),
                                                  __builtin_elementwise_max(mag(w[2]), mag(w[3])));
        const uint16_t b = m.x > m.y ? m.x : m.y;
        return __float_as_uint((float)__builtin_bit_cast(_Float16, b));
    }
}

// The codes of eight values / 2^(byte - 127), packed (0 for byte 255).  The
// scaled conversions round to nearest even and saturate at 6; compared on the
// device with the rounding written out for every bf16 and fp16 value at
// scales over the whole range: no difference.
template <int kIn>
__device__ __forceinline__ uint32_t mx_codes8(const uint32_t (&w)[kIn == kMxF32 ? 8 : 4], uint32_t byte) {
    const float sc = __uint_as_float(byte << 23);
    uint32_t q = 0;
    if constexpr (kIn == kMxF32) {
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __uint_as_float(w[0]), __uint_as_float(w[1]), sc, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __uint_as_float(w[2]), __uint_as_float(w[3]), sc, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __uint_as_float(w[4]), __uint_as_float(w[5]), sc, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __uint_as_float(w[6]), __uint_as_float(w[7]), sc, 3);
    } else if constexpr (kIn == kMxBf16) {
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, w[0]), sc, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, w[1]), sc, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, w[2]), sc, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, w[3]), sc, 3);
    } else {
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, w[0]), sc, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, w[1]), sc, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, w[2]), sc, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, w[3]), sc, 3);
    }
    return byte == 255u ? 0u : q;
}

// Eight consecutive values of a row (16-byte aligned) as packed words.
template <int kIn, bool kOnce>
__device__ __forceinline__ void mx_load8(const void* x, int64_t elem, uint32_t (&w)[kIn == kMxF32 ? 8 : 4]) {
    auto load = [](const u32x4* p) { return kOnce ? __builtin_nontemporal_load(p) : *p; };
    if constexpr (kIn == kMxF32) {
        const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const float*>(x) + elem);
        const u32x4 a = load(p), b = load(p + 1);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    } else {
        const u32x4 a = load(reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(x) + elem));
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
}

// Max over the four lanes of a quad (a group's lanes, eight values each).
__device__ __forceinline__ uint32_t quad_max_u32(uint32_t v) {
    uint32_t t = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false);  // quad_perm [1,0,3,2]
    v = v > t ? v : t;
    t = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false);           // quad_perm [2,3,0,1]
    return v > t ? v : t;
}

}  // namespace kbn
