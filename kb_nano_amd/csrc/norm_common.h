// Device helpers of the norm kernels (norm.hip, norm_gated.hip): rows as buffer
// descriptors, eight values a lane in bf16, fp16 or fp32, and the steps of the
// 1x128 quantization of fp32 values.
#pragma once

#include "kbn_common.h"

namespace kbn {
namespace {

constexpr float kGroupEps = 1e-10f;    // absmax floor of the scale (rmsnorm_quant.cu:75)

// Two floats rounded to bf16 (nearest even) and packed, lo in the low half:
// one v_cvt_pk_bf16_f32.
__device__ __forceinline__ uint32_t pack_bf16_rne(float lo, float hi) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}

__device__ __forceinline__ float bf16_at(const u32x4& v, int j) {
    const uint32_t word = v[j >> 1];
    return (j & 1) ? bf16hi(word) : bf16lo(word);
}

// Row descriptor: `bytes` bytes from p; buffer accesses past them read zero
// or are dropped, so no access is branched around and every token issues the
// same memory instructions (which keeps the compiler's counter waits exact).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, (int)kRsrcWord3);
}

// Cache-policy operand of the row loads: non-temporal (each row is read once;
// at H = 7168, M = 4096 this is 20.5 against 22.4 us plain and 55.6 against
// 58.2 us with the residual add).
constexpr int kNtLoad = 2;

// Clamp to the e4m3 range as the reference does (fminf(fmaxf(v, -448), 448),
// rmsnorm_quant.cu:82): one v_med3_f32, which has the same IEEE minNum/maxNum
// semantics (NaN -> -448).
__device__ __forceinline__ float clamp448(float v) { return __builtin_amdgcn_fmed3f(v, -kFp8Max, kFp8Max); }

// Factor that divides by the power-of-two scale sc exactly: its reciprocal,
// or 0 for an infinite scale (a group whose absmax overflowed), so that
// v * 0 gives v / inf's +-0 for finite v and NaN (clamped to -448) for
// infinite v, as the reference's division does.
__device__ __forceinline__ float inv_scale(float sc) { return sc < __builtin_inff() ? pow2_recip(sc) : 0.f; }

constexpr int kNormBf16 = 0, kNormF16 = 1, kNormF32 = 2;   // element type codes

template <int kT>
constexpr int elt_bytes() { return kT == kNormF32 ? 4 : 2; }

// Eight elements at byte offset `off` as fp32 (reads past the range are zeros).
template <int kT>
__device__ __forceinline__ void load8(__amdgpu_buffer_rsrc_t rs, int off, float (&v)[8]) {
    if constexpr (kT == kNormF32) {
        const u32x4 lo = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, kNtLoad);
        const u32x4 hi = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 16, 0, kNtLoad);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = __uint_as_float(lo[j]);
            v[4 + j] = __uint_as_float(hi[j]);
        }
    } else {
        const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, kNtLoad);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (kT == kNormBf16) {
                v[2 * j] = bf16lo(w[j]);
                v[2 * j + 1] = bf16hi(w[j]);
            } else {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const uint32_t word = w[j];   // (a vector element is not a bit_cast operand)
                const h2 h = __builtin_bit_cast(h2, word);
                v[2 * j] = (float)h.x;
                v[2 * j + 1] = (float)h.y;
            }
        }
    }
}

// Two fp32 values rounded to the 16-bit type (nearest even), packed.
template <int kT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (kT == kNormBf16) {
        return pack_bf16_rne(lo, hi);
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, h2{(_Float16)lo, (_Float16)hi});
    }
}

// v rounded to the type (nearest even), as fp32.
template <int kT>
__device__ __forceinline__ float round_to(float v) {
    if constexpr (kT == kNormBf16) return __uint_as_float(pack_bf16_rne(v, 0.f) << 16);
    else if constexpr (kT == kNormF16) return (float)(_Float16)v;
    else return v;
}

// Eight fp32 values stored in the type at byte offset `off` (dropped past the range).
template <int kT>
__device__ __forceinline__ void store8(__amdgpu_buffer_rsrc_t rs, int off, const float (&v)[8]) {
    if constexpr (kT == kNormF32) {
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])}, rs,
            off, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])}, rs,
            off + 16, 0, 0);
    } else {
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4{pack2<kT>(v[0], v[1]), pack2<kT>(v[2], v[3]), pack2<kT>(v[4], v[5]), pack2<kT>(v[6], v[7])}, rs,
            off, 0, 0);
    }
}

}  // namespace
}  // namespace kbn
