// MXFP4 quantization and back, and the C entries of the format: these two, the
// product (mxfp4_gemm.hip) and the linear that chains them.
#include "mxfp4_gemm.h"

#include <algorithm>

namespace kbn {

typedef float v4f __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ quant ---

constexpr int kQuantThreads = 256;

// A lane takes eight values of kRows rows, four lanes a group.  Memory bound.
// Many values (9 Mi and more) are read as ones that are not needed again (kOnce),
// which leaves the caches to the codes and to what was written last, and 16-bit
// rows four at a time, for more loads in flight.  us, without / with: 8192 x 18432
// bf16 66.1 / 59.7, which is 6.4 TB/s, 4096 x 7168 16.7 / 13.9, 512 x 18432 6.5 / 6.2,
// but 1024 x 7168 4.8 / 5.6; 8192 x 8192 fp32 and back 134.7 / 104.9 (alone 53.0 /
// 54.3; four rows 55.7).
template <int kIn, int kRows, bool kOnce>
__global__ __launch_bounds__(kQuantThreads) void mxfp4_quant_kernel(const void* x, int64_t ld_x, int64_t M, int64_t K,
                                                                   uint8_t* codes, int64_t ld_c, uint8_t* scales,
                                                                   int64_t ld_s) {
    const int64_t k = ((int64_t)blockIdx.x * kQuantThreads + threadIdx.x) * 8;
    if (k >= K) return;   // whole groups: K is a multiple of 32
    for (int64_t m0 = (int64_t)blockIdx.y * kRows; m0 < M; m0 += (int64_t)gridDim.y * kRows) {
        uint32_t w[kRows][kIn == kMxF32 ? 8 : 4];
#pragma unroll
        for (int r = 0; r < kRows; ++r) mx_load8<kIn, kOnce>(x, (m0 + r < M ? m0 + r : M - 1) * ld_x + k, w[r]);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int64_t m = m0 + r;
            if (m >= M) break;
            const uint32_t byte = mx_scale_byte(quad_max_u32(mx_absmax8<kIn>(w[r])));
            *reinterpret_cast<uint32_t*>(codes + m * ld_c + k / 2) = mx_codes8<kIn>(w[r], byte);
            if ((threadIdx.x & 3) == 0) scales[m * ld_s + k / kMxGroup] = (uint8_t)byte;
        }
    }
}

// Memory bound: 4096 x 18432 to bf16 28.5 us, 6.7 TB/s; 8192 x 8192 to fp32 47
// us, 6.5 TB/s.
template <int kOut>
__global__ __launch_bounds__(kQuantThreads) void mxfp4_dequant_kernel(const uint8_t* codes, int64_t ld_c,
                                                                     const uint8_t* scales, int64_t ld_s, int64_t M,
                                                                     int64_t K, void* out, int64_t ld_o) {
    const int64_t k = ((int64_t)blockIdx.x * kQuantThreads + threadIdx.x) * 8;
    if (k >= K) return;
    for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
        const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + m * ld_c + k / 2);
        const uint32_t byte = scales[m * ld_s + k / kMxGroup];
        // byte 0 stands for 2^-127: the conversion reads the exponent field
        // alone, and 0 there means just that; 255 gives NaN
        const float sc = __uint_as_float(byte << 23);
        if constexpr (kOut == kMxF32) {
            const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, sc, 1),
                        c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, sc, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, sc, 3);
            v4f* p = reinterpret_cast<v4f*>(static_cast<float*>(out) + m * ld_o + k);
            p[0] = v4f{a.x, a.y, b.x, b.y};
            p[1] = v4f{c.x, c.y, d.x, d.y};
        } else {
            u32x4 o;
            if constexpr (kOut == kMxBf16) {
                o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, sc, 0));
                o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, sc, 1));
                o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, sc, 2));
                o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, sc, 3));
            } else {
                o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, sc, 0));
                o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, sc, 1));
                o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, sc, 2));
                o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, sc, 3));
            }
            *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(out) + m * ld_o + k) = o;
        }
    }
}

static dim3 quant_grid(int64_t M, int64_t K, int rows = 1) {
    return dim3((unsigned)((K / 8 + kQuantThreads - 1) / kQuantThreads), (unsigned)std::min<int64_t>((M + rows - 1) / rows, 32768));
}

// Rows that a product reads (`near`) are at 32-bit offsets from their tile's
// first; other rows may lie any distance apart.
static int check_rows(const char* what, const char* name, int64_t ld, int64_t least, int64_t multiple, const void* ptr,
                      int64_t align, bool near = false) {
    KBN_CHECK_ARG(ld >= least && ld % multiple == 0, "%s: %s row stride %lld must be a multiple of %lld and at least %lld", what,
                  name, (long long)ld, (long long)multiple, (long long)least);
    KBN_CHECK_ARG(!near || ld < (1LL << 31) / 256, "%s: %s row stride %lld is too large", what, name, (long long)ld);
    KBN_CHECK_ARG(ptr && reinterpret_cast<uintptr_t>(ptr) % align == 0, "%s: %s must be %lld-byte aligned", what, name,
                  (long long)align);
    return 0;
}

static int quant_args(const char* what, int dtype, int64_t M, int64_t K) {
    KBN_CHECK_ARG(dtype >= 0 && dtype <= 2, "%s: unknown dtype code %d", what, dtype);
    KBN_CHECK_ARG(M >= 0 && K >= 0 && M < (1LL << 31) && K < (1LL << 31), "%s: bad size M=%lld K=%lld", what, (long long)M,
                  (long long)K);
    KBN_CHECK_ARG(K % kMxGroup == 0, "%s: K=%lld must be a multiple of %d", what, (long long)K, kMxGroup);
    return 0;
}

static int quant_launch(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ld_x, void* codes, int64_t ld_c,
                        void* scales, int64_t ld_s, hipStream_t st) {
    const bool many = M * K >= 9 << 20;
    auto* const kernel = x_dtype == kMxF32    ? many ? mxfp4_quant_kernel<kMxF32, 1, true> : mxfp4_quant_kernel<kMxF32, 1, false>
                         : x_dtype == kMxBf16 ? many ? mxfp4_quant_kernel<kMxBf16, 4, true> : mxfp4_quant_kernel<kMxBf16, 1, false>
                         : many               ? mxfp4_quant_kernel<kMxF16, 4, true> : mxfp4_quant_kernel<kMxF16, 1, false>;
    kernel<<<quant_grid(M, K, many && x_dtype != kMxF32 ? 4 : 1), kQuantThreads, 0, st>>>(x, ld_x, M, K, (uint8_t*)codes, ld_c, (uint8_t*)scales, ld_s);
    KBN_CHECK_LAUNCH("mxfp4_quant");
    return 0;
}

static int gemm_args(const char* what, int64_t M, int64_t N, int64_t K) {
    // rows and columns are counted in 32 bits, a tile past the last ones too
    KBN_CHECK_ARG(M >= 0 && N >= 0 && K > 0 && M <= (1LL << 30) && N <= (1LL << 30) && K < (1LL << 31),
                  "%s: bad size M=%lld N=%lld K=%lld", what, (long long)M, (long long)N, (long long)K);
    KBN_CHECK_ARG(K % 128 == 0, "%s: K=%lld must be a multiple of 128", what, (long long)K);
    return 0;
}

}  // namespace kbn

using namespace kbn;

extern "C" int kbn_mxfp4_quant(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ld_x, void* codes, int64_t ld_codes,
                               void* scales, int64_t ld_scales, void* stream) {
    const char* what = "mxfp4_quant";
    if (quant_args(what, x_dtype, M, K)) return 1;
    if (M == 0 || K == 0) return 0;
    if (check_rows(what, "input", ld_x, K, 8, x, 16) || check_rows(what, "codes", ld_codes, K / 2, 4, codes, 4) ||
        check_rows(what, "scales", ld_scales, K / kMxGroup, 1, scales, 1))
        return 1;
    return quant_launch(x, x_dtype, M, K, ld_x, codes, ld_codes, scales, ld_scales, (hipStream_t)stream);
}

extern "C" int kbn_mxfp4_dequant(const void* codes, int64_t ld_codes, const void* scales, int64_t ld_scales, int64_t M, int64_t K,
                                 void* out, int out_dtype, int64_t ld_out, void* stream) {
    const char* what = "mxfp4_dequant";
    if (quant_args(what, out_dtype, M, K)) return 1;
    if (M == 0 || K == 0) return 0;
    if (check_rows(what, "codes", ld_codes, K / 2, 4, codes, 4) ||
        check_rows(what, "scales", ld_scales, K / kMxGroup, 1, scales, 1) || check_rows(what, "output", ld_out, K, 8, out, 16))
        return 1;
    auto* const kernel = out_dtype == kMxBf16 ? mxfp4_dequant_kernel<kMxBf16>
                         : out_dtype == kMxF16 ? mxfp4_dequant_kernel<kMxF16> : mxfp4_dequant_kernel<kMxF32>;
    kernel<<<quant_grid(M, K), kQuantThreads, 0, (hipStream_t)stream>>>((const uint8_t*)codes, ld_codes, (const uint8_t*)scales,
                                                                       ld_scales, M, K, out, ld_out);
    KBN_CHECK_LAUNCH(what);
    return 0;
}

extern "C" int64_t kbn_mxfp4_gemm_nt_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 128) return 0;
    return mxfp4_plan_bytes(mxfp4_plan(M, N, K), M, N);
}

extern "C" int kbn_mxfp4_gemm_nt(const void* A, int64_t lda, const void* sA, int64_t ld_sa, const void* W, int64_t ldw,
                                 const void* sW, int64_t ld_sw, void* D, int64_t ldd, int64_t M, int64_t N, int64_t K,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "mxfp4_gemm_nt";
    if (gemm_args(what, M, N, K)) return 1;
    if (M == 0 || N == 0) return 0;
    if (check_rows(what, "A", lda, K / 2, 16, A, 16, true) || check_rows(what, "A scales", ld_sa, K / kMxGroup, 4, sA, 4, true) ||
        check_rows(what, "W", ldw, K / 2, 16, W, 16, true) || check_rows(what, "W scales", ld_sw, K / kMxGroup, 4, sW, 4, true) ||
        check_rows(what, "output", ldd, N, 1, D, 2))
        return 1;
    const int64_t need = kbn_mxfp4_gemm_nt_workspace_bytes(M, N, K);
    KBN_CHECK_ARG(workspace_bytes >= need && (need == 0 || aligned16(workspace)), "%s: workspace of %lld bytes needed, got %lld",
                  what, (long long)need, (long long)workspace_bytes);
    MxGemmArgs p{(const uint8_t*)A, lda, (const uint8_t*)sA, ld_sa, (const uint8_t*)W, ldw, (const uint8_t*)sW, ld_sw,
                 (uint16_t*)D, ldd, (int)M, (int)N, (int)K};
    return mxfp4_gemm_launch(p, (float*)workspace, (hipStream_t)stream);
}

// x -> codes and scales in the workspace -> product.  Few rows of 16-bit values
// go in one launch, without those: each workgroup of the few-rows kernel
// quantizes them for itself.  us in a graph with the weights in memory, one
// launch / two: 1 x 10240 x 8192 10.3 / 12.0, 1 x 2048 x 2048 3.8 / 4.8, 1 x 36864 x 7168
// 26.4 / 25.9, 4 x 10240 x 8192 11.7 / 13.0, 4 x 2048 x 2048 4.1 / 5.3, 4 x 36864 x 7168
// 28.0 / 26.5 (an eager call saves a launch's host time as well); 8 rows 2048 x 2048
// 4.3 / 5.1, 10240 x 8192 13.2 / 13.1, 4608 x 7168 8.9 / 9.2, but 36864 x 7168 32.0 /
// 26.9: up to 8 where every CU has one workgroup.  16 rows 2048 x 2048 4.9 / 5.2, 7168 x
// 2048 5.9 / 6.1, 4096 x 4096 6.5 / 6.2, 8192 x 8192 11.7 / 10.9: there up to K = 2048.
static bool linear_fused(int64_t M, int64_t N, int64_t K, int x_dtype) {
    return x_dtype != kMxF32 && (M <= 4 || (N <= 48 * cu_count() && (M <= 8 || (M <= 16 && K <= 2048))));
}
static int64_t linear_operand_bytes(int64_t M, int64_t K) { return (M * (K / 2 + K / kMxGroup) + 255) / 256 * 256; }

extern "C" int64_t kbn_mxfp4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int x_dtype) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 128 || linear_fused(M, N, K, x_dtype)) return 0;
    return linear_operand_bytes(M, K) + kbn_mxfp4_gemm_nt_workspace_bytes(M, N, K);
}

extern "C" int kbn_mxfp4_linear(const void* x, int x_dtype, int64_t ld_x, const void* W, int64_t ldw, const void* sW,
                                int64_t ld_sw, void* D, int64_t ldd, int64_t M, int64_t N, int64_t K, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    const char* what = "mxfp4_linear";
    if (quant_args(what, x_dtype, M, K) || gemm_args(what, M, N, K)) return 1;
    if (M == 0 || N == 0) return 0;
    if (check_rows(what, "input", ld_x, K, 8, x, 16, linear_fused(M, N, K, x_dtype)) ||
        check_rows(what, "W", ldw, K / 2, 16, W, 16, true) || check_rows(what, "W scales", ld_sw, K / kMxGroup, 4, sW, 4, true) ||
        check_rows(what, "output", ldd, N, 1, D, 2))
        return 1;
    const int64_t need = kbn_mxfp4_linear_workspace_bytes(M, N, K, x_dtype);
    KBN_CHECK_ARG(workspace_bytes >= need && (need == 0 || aligned16(workspace)), "%s: workspace of %lld bytes needed, got %lld",
                  what, (long long)need, (long long)workspace_bytes);
    if (linear_fused(M, N, K, x_dtype)) {
        MxGemmArgs p{nullptr, ld_x, nullptr, 0, (const uint8_t*)W, ldw, (const uint8_t*)sW, ld_sw, (uint16_t*)D, ldd,
                     (int)M, (int)N, (int)K};
        p.X = x;
        return mxfp4_rows_launch(p, mxfp4_plan(M, N, K).rf, x_dtype, (hipStream_t)stream);
    }
    uint8_t *codes = (uint8_t*)workspace, *scales = codes + M * (K / 2), *rest = codes + linear_operand_bytes(M, K);
    if (const int rc = quant_launch(x, x_dtype, M, K, ld_x, codes, K / 2, scales, K / kMxGroup, (hipStream_t)stream)) return rc;
    MxGemmArgs p{codes, K / 2, scales, K / kMxGroup, (const uint8_t*)W, ldw, (const uint8_t*)sW, ld_sw, (uint16_t*)D, ldd,
                 (int)M, (int)N, (int)K};
    return mxfp4_gemm_launch(p, (float*)rest, (hipStream_t)stream);
}

extern "C" int kbn_debug_mxfp4_plan(int64_t M, int64_t N, int64_t K, int x_dtype, int64_t* out) {
    const char* what = "debug_mxfp4_plan";
    KBN_CHECK_ARG(out && M > 0 && N > 0 && x_dtype >= -1 && x_dtype <= 2, "%s: bad arguments", what);
    if (gemm_args(what, M, N, K)) return 1;
    const MxPlan plan = mxfp4_plan(M, N, K);
    const bool fused = x_dtype >= 0 && linear_fused(M, N, K, x_dtype);
    const int64_t v[6] = {plan.bm, plan.bn, plan.splits, plan.rf, fused ? mxfp4_value_rows(M) : 0,
                          x_dtype < 0 ? kbn_mxfp4_gemm_nt_workspace_bytes(M, N, K) : kbn_mxfp4_linear_workspace_bytes(M, N, K, x_dtype)};
    std::copy(v, v + 6, out);
    return 0;
}
