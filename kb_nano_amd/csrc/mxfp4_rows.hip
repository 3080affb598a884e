// MXFP4 product for few activation rows (M <= 64), which streams the weight.
//
// A workgroup owns 16 RF weight rows and all activation rows (CG groups of
// 16); its wavefronts split K, so nothing in the loop is shared and there is
// no barrier until their sums meet in LDS, added in wavefront order.  Each
// wavefront has a private ring of kDepth stages of 256 K.  Weight codes could be
// loaded straight into the matrix instruction's layout (lane: row l & 15,
// group l >> 4), but neighbouring lanes then read different rows, and the
// weight stream reaches 4.2 TB/s where whole 128-byte lines (eight lanes a row)
// reach 5.3 (45 MB; 5.9 and 6.6 at 235 MB): so lines go to LDS by direct loads,
// and fragments are read from there.
//
// v_mfma_scale_f32_16x16x128_f8f6f4, weight rows first: a lane's four sums are
// neighbours in one output row.
//
// Bound by what a CU takes from memory, 28 to 32 B/ns, and the start of the
// stream.  1 x 10240 x 8192 8.8 us of kernel, 5.1 TB/s, 9.6 back to back with the
// quantization in it; 1 x 36864 x 7168 23.8, 5.9; 64 x 2048 x 2048 4.3 us, of which a
// launch is 2.3.  Each workgroup also loads all activation codes, at 64 rows as
// many bytes as 64 weight rows: 64 x 8192 x 8192 13.1 us, 2.8 TB/s.
//
// kX rows of bf16 or fp16 activations (kX > 0, M <= kX) are quantized by the
// kernel itself: a lane of the second operand is one scale group of one row,
// so its 32 values, their maximum, scale and codes stay in the lane.
#include "mxfp4_gemm.h"

#include "gemm_kernel.h"

namespace kbn {

typedef float v4f __attribute__((ext_vector_type(4)));

// Four wavefronts and two stages: more of either takes more LDS, so fewer
// workgroups a CU (1 x 10240 x 8192, 64 weight rows a workgroup: 11.1 us, four
// stages 11.5, eight wavefronts 12.0).
constexpr int kRowsWaves = 4, kRowsDepth = 2;

template <int RF, int CG, int kX, int kIn, int kWaves, int kDepth>
__global__ __launch_bounds__(kWaves * 64) void mxfp4_rows_kernel(const MxGemmArgs p) {
    // a wavefront's stage: weight rows, then activation rows (codes: 128 bytes a
    // row; values: 512), and for every second stage the scale bytes of 512 K
    constexpr int kW = RF * 2048, kA = kX ? (kX + 1) / 2 * 1024 : CG * 2048, kStage = kW + kA;
    constexpr int kLoads = kStage / 1024;                       // direct loads of 1 KB
    constexpr int kScaleRows = 16 * (RF + (kX ? 0 : CG)), kScale = kScaleRows * 16, kScaleLoads = kScaleRows / 16;
    constexpr int kScaleBufs = kDepth / 2 + 1, kWave = kDepth * kStage + kScaleBufs * kScale;
    constexpr int kSums = RF * CG * 4 * 64 * 4;                 // bytes of a wavefront's sums
    static_assert(kDepth % 2 == 0);
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kWaves * (kWave > kSums ? kWave : kSums)];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * (16 * RF), units = (p.K + 255) / 256;
    const int from = units * wave / kWaves, S = units * (wave + 1) / kWaves - from;
    const int k0 = from * 256, k_len = min(p.K, k0 + S * 256) - k0;   // K of this wavefront
    const int rows_w = min(p.N - n0, 16 * RF);

    // rows past the end, and what lies behind k_len, read as zeros
    const v4i dW = make_desc(p.W + (int64_t)n0 * p.ldw + k0 / 2, (rows_w - 1) * p.ldw + k_len / 2);
    const v4i dsW = make_desc(p.sW + (int64_t)n0 * p.ld_sw + k0 / 32, (rows_w - 1) * p.ld_sw + k_len / 32);
    const v4i dA = kX ? make_desc(static_cast<const uint16_t*>(p.X) + k0, ((int64_t)(p.M - 1) * p.lda + k_len) * 2)
                      : make_desc(p.A + k0 / 2, (p.M - 1) * p.lda + k_len / 2);
    const v4i dsA = make_desc(p.sA + k0 / 32, (p.M - 1) * p.ld_sa + k_len / 32);
    const uint32_t lds = (uint32_t)(uintptr_t)smem + (uint32_t)wave * kWave;
    const uint8_t* const ring = smem + wave * kWave;
    const uint8_t* const scales = ring + kDepth * kStage;
    const uint32_t lds_scales = lds + kDepth * kStage;

    // code rows: load j brings rows 8 j .. 8 j + 7, chunk c of row q to slot c ^ swz(q)
    int voff[kLoads];
    uint32_t behind = 0;   // bit j: this lane's part of load j lies in the second half of a stage
    static_for<kLoads>([&](auto j_) {
        constexpr int j = decltype(j_)::value;
        if constexpr (kX && j >= RF * 2) {
            const int row = (j - RF * 2) * 2 + (lane >> 5);
            voff[j] = row < p.M ? row * (int)p.lda * 2 + (lane & 31) * 16 : kOob;
            behind |= (lane & 31) >= 16 ? 1u << j : 0u;
        } else {
            const int q = j * 8 + (lane >> 3), chunk = (lane & 7) ^ swz(q);
            voff[j] = (j < RF * 2 ? q * (int)p.ldw : (q - RF * 16) * (int)p.lda) + chunk * 16;
            behind |= chunk >= 4 ? 1u << j : 0u;
        }
    });
    int svoff[kScaleLoads];   // load j: 16 rows of 16 bytes, four lanes a row
#pragma unroll
    for (int j = 0; j < kScaleLoads; ++j) {
        const int q = j * 16 + (lane >> 2);
        svoff[j] = (j < RF ? q * (int)p.ld_sw : (q - RF * 16) * (int)p.ld_sa) + (lane & 3) * 4;
    }
    auto issue = [&](int buf, int s) {
        v4i w = dW, a = dA;
        if (s >= S) w[2] = a[2] = 0;
        const bool half = (s + 1) * 256 > k_len;
        const uint32_t base = lds + (uint32_t)buf * kStage;
        static_for<kLoads>([&](auto j_) {
            constexpr int j = decltype(j_)::value;
            const int v = half && (behind >> j & 1) ? kOob : voff[j];
            if constexpr (j < RF * 2) dma_b128<j * 1024, true>(w, base, v, s * 128);
            else dma_b128<j * 1024, false>(a, base, v, s * (kX ? 512 : 128));
        });
    };
    // bytes behind k_len: another row's, masked when they are read
    auto issue_scales = [&](int o) {
        v4i w = dsW, a = dsA;
        if (2 * o >= S) w[2] = a[2] = 0;
        const uint32_t base = lds_scales + (uint32_t)(o % kScaleBufs) * kScale;
        static_for<kScaleLoads>([&](auto j_) {
            constexpr int j = decltype(j_)::value;
            dma_b32<j * 256>(j < RF ? w : a, base, svoff[j], o * 16);
        });
    };

    v4f acc[RF][CG] = {};
    auto frag = [&](const uint8_t* at, int q, int j) -> v8i {   // rows q .. q + 15 of a stage, K half j
        const u32x4 v = *reinterpret_cast<const u32x4*>(at + (q + r) * 128 + (((4 * j + g) ^ swz(r)) << 4));
        return v8i{(int)v.x, (int)v.y, (int)v.z, (int)v.w};
    };
    auto use = [&](int buf, int s) {
        const uint8_t *at = ring + buf * kStage, *sc = scales + (s / 2 % kScaleBufs) * kScale + (s & 1) * 8;
        v8i w[2][RF], a[2][CG];
        int sw[2][RF], sa[2][CG];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t keep = s * 256 + j * 128 < k_len ? 0xFFu : 0u;
#pragma unroll
            for (int i = 0; i < RF; ++i) {
                w[j][i] = frag(at, 16 * i, j);
                sw[j][i] = (int)(*reinterpret_cast<const uint32_t*>(sc + (16 * i + r) * 16 + 4 * j) >> (8 * g) & keep);
            }
            if constexpr (kX > 0) {
                const uint8_t* x = at + kW + (r < kX ? r : 0) * 512 + j * 256 + g * 64;
                uint32_t v[4][4], m = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const u32x4 q = *reinterpret_cast<const u32x4*>(x + e * 16);
                    v[e][0] = q.x; v[e][1] = q.y; v[e][2] = q.z; v[e][3] = q.w;
                    m = max(m, mx_absmax8<kIn>(v[e]));
                }
                const uint32_t byte = mx_scale_byte(m);
                a[j][0] = v8i{(int)mx_codes8<kIn>(v[0], byte), (int)mx_codes8<kIn>(v[1], byte), (int)mx_codes8<kIn>(v[2], byte),
                              (int)mx_codes8<kIn>(v[3], byte)};
                sa[j][0] = (int)byte;
            } else {
#pragma unroll
                for (int i = 0; i < CG; ++i) {
                    a[j][i] = frag(at + kW, 16 * i, j);
                    sa[j][i] = (int)(*reinterpret_cast<const uint32_t*>(sc + (16 * (RF + i) + r) * 16 + 4 * j) >> (8 * g) & keep);
                }
            }
        }
        wait_lds();   // all of the stage is read: its buffer may be filled again
        issue(buf, s + kDepth);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < RF; ++i)
#pragma unroll
                for (int c = 0; c < CG; ++c)
                    acc[i][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[j][i], a[j][c], acc[i][c], 4, 4, 0, sw[j][i], 0,
                                                                                   sa[j][c]);
    };

    // in flight: kDepth stages, their scales just ahead of each pair
    static_for<kDepth>([&](auto b_) {
        constexpr int b = decltype(b_)::value;
        if constexpr (b % 2 == 0) issue_scales(b / 2);
        issue(b, b);
    });
    for (int s = 0; s < S; s += kDepth) {
        static_for<kDepth>([&](auto b_) {
            constexpr int b = decltype(b_)::value;
            // behind stage s + b: kDepth - 1 stages and the scales issued among
            // them (those of an even stage go ahead of it)
            wait_dma_n<(kDepth - 1) * kLoads + (kDepth - 1 + (b & 1)) / 2 * kScaleLoads>();
            if constexpr (b % 2 == 0) issue_scales((s + b + kDepth) / 2);
            use(b, s + b);
        });
    }
    wait_dma();
    __syncthreads();

    float* sums = reinterpret_cast<float*>(smem) + wave * (kSums / 4);
#pragma unroll
    for (int i = 0; i < RF; ++i)
#pragma unroll
        for (int c = 0; c < CG; ++c)
            *reinterpret_cast<v4f*>(sums + ((i * CG + c) * 64 + lane) * 4) = acc[i][c];
    __syncthreads();
    for (int q = wave; q < RF * CG; q += kWaves) {
        v4f y = {};
#pragma unroll
        for (int v = 0; v < kWaves; ++v) y += *reinterpret_cast<const v4f*>(smem + v * kSums + (q * 64 + lane) * 16);
        const int m = (q % CG) * 16 + r, n = n0 + (q / CG) * 16 + 4 * g;
        if (m >= p.M || n >= p.N) continue;
        uint16_t* d = p.D + (int64_t)m * p.ldd + n;
        if (n + 4 <= p.N && p.ldd % 4 == 0 && (reinterpret_cast<uintptr_t>(p.D) & 7) == 0) {
            *reinterpret_cast<u32x2*>(d) = u32x2{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < p.N) d[e] = (uint16_t)pack_bf16(y[e], 0.0f);
        }
    }
}

template <int RF, int CG, int kX, int kIn>
static int launch(const MxGemmArgs& p, hipStream_t st) {
    mxfp4_rows_kernel<RF, CG, kX, kIn, kRowsWaves, kRowsDepth><<<(p.N + 16 * RF - 1) / (16 * RF), kRowsWaves * 64, 0, st>>>(p);
    KBN_CHECK_LAUNCH("mxfp4_gemm_nt");
    return 0;
}
template <int CG, int kX, int kIn>
static int launch_for(const MxGemmArgs& p, int rf, hipStream_t st) {
    if (rf == 1) return launch<1, CG, kX, kIn>(p, st);
    if (rf == 2) return launch<2, CG, kX, kIn>(p, st);
    if constexpr (CG < 4 && kX < 8)   // 64 rows have a cheaper tile, 5 to 16 rows of values come with N <= 48 CUs
        if (rf == 4) return launch<4, CG, kX, kIn>(p, st);
    return launch<3, CG, kX, kIn>(p, st);
}

template <int kIn>
static int launch_values(const MxGemmArgs& p, int rf, hipStream_t st) {
    switch (mxfp4_value_rows(p.M)) {
        case 2: return launch_for<1, 2, kIn>(p, rf, st);
        case 4: return launch_for<1, 4, kIn>(p, rf, st);
        case 8: return launch_for<1, 8, kIn>(p, rf, st);
        default: return launch_for<1, 16, kIn>(p, rf, st);
    }
}

int mxfp4_rows_launch(const MxGemmArgs& p, int rf, int x_dtype, hipStream_t st) {
    if (p.X) return x_dtype == kMxBf16 ? launch_values<kMxBf16>(p, rf, st) : launch_values<kMxF16>(p, rf, st);
    switch ((p.M + 15) / 16) {
        case 1: return launch_for<1, 0, kMxBf16>(p, rf, st);
        case 2: return launch_for<2, 0, kMxBf16>(p, rf, st);
        case 3: return launch_for<3, 0, kMxBf16>(p, rf, st);
        default: return launch_for<4, 0, kMxBf16>(p, rf, st);
    }
}

}  // namespace kbn
