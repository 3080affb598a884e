// The router's product: logits[t, e] = sum_h x[t, h] w[e, h] in fp32.
//
// Few experts (8 to some hundred) and a long sum: what bounds it is reading w
// (few tokens) or x (many).  No operand is worth the LDS: both are read
// straight into the registers that the matrix instruction takes, 16 bytes a
// lane, and the wavefronts of a workgroup share one tile of logits and split
// its K instead, unit by unit, their sums meeting in LDS in wavefront order
// (the same bits on every run; no second launch, no workspace).
//
// fp32 operands go through the 16-bit matrix instruction as well: a float is
// the exact sum of three bf16 numbers (8 + 8 + 8 bits of its significand, cut
// off by clearing low bits), and the products of pieces down to 2^-16 of the
// largest are added, as good as fp32 products.
#include "kbn_common.h"

namespace kbn {
namespace {

enum : int { kG16b = 0, kG16f = 1, kG32 = 2 };   // dtype codes: bf16, fp16, fp32

struct GateArgs {
    const void* x;
    int64_t ld_x;
    const void* w;
    int64_t ld_w;
    float* out;
    int64_t ld_o;
    int T, E, H;
};

template <int kD> constexpr int bytes_of() { return kD == kG32 ? 4 : 2; }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, (int)kRsrcWord3);
}

// Eight consecutive values of a row as they lie in memory.
template <int kD> struct Raw8 { u32x4 v[kD == kG32 ? 2 : 1]; };

template <int kD>
__device__ __forceinline__ Raw8<kD> load_raw8(__amdgpu_buffer_rsrc_t rs, int off) {
    Raw8<kD> r;
    r.v[0] = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0);
    if constexpr (kD == kG32) r.v[1] = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 16, 0);
    return r;
}

template <int kD>
__device__ __forceinline__ void to_floats(const Raw8<kD>& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kD == kG32) {
            f[i] = __uint_as_float(r.v[0][i]);
            f[4 + i] = __uint_as_float(r.v[1][i]);
        } else {
            const uint32_t w = r.v[0][i];
            if constexpr (kD == kG16b) {
                f[2 * i] = bf16lo(w);
                f[2 * i + 1] = bf16hi(w);
            } else {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const h2 h = __builtin_bit_cast(h2, w);
                f[2 * i] = (float)h.x;
                f[2 * i + 1] = (float)h.y;
            }
        }
    }
}

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// bf16 pieces of a lane's eight values: kP of them, whose sum they are.
template <int kP> struct Pieces { u32x4 p[kP]; };

template <int kD, int kP>
__device__ __forceinline__ Pieces<kP> split(const Raw8<kD>& r) {
    Pieces<kP> o;
    if constexpr (kP == 1) {
        o.p[0] = r.v[0];
    } else {
        float f[8];
        to_floats<kD>(r, f);
#pragma unroll
        for (int k = 0; k < kP; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a = __float_as_uint(f[2 * i]), b = __float_as_uint(f[2 * i + 1]);
                o.p[k][i] = __builtin_amdgcn_perm(b, a, 0x07060302u);   // the upper halves
                if (k + 1 < kP) {
                    // infinities and NaN stay whole in the first piece
                    const float ra = f[2 * i] - __uint_as_float(a & 0xFFFF0000u);
                    const float rb = f[2 * i + 1] - __uint_as_float(b & 0xFFFF0000u);
                    f[2 * i] = (a & 0x7F800000u) == 0x7F800000u ? 0.f : ra;
                    f[2 * i + 1] = (b & 0x7F800000u) == 0x7F800000u ? 0.f : rb;
                }
            }
    }
    return o;
}

template <bool kHalf>
__device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, const f32x4& c) {
    if constexpr (kHalf)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A tile of 16 kTM tokens x 16 kTE experts by a workgroup of kNW wavefronts;
// kDepth units of 64 K in flight a wavefront.
template <int kTM, int kTE, int kNW, int kDepth, int kX, int kW>
__global__ __launch_bounds__(64 * kNW) void router_gemm_tile_kernel(const GateArgs a) {
    __shared__ f32x4 part[kNW * kTM * kTE * 64];
    constexpr int bx = bytes_of<kX>(), bw = bytes_of<kW>();
    // two pieces hold fp16's 11 bits where the other side is bf16 pieces
    constexpr int PX = kX == kG32 ? 3 : (kX == kG16f && kW == kG32) ? 2 : 1;
    constexpr int PW = kW == kG32 ? 3 : 1;
    constexpr bool kHalf = kX == kG16f && kW == kG16f;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t0 = blockIdx.y * 16 * kTM, e0 = blockIdx.x * 16 * kTE;
    const int nt = min(16 * kTM, a.T - t0), ne = min(16 * kTE, a.E - e0);
    // rows past the tile's last lie outside the descriptors and read zeros
    const __amdgpu_buffer_rsrc_t xr =
        rsrc(static_cast<const uint8_t*>(a.x) + (int64_t)t0 * a.ld_x * bx, (int)(((int64_t)(nt - 1) * a.ld_x + a.H) * bx));
    const __amdgpu_buffer_rsrc_t wr =
        rsrc(static_cast<const uint8_t*>(a.w) + (int64_t)e0 * a.ld_w * bw, (int)(((int64_t)(ne - 1) * a.ld_w + a.H) * bw));
    const int row = lane & 15, q = lane >> 4;
    int xo[kTM], wo[kTE];
#pragma unroll
    for (int i = 0; i < kTM; ++i) xo[i] = 16 * i + row < nt ? ((16 * i + row) * (int)a.ld_x + 16 * q) * bx : kOob;
#pragma unroll
    for (int i = 0; i < kTE; ++i) wo[i] = 16 * i + row < ne ? ((16 * i + row) * (int)a.ld_w + 16 * q) * bw : kOob;
    // lane q of a row owns K 16 q .. 16 q + 15 of the unit, eight in each of two
    // products (any order of K will do, if both operands have the same): the
    // loads of a unit cover whole 128-byte lines
    Raw8<kX> xb[kDepth][kTM][2];
    Raw8<kW> wb[kDepth][kTE][2];
    auto load = [&](int d, int u) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int k = 64 * u + 16 * q + 8 * s;
            const bool in = k < a.H;   // H is a multiple of 8
#pragma unroll
            for (int i = 0; i < kTM; ++i)
                xb[d][i][s] = load_raw8<kX>(xr, in && xo[i] >= 0 ? xo[i] + (64 * u + 8 * s) * bx : kOob);
#pragma unroll
            for (int i = 0; i < kTE; ++i)
                wb[d][i][s] = load_raw8<kW>(wr, in && wo[i] >= 0 ? wo[i] + (64 * u + 8 * s) * bw : kOob);
        }
    };
    f32x4 acc[kTM][kTE];
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
        for (int j = 0; j < kTE; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](int d) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            Pieces<PX> px[kTM];
            Pieces<PW> pw[kTE];
#pragma unroll
            for (int i = 0; i < kTM; ++i) px[i] = split<kX, PX>(xb[d][i][s]);
#pragma unroll
            for (int j = 0; j < kTE; ++j) pw[j] = split<kW, PW>(wb[d][j][s]);
#pragma unroll
            for (int sum = PX + PW - 2; sum >= 0; --sum) {   // the smallest products first
                if (sum > 2) continue;
#pragma unroll
                for (int m = 0; m < PX; ++m) {
                    const int n = sum - m;
                    if (n < 0 || n >= PW) continue;
#pragma unroll
                    for (int i = 0; i < kTM; ++i)
#pragma unroll
                        for (int j = 0; j < kTE; ++j) acc[i][j] = mma<kHalf>(px[i].p[m], pw[j].p[n], acc[i][j]);
                }
            }
        }
    };
    const int units = (a.H + 63) / 64;
#pragma unroll
    for (int d = 0; d < kDepth; ++d) load(d, wave + d * kNW);
    for (int u = wave; u < units; u += kNW * kDepth) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            multiply(d);
            load(d, u + (d + kDepth) * kNW);
        }
    }
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
        for (int j = 0; j < kTE; ++j) part[((wave * kTM + i) * kTE + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int s = threadIdx.x; s < kTM * kTE * 64; s += 64 * kNW) {
        f32x4 v = part[s];
#pragma unroll
        for (int n = 1; n < kNW; ++n) v += part[n * kTM * kTE * 64 + s];
        const int l = s & 63, tile = s >> 6;
        const int e = 16 * (tile % kTE) + (l & 15), t = 16 * (tile / kTE) + 4 * (l >> 4);
        if (e < ne) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (t + i < nt) a.out[(int64_t)(t0 + t + i) * a.ld_o + e0 + e] = v[i];
        }
    }
}

// Few tokens: a workgroup for one expert, whose row it reads once; fp32
// multiply-adds, lanes and wavefronts summed by butterfly and in order.
constexpr int kRowWaves = 4;

template <int kN, int kX, int kW>
__global__ __launch_bounds__(64 * kRowWaves) void router_gemm_rows_kernel(const GateArgs a) {
    __shared__ float part[kRowWaves][kN];
    constexpr int bx = bytes_of<kX>(), bw = bytes_of<kW>();
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int e = blockIdx.x;
    // past the row's end both operands read zeros
    const __amdgpu_buffer_rsrc_t wr = rsrc(static_cast<const uint8_t*>(a.w) + (int64_t)e * a.ld_w * bw, a.H * bw);
    float acc[kN];
#pragma unroll
    for (int t = 0; t < kN; ++t) acc[t] = 0.f;
    for (int k = (wave * 64) * 8; k < a.H; k += 64 * kRowWaves * 8) {
        const int at = k + 8 * lane;
        const Raw8<kW> wv = load_raw8<kW>(wr, at * bw);
        Raw8<kX> xv[kN];
#pragma unroll
        for (int t = 0; t < kN; ++t) {
            const __amdgpu_buffer_rsrc_t xr =
                rsrc(static_cast<const uint8_t*>(a.x) + (int64_t)min(t, a.T - 1) * a.ld_x * bx, a.H * bx);
            xv[t] = load_raw8<kX>(xr, at * bx);
        }
        float wf[8];
        to_floats<kW>(wv, wf);
#pragma unroll
        for (int t = 0; t < kN; ++t) {
            float xf[8];
            to_floats<kX>(xv[t], xf);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[t] = fmaf(xf[j], wf[j], acc[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < kN; ++t)
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) acc[t] += __shfl_xor(acc[t], d, 64);
    if (lane == 0) {
#pragma unroll
        for (int t = 0; t < kN; ++t) part[wave][t] = acc[t];
    }
    __syncthreads();
    if ((int)threadIdx.x < min(kN, a.T)) {
        float v = part[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < kRowWaves; ++w) v += part[w][threadIdx.x];
        a.out[(int64_t)threadIdx.x * a.ld_o + e] = v;
    }
}

constexpr int kRowTokens = 8;   // most tokens of the rows kernel

template <int kX, int kW>
void launch(const GateArgs& a, hipStream_t st) {
    if (a.T <= kRowTokens) {
        const dim3 grid((unsigned)a.E), block(64 * kRowWaves);
        if (a.T <= 1) router_gemm_rows_kernel<1, kX, kW><<<grid, block, 0, st>>>(a);
        else if (a.T <= 2) router_gemm_rows_kernel<2, kX, kW><<<grid, block, 0, st>>>(a);
        else if (a.T <= 4) router_gemm_rows_kernel<4, kX, kW><<<grid, block, 0, st>>>(a);
        else router_gemm_rows_kernel<8, kX, kW><<<grid, block, 0, st>>>(a);
        return;
    }
    // the largest tile that still gives every CU a workgroup
    const int cus = cu_count();
    auto groups = [&](int tm, int te) {
        return (int64_t)((a.T + 16 * tm - 1) / (16 * tm)) * ((a.E + 16 * te - 1) / (16 * te));
    };
    auto grid = [&](int tm, int te) {
        return dim3((unsigned)((a.E + 16 * te - 1) / (16 * te)), (unsigned)((a.T + 16 * tm - 1) / (16 * tm)));
    };
    if (groups(4, 4) >= cus) router_gemm_tile_kernel<4, 4, 4, 2, kX, kW><<<grid(4, 4), dim3(256), 0, st>>>(a);
    else if (groups(2, 2) >= cus) router_gemm_tile_kernel<2, 2, 8, 2, kX, kW><<<grid(2, 2), dim3(512), 0, st>>>(a);
    else router_gemm_tile_kernel<1, 1, 16, 2, kX, kW><<<grid(1, 1), dim3(1024), 0, st>>>(a);
}

}  // namespace
}  // namespace kbn

using namespace kbn;

extern "C" int kbn_moe_router_gemm(const void* x, int x_dtype, int64_t ld_x, const void* w, int w_dtype, int64_t ld_w,
                                   float* out, int64_t ld_out, int64_t T, int64_t E, int64_t H, void* stream) {
    const char* what = "moe_router_gemm";
    KBN_CHECK_ARG(x_dtype >= 0 && x_dtype <= 2 && w_dtype >= 0 && w_dtype <= 2,
                  "%s: dtype codes %d and %d (0 bf16, 1 fp16, 2 fp32)", what, x_dtype, w_dtype);
    KBN_CHECK_ARG(w_dtype == x_dtype || w_dtype == kG32, "%s: weights must have the rows' dtype or be fp32", what);
    KBN_CHECK_ARG(T >= 0 && T <= 0x7FFFFFFFLL - 64 && E >= 1 && E <= 65535 * 16, "%s: bad sizes T=%lld, E=%lld", what,
                  (long long)T, (long long)E);
    KBN_CHECK_ARG(H >= 8 && H % 8 == 0 && H <= (1 << 22), "%s: H=%lld must be a multiple of 8 in [8, 2^22]", what, (long long)H);
    if (T == 0) return 0;
    KBN_CHECK_ARG(x && w && out, "%s: null pointer", what);
    const int bx = x_dtype == kG32 ? 4 : 2, bw = w_dtype == kG32 ? 4 : 2;
    KBN_CHECK_ARG(aligned16(x) && aligned16(w) && ld_x >= H && ld_w >= H && ld_x * bx % 16 == 0 && ld_w * bw % 16 == 0,
                  "%s: rows must be 16-byte aligned with strides of at least H", what);
    KBN_CHECK_ARG(ld_x < (1 << 23) && ld_w < (1 << 23), "%s: row strides must be below 2^23 elements", what);
    KBN_CHECK_ARG(ld_out >= E && (reinterpret_cast<uintptr_t>(out) & 3u) == 0, "%s: bad output rows", what);
    GateArgs a{x, ld_x, w, ld_w, out, ld_out, (int)T, (int)E, (int)H};
    KBN_CHECK_ARG((T + 15) / 16 <= 65535, "%s: T=%lld is more than 2^20 - 16 rows", what, (long long)T);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (x_dtype == kG16b) w_dtype == kG16b ? launch<kG16b, kG16b>(a, st) : launch<kG16b, kG32>(a, st);
    else if (x_dtype == kG16f) w_dtype == kG16f ? launch<kG16f, kG16f>(a, st) : launch<kG16f, kG32>(a, st);
    else launch<kG32, kG32>(a, st);
    KBN_CHECK_LAUNCH(what);
    return 0;
}
