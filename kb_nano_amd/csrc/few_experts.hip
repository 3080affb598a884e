// A mixture-of-experts layer for at most 64 tokens, in two launches:
//   h[t, e]  = silu(G_e x_t) * (U_e x_t)          (gate_up_kernel)
//   out[t]   = sum_e c[t, e] W2_e h[t, e]          (down_kernel)
// with w13[e] = [G_e | U_e] and c[t, e] the sum of token t's routing weights
// of the slots that name expert e; ids outside [0, E) count for nothing.
// Weights are FP8 codes with fp32 128x128 block scales, or MXFP4.
//
// At these sizes the layer is the time to stream each named expert's weights
// once, so the activations are not quantized: weight codes widen exactly to
// bf16 (an MXFP4 code with its power-of-two scale too) and run through the
// bf16 matrix instruction, 16 weight rows by 16 tokens, sums in fp32.  FP8
// block scales multiply each 128-K block's fp32 sum.  An operand with more
// than bf16's 8 significant bits (fp16 activations, and h, which has fp32's)
// goes as a pair of bf16 values, x = hi + lo, hi the nearest and lo the
// nearest to the rest: 16 bits and more, for one more matrix instruction on
// operands that are there already.
//
// A token is a column: lane l of a 16-column group serves token 16 group +
// (l & 15), and an expert's columns of other tokens read as zeros.  The down
// kernel owns 16 output columns of every token over all experts, so the sum
// over experts stays in registers, in a fixed order.
#include "mxfp4.h"

#include <algorithm>
#include <type_traits>

namespace kbn {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxTokens = 64, kMaxTopk = 32, kMaxExperts = 1024;
enum WFormat : int { kWFp8 = 0, kWMxfp4 = 1 };

struct ExpertsArgs {
    const void* x;
    int64_t ld_x;
    const uint8_t *w13, *w2;
    const void *s13, *s2;      // fp32 [E, rows/128, K/128] or bytes [E, rows, K/32]
    const void* ids;
    int id64;
    const float* weights;
    int T, H, I, E, topk;
    uint16_t* h;               // hi then lo, each [T * topk, I]; row t * topk + first slot of the expert
    void* out;
    int64_t ld_out;
};

__device__ __forceinline__ int expert_of(const ExpertsArgs& p, int pair) {
    const int64_t e = p.id64 ? static_cast<const int64_t*>(p.ids)[pair] : static_cast<const int32_t*>(p.ids)[pair];
    return e >= 0 && e < p.E ? (int)e : -1;
}

// First slot of token t that names expert e (-1: none), and the sum of the
// weights of all that do.
__device__ __forceinline__ int find_slot(const int* ids, const float* weights, int topk, int t, int e, float& c) {
    int slot = -1;
    c = 0.0f;
    for (int j = 0; j < topk; ++j)
        if (ids[t * topk + j] == e) {
            c += weights[t * topk + j];
            if (slot < 0) slot = j;
        }
    return slot;
}

// 128 K of 16 weight rows: lane (row l & 15, part l >> 4).
//   FP8: the lane holds k = 64 j + 16 part .. + 15 for j = 0, 1;
//   MXFP4: k = 32 part .. + 31, one scale group.
template <int kW>
struct WFrag {
    u32x4 q[kW == kWFp8 ? 2 : 1];
    uint32_t byte;   // MXFP4
};
template <int kW>
__device__ __forceinline__ WFrag<kW> load_w(const uint8_t* row, const uint8_t* srow, int k, int part) {
    WFrag<kW> f;
    if constexpr (kW == kWFp8) {
        f.q[0] = *reinterpret_cast<const u32x4*>(row + k + 16 * part);
        f.q[1] = *reinterpret_cast<const u32x4*>(row + k + 64 + 16 * part);
        f.byte = 0;
    } else {
        f.q[0] = *reinterpret_cast<const u32x4*>(row + k / 2 + 16 * part);
        f.byte = srow[k / 32 + part];
    }
    return f;
}
// The i-th (of four) eight values of a fragment, in bf16 (exact).
template <int kW>
__device__ __forceinline__ bf16x8 widen_w(const WFrag<kW>& f, int i) {
    u32x4 r;
    if constexpr (kW == kWFp8) {
        const uint32_t a = i & 1 ? f.q[i >> 1].z : f.q[i >> 1].x, b = i & 1 ? f.q[i >> 1].w : f.q[i >> 1].y;
        r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
        r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
        r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
        r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
    } else {
        const float sc = __uint_as_float(f.byte << 23);
        const uint32_t a = f.q[0][i];
        r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, sc, 0));
        r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, sc, 1));
        r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, sc, 2));
        r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, sc, 3));
    }
    return __builtin_bit_cast(bf16x8, r);
}
// K offset, within the 128, of a lane's i-th eight values.
template <int kW>
__device__ __forceinline__ int k_of(int i, int part) {
    return kW == kWFp8 ? 64 * (i >> 1) + 16 * part + 8 * (i & 1) : 32 * part + 8 * i;
}

__device__ __forceinline__ v4f mfma(bf16x8 a, bf16x8 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The rest of v beside its nearest bf16 (0 beside an infinity).
__device__ __forceinline__ __bf16 low_part(float v, __bf16 hi) {
    return fabsf((float)hi) == __builtin_inff() ? (__bf16)0.0f : (__bf16)(v - (float)hi);
}
// x = hi + lo
__device__ __forceinline__ void split8(f16x8 x, bf16x8& hi, bf16x8& lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = (float)x[i];
        const __bf16 a = (__bf16)v;
        hi[i] = a;
        lo[i] = low_part(v, a);
    }
}

// The token ids in LDS: -1 for those that name no expert.
__device__ __forceinline__ void load_ids(const ExpertsArgs& p, int* ids, float* weights, int tid, int n) {
    for (int i = tid; i < p.T * p.topk; i += n) {
        ids[i] = expert_of(p, i);
        if (weights) weights[i] = p.weights[i];
    }
}

constexpr int kWaves = 4;

// Workgroup: 16 rows of h (16 gate and 16 up rows) of one expert, K split over
// the wavefronts.  slot: a routed pair whose expert no earlier pair names
// (by_pair), or an expert.
template <int kW, bool kF16, int kGroups>
__global__ __launch_bounds__(kWaves * 64) void gate_up_kernel(const ExpertsArgs p, int by_pair) {
    __shared__ int ids[kMaxTokens * kMaxTopk];
    __shared__ float red[kWaves][2][kGroups][4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = lane >> 4, col = lane & 15;
    const int e = by_pair ? expert_of(p, blockIdx.y) : (int)blockIdx.y;
    if (e < 0) return;
    load_ids(p, ids, nullptr, tid, kWaves * 64);
    __syncthreads();
    if (by_pair)
        for (int i = 0; i < (int)blockIdx.y; ++i)
            if (ids[i] == e) return;   // an earlier pair's workgroup has this expert
    int slot[kGroups];
    bool any = false;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int t = 16 * g + col;
        slot[g] = -1;
        if (t < p.T)
            for (int j = p.topk - 1; j >= 0; --j)
                if (ids[t * p.topk + j] == e) slot[g] = j;
        any |= __ballot(slot[g] >= 0) != 0;
    }
    if (!any) return;
    const int i0 = blockIdx.x * 16, KB = p.H / 128;
    const int64_t rows = (int64_t)e * 2 * p.I, gr = rows + i0 + col, ur = gr + p.I;
    const int64_t ldw = kW == kWFp8 ? p.H : p.H / 2, lds = p.H / 32;
    const uint8_t* const w[2] = {p.w13 + gr * ldw, p.w13 + ur * ldw};
    const uint8_t* sb[2] = {nullptr, nullptr};
    const float* sf[2] = {nullptr, nullptr};
    if constexpr (kW == kWFp8) {
        const float* s = static_cast<const float*>(p.s13) + (rows / 128) * KB;
        sf[0] = s + (int64_t)(i0 / 128) * KB;
        sf[1] = s + (int64_t)((p.I + i0) / 128) * KB;
    } else {
        sb[0] = static_cast<const uint8_t*>(p.s13) + gr * lds;
        sb[1] = static_cast<const uint8_t*>(p.s13) + ur * lds;
    }
    v4f acc[2][kGroups] = {};
    for (int kb = wave; kb < KB; kb += kWaves) {
        const int k = kb * 128;
        WFrag<kW> f[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) f[h] = load_w<kW>(w[h], sb[h], k, part);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            if (__ballot(slot[g] >= 0) == 0) continue;
            bf16x8 hi[4] = {}, lo[4] = {};
            if (slot[g] >= 0) {
                const uint16_t* x = static_cast<const uint16_t*>(p.x) + (int64_t)(16 * g + col) * p.ld_x + k;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u32x4 v = *reinterpret_cast<const u32x4*>(x + k_of<kW>(i, part));
                    if constexpr (kF16) split8(__builtin_bit_cast(f16x8, v), hi[i], lo[i]);
                    else hi[i] = __builtin_bit_cast(bf16x8, v);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                v4f s = kW == kWFp8 ? v4f{} : acc[h][g];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bf16x8 a = widen_w<kW>(f[h], i);
                    s = mfma(a, hi[i], s);
                    if constexpr (kF16) s = mfma(a, lo[i], s);
                }
                if constexpr (kW == kWFp8) acc[h][g] += s * sf[h][kb];
                else acc[h][g] = s;
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[wave][h][g][i][lane] = acc[h][g][i];
    __syncthreads();
    const int64_t pairs = (int64_t)p.T * p.topk;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {   // lane (part, col), register i = wave: row i0 + 4 part + wave of token 16 g + col
        if (slot[g] < 0) continue;
        float gate = 0.0f, up = 0.0f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            gate += red[v][0][g][wave][lane];
            up += red[v][1][g][wave][lane];
        }
        const float y = gate / (1.0f + __expf(-gate)) * up;
        const int64_t at = ((int64_t)(16 * g + col) * p.topk + slot[g]) * p.I + i0 + 4 * part + wave;
        const __bf16 hi = (__bf16)y;
        p.h[at] = __builtin_bit_cast(uint16_t, hi);
        p.h[pairs * p.I + at] = __builtin_bit_cast(uint16_t, low_part(y, hi));
    }
}

// Workgroup: 16 output columns of every token; the (expert, 128 K) blocks of
// the named experts are split into one run for each wavefront.
template <int kW, bool kF16, int kGroups>
__global__ __launch_bounds__(kWaves * 64) void down_kernel(const ExpertsArgs p) {
    __shared__ int ids[kMaxTokens * kMaxTopk];
    __shared__ float weights[kMaxTokens * kMaxTopk];
    __shared__ uint32_t named[kMaxExperts / 32];
    __shared__ uint16_t list[kMaxExperts];
    __shared__ int count;
    __shared__ float red[kWaves][kGroups][4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = lane >> 4, col = lane & 15;
    if (tid < kMaxExperts / 32) named[tid] = 0;
    load_ids(p, ids, weights, tid, kWaves * 64);
    __syncthreads();
    for (int i = tid; i < p.T * p.topk; i += kWaves * 64)
        if (ids[i] >= 0) atomicOr(&named[ids[i] >> 5], 1u << (ids[i] & 31));
    __syncthreads();
    if (tid == 0) {
        int n = 0;
        for (int i = 0; i < kMaxExperts / 32; ++i)
            for (uint32_t b = named[i]; b; b &= b - 1) list[n++] = (uint16_t)(32 * i + __ffs((int)b) - 1);
        count = n;
    }
    __syncthreads();
    const int KB = p.I / 128, n0 = blockIdx.x * 16;
    const int units = count * KB, from = (int)((int64_t)units * wave / kWaves), to = (int)((int64_t)units * (wave + 1) / kWaves);
    const int64_t ldw = kW == kWFp8 ? p.I : p.I / 2, lds = p.I / 32, pairs = (int64_t)p.T * p.topk;
    v4f acc[kGroups] = {};
    int slot[kGroups], have = -1;
    float c[kGroups];
    const uint8_t *w = nullptr, *sb = nullptr;
    const float* sf = nullptr;
    for (int u = from; u < to; ++u) {
        const int a = u / KB, kb = u - a * KB, k = kb * 128;
        if (a != have) {
            have = a;
            const int e = list[a];
            const int64_t row = (int64_t)e * p.H + n0 + col;
            w = p.w2 + row * ldw;
            if constexpr (kW == kWFp8) sf = static_cast<const float*>(p.s2) + ((int64_t)e * (p.H / 128) + n0 / 128) * KB;
            else sb = static_cast<const uint8_t*>(p.s2) + row * lds;
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                slot[g] = -1;
                c[g] = 0.0f;
                if (16 * g + col < p.T) slot[g] = find_slot(ids, weights, p.topk, 16 * g + col, e, c[g]);
            }
        }
        const WFrag<kW> f = load_w<kW>(w, sb, k, part);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            if (__ballot(slot[g] >= 0) == 0) continue;
            bf16x8 hi[4] = {}, lo[4] = {};
            if (slot[g] >= 0) {
                const uint16_t* h = p.h + ((int64_t)(16 * g + col) * p.topk + slot[g]) * p.I + k;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    hi[i] = *reinterpret_cast<const bf16x8*>(h + k_of<kW>(i, part));
                    lo[i] = *reinterpret_cast<const bf16x8*>(h + pairs * p.I + k_of<kW>(i, part));
                }
            }
            v4f s = {};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bf16x8 x = widen_w<kW>(f, i);
                s = mfma(x, hi[i], s);
                s = mfma(x, lo[i], s);
            }
            // other tokens' columns stay as they are: zeros times an expert's
            // NaN weight would not be zeros
            if (slot[g] >= 0) acc[g] += s * (kW == kWFp8 ? c[g] * sf[kb] : c[g]);
        }
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wave][g][i][lane] = acc[g][i];
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int t = 16 * g + col;
        if (t >= p.T) continue;
        float y = 0.0f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) y += red[v][g][wave][lane];
        uint16_t* o = static_cast<uint16_t*>(p.out) + (int64_t)t * p.ld_out + n0 + 4 * part + wave;
        if constexpr (kF16) *o = __builtin_bit_cast(uint16_t, (_Float16)y);
        else *o = __builtin_bit_cast(uint16_t, (__bf16)y);
    }
}

template <int kW, bool kF16, int kGroups>
static int launch(const ExpertsArgs& p, hipStream_t st) {
    const int pairs = p.T * p.topk, by_pair = pairs <= p.E;
    gate_up_kernel<kW, kF16, kGroups><<<dim3(p.I / 16, by_pair ? pairs : p.E), kWaves * 64, 0, st>>>(p, by_pair);
    KBN_CHECK_LAUNCH("few_token_experts");
    down_kernel<kW, kF16, kGroups><<<p.H / 16, kWaves * 64, 0, st>>>(p);
    KBN_CHECK_LAUNCH("few_token_experts");
    return 0;
}

template <int kW, bool kF16>
static int launch_for(const ExpertsArgs& p, hipStream_t st) {
    return p.T <= 16 ? launch<kW, kF16, 1>(p, st) : p.T <= 32 ? launch<kW, kF16, 2>(p, st) : launch<kW, kF16, 4>(p, st);
}

}  // namespace kbn

using namespace kbn;

extern "C" int64_t kbn_few_token_experts_workspace_bytes(int64_t T, int64_t topk, int64_t I) {
    if (T < 0 || T > kMaxTokens || topk < 1 || topk > kMaxTopk || I < 0 || I >= (1LL << 31)) return 0;
    return T * topk * I * 4;
}

extern "C" int kbn_few_token_experts(const void* x, int x_dtype, int64_t ld_x, const void* w13, const void* s13, const void* w2,
                                     const void* s2, int w_format, const float* topk_weights, const void* topk_ids, int id_bytes,
                                     int64_t T, int64_t topk, int64_t E, int64_t H, int64_t I, void* out, int64_t ld_out,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "few_token_experts";
    KBN_CHECK_ARG(x_dtype == kMxBf16 || x_dtype == kMxF16, "%s: unknown dtype code %d (0 bf16, 1 fp16)", what, x_dtype);
    KBN_CHECK_ARG(w_format == kWFp8 || w_format == kWMxfp4, "%s: unknown weight format %d", what, w_format);
    KBN_CHECK_ARG(id_bytes == 4 || id_bytes == 8, "%s: ids of %d bytes", what, id_bytes);
    KBN_CHECK_ARG(T >= 0 && T <= kMaxTokens, "%s: T=%lld tokens, at most %d", what, (long long)T, kMaxTokens);
    KBN_CHECK_ARG(topk >= 1 && topk <= kMaxTopk, "%s: top_k=%lld outside [1, %d]", what, (long long)topk, kMaxTopk);
    KBN_CHECK_ARG(E >= 1 && E <= kMaxExperts, "%s: num_experts=%lld outside [1, %d]", what, (long long)E, kMaxExperts);
    KBN_CHECK_ARG(H > 0 && I > 0 && H % 128 == 0 && I % 128 == 0 && H < (1 << 24) && I < (1 << 24),
                  "%s: H=%lld and I=%lld must be multiples of 128", what, (long long)H, (long long)I);
    if (T == 0) return 0;
    KBN_CHECK_ARG(ld_x >= H && ld_x % 8 == 0 && x && aligned16(x), "%s: input rows must be 16-byte aligned", what);
    KBN_CHECK_ARG(ld_out >= H && out && reinterpret_cast<uintptr_t>(out) % 2 == 0, "%s: output row stride %lld below H=%lld", what,
                  (long long)ld_out, (long long)H);
    KBN_CHECK_ARG(w13 && w2 && s13 && s2 && topk_weights && topk_ids, "%s: null pointer", what);
    KBN_CHECK_ARG(aligned16(w13) && aligned16(w2), "%s: weights must be 16-byte aligned", what);
    KBN_CHECK_ARG(reinterpret_cast<uintptr_t>(s13) % 4 == 0 && reinterpret_cast<uintptr_t>(s2) % 4 == 0,
                  "%s: weight scales must be 4-byte aligned", what);
    const int64_t need = kbn_few_token_experts_workspace_bytes(T, topk, I);
    KBN_CHECK_ARG(workspace_bytes >= need && aligned16(workspace) && workspace, "%s: workspace of %lld bytes needed, got %lld",
                  what, (long long)need, (long long)workspace_bytes);
    const ExpertsArgs p{x, ld_x, (const uint8_t*)w13, (const uint8_t*)w2, s13, s2, topk_ids, id_bytes == 8, topk_weights,
                        (int)T, (int)H, (int)I, (int)E, (int)topk, (uint16_t*)workspace, out, ld_out};
    const hipStream_t st = (hipStream_t)stream;
    if (w_format == kWFp8) return x_dtype == kMxF16 ? launch_for<kWFp8, true>(p, st) : launch_for<kWFp8, false>(p, st);
    return x_dtype == kMxF16 ? launch_for<kWMxfp4, true>(p, st) : launch_for<kWMxfp4, false>(p, st);
}
