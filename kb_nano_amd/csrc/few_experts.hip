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
// bf16 matrix instruction, 16 weight rows by 16 activation rows, sums in fp32.
// FP8 block scales multiply each 128-K block's fp32 sum.  fp16 activations meet
// FP8 codes in fp16, where those are exact as well.  Another operand with more
// than bf16's 8 significant bits (fp16 activations of MXFP4 weights, whose
// scales pass fp16's range, and h, which has fp32's) goes as a pair of bf16
// values, x = hi + lo, hi the nearest and lo the nearest to the rest: 16 bits
// and more, for one more matrix instruction on weights that are there already.
// Few rows an expert: bound by the weight stream, which a large read reaches 6.6
// TB/s with: 64 tokens over 256 experts (7168, 2048) 1440 to 1475 us, 6.6 to 6.8
// TB/s; 16 of fp16 over 128 (4096, 1536) 243 to 254 us, 6.0 to 6.3; 5 over those in
// MXFP4 69 us, 5.1; one token on an eighth of the 256, 44 MB, 14.8 us, of which two
// launches and their joins are about six.  fp16 activations of MXFP4 weights take
// twice the matrix instructions: 5 tokens 112 us (bf16 in the same run 74), 64 over
// 64 (7168, 1024) 329 (237).
// Many rows an expert: 2 to 5 times the weights' time (64 tokens over 8 experts
// (4096, 14336), 16 rows each, 443 us against 214), as a stage's activations serve
// 16 or 32 weight rows only and more than 16 rows read the weights again; the
// sorted-token layer is faster there.
//
// Both kernels stream like the few-rows MXFP4 product: each wavefront has a
// private LDS ring filled by direct loads of whole 128-byte weight lines (a
// stage: 128 K of FP8, 256 K of MXFP4, and the activations of that K), no
// barrier in the loop.  An expert's tokens are taken kR at a time, a pass; one
// pass is the rule (2 tokens an expert at 64 tokens and 256 experts with 8 a
// token); further ones read the weights again, as far as L2 has lost them.
#include "mxfp4.h"

#include "gemm_kernel.h"

#include <cmath>

namespace kbn {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// A lambda that holds direct loads is inlined: a call would pass its scalar
// operands in vector registers.
#define KBN_INLINE __attribute__((always_inline))

constexpr int kMaxTokens = 64, kMaxTopk = 32, kMaxExperts = 1024;
enum WFormat : int { kWFp8 = 0, kWMxfp4 = 1 };

// A pass of an expert, and a row of one: what the gate/up launch writes down
// for the down launch.
struct Pass {
    uint16_t expert, rows;
    int first_row;
};
struct Row {
    uint16_t pair, token;   // pair: token * topk + slot
    float weight;
};

struct ExpertsArgs {
    const void* x;
    int64_t ld_x;
    const uint8_t *w13, *w2;
    const void *s13, *s2;      // fp32 [E, rows/128, K/128] or bytes [E, rows, K/32]
    const void* ids;
    int id64;
    const float* weights;
    int T, H, I, E, topk;
    int* count;                // passes
    Pass* passes;              // [T * topk]
    Row* rows;                 // [T * topk]
    uint16_t* h;               // [T * topk][I / 128][hi 128, lo 128]; row t * topk + first slot of the expert
    void* out;
    int64_t ld_out;
};

__device__ __forceinline__ int expert_of(const ExpertsArgs& p, int pair) {
    const int64_t e = p.id64 ? static_cast<const int64_t*>(p.ids)[pair] : static_cast<const int32_t*>(p.ids)[pair];
    return e >= 0 && e < p.E ? (int)e : -1;
}

// The i-th eight values of a lane's 16 bytes of weight codes (FP8: i < 2,
// MXFP4: i < 4), in bf16 (exact); byte: the MXFP4 group's scale.
template <int kW>
__device__ __forceinline__ bf16x8 widen_w(const u32x4& q, int i, uint32_t byte) {
    u32x4 r;
    if constexpr (kW == kWFp8) {
        const uint32_t a = i ? q.z : q.x, b = i ? q.w : q.y;
        r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
        r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
        r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
        r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
    } else {
        const float sc = __uint_as_float(byte << 23);
        const uint32_t a = q[i];
        r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, sc, 0));
        r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, sc, 1));
        r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, sc, 2));
        r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, sc, 3));
    }
    return __builtin_bit_cast(bf16x8, r);
}

// FP8 codes in fp16 (exact too), for fp16 activations.
__device__ __forceinline__ f16x8 widen_half(const u32x4& q, int i) {
    const uint32_t a = i ? q.z : q.x, b = i ? q.w : q.y;
    u32x4 r;
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true));
    return __builtin_bit_cast(f16x8, r);
}

__device__ __forceinline__ v4f mfma(bf16x8 a, bf16x8 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma(f16x8 a, f16x8 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
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

// A uniform load through the scalar cache: it leaves the count of vector loads
// in flight alone.
__device__ __forceinline__ float scalar_load(const float* p, int64_t i) {
    typedef const float __attribute__((address_space(4))) * Const;
    return ((Const)(uintptr_t)p)[i];
}


// What a wavefront's stage holds: 16 RF weight rows of 128 bytes, kR activation
// rows (kRowBytes each) and, for MXFP4, 8 scale bytes a weight row.  Sixteen-byte
// chunk c of a weight row q lies in slot c ^ swz(q), that of activation row r in
// slot c ^ (r & 15): no two lanes that read together share a bank.
template <int kW, int RF, int kR, int kRowBytes>
struct StageOf {
    static constexpr int kK = kW == kWFp8 ? 128 : 256;
    static constexpr int kWLoads = 2 * RF, kXLoads = kR * kRowBytes / 1024, kScaleLoads = kW == kWMxfp4;
    static constexpr int kLoads = kWLoads + kXLoads + kScaleLoads;
    static constexpr int kXAt = kWLoads * 1024, kScaleAt = kXAt + kXLoads * 1024, kBytes = kScaleAt + kScaleLoads * 256;
    static constexpr int kParts = kW == kWFp8 ? 2 : 4;   // matrix instructions per 16 bytes of codes

    // fragment f's codes, half j of the stage's K
    static __device__ __forceinline__ u32x4 w(const uint8_t* at, int f, int j, int r, int part) {
        return *reinterpret_cast<const u32x4*>(at + (16 * f + r) * 128 + (((4 * j + part) ^ swz(r)) << 4));
    }
    static __device__ __forceinline__ uint32_t scale(const uint8_t* at, int f, int j, int r, int part) {
        if constexpr (kW == kWFp8) return 0;
        else return *reinterpret_cast<const uint32_t*>(at + kScaleAt + (16 * f + r) * 8 + 4 * j) >> (8 * part) & 0xFFu;
    }
    // chunk c of activation row r (rows past kR: any other, their results go nowhere)
    static __device__ __forceinline__ u32x4 x(const uint8_t* at, int r, int c) {
        return *reinterpret_cast<const u32x4*>(at + kXAt + (r % kR) * kRowBytes + ((c ^ (r % kR)) << 4));
    }
};

// The routing written down for the down launch: the named experts in order,
// each one's tokens in order, kR rows a pass.  One workgroup.
template <int kWaves>
__device__ void write_passes(const ExpertsArgs& p, int kR, int* ids, float* weights) {
    __shared__ uint32_t named[kMaxExperts / 32];
    __shared__ int list[kMaxExperts], total, sums[2][kWaves];
    const int tid = threadIdx.x, n = kWaves * 64, pairs = p.T * p.topk;
    for (int i = tid; i < kMaxExperts / 32; i += n) named[i] = 0;
    for (int i = tid; i < pairs; i += n) {
        ids[i] = expert_of(p, i);
        weights[i] = p.weights[i];
    }
    __syncthreads();
    for (int i = tid; i < pairs; i += n)
        if (ids[i] >= 0) atomicOr(&named[ids[i] >> 5], 1u << (ids[i] & 31));
    __syncthreads();
    if (tid < 64) {   // the named experts' numbers, in order
        uint32_t w = tid < kMaxExperts / 32 ? named[tid] : 0;
        int at = __popc(w);
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(at, d);
            if (tid >= d) at += o;
        }
        if (tid == 63) total = at;
        at -= __popc(w);
        for (; w; w &= w - 1) list[at++] = 32 * tid + __ffs((int)w) - 1;
    }
    __syncthreads();
    int pass0 = 0, row0 = 0;
    for (int from = 0; from < total; from += n) {
        const int e = from + tid < total ? list[from + tid] : -1;
        int rows = 0;
        if (e >= 0)
            for (int t = 0; t < p.T; ++t) {
                bool hit = false;
                for (int j = 0; j < p.topk; ++j) hit |= ids[t * p.topk + j] == e;
                rows += hit;
            }
        int np = (rows + kR - 1) / kR, ends_p = np, ends_r = rows;
        for (int d = 1; d < 64; d *= 2) {
            const int a = __shfl_up(ends_p, d), b = __shfl_up(ends_r, d);
            if ((tid & 63) >= d) {
                ends_p += a;
                ends_r += b;
            }
        }
        if ((tid & 63) == 63) {
            sums[0][tid >> 6] = ends_p;
            sums[1][tid >> 6] = ends_r;
        }
        __syncthreads();
        int ps = pass0 + ends_p - np, rs = row0 + ends_r - rows;
        for (int w = 0; w < kWaves; ++w) {
            if (w < (tid >> 6)) {
                ps += sums[0][w];
                rs += sums[1][w];
            }
            pass0 += sums[0][w];
            row0 += sums[1][w];
        }
        __syncthreads();
        for (int q = 0; q < np; ++q) p.passes[ps + q] = Pass{(uint16_t)e, (uint16_t)min(kR, rows - q * kR), rs + q * kR};
        if (e >= 0)
            for (int t = 0; t < p.T; ++t) {
                int slot = -1;
                float c = 0.0f;
                for (int j = 0; j < p.topk; ++j)
                    if (ids[t * p.topk + j] == e) {
                        c += weights[t * p.topk + j];
                        if (slot < 0) slot = j;
                    }
                if (slot >= 0) p.rows[rs++] = Row{(uint16_t)(t * p.topk + slot), (uint16_t)t, c};
            }
    }
    if (tid == 0) *p.count = pass0;
}

// Workgroup 0 writes the passes.  The others own `run` tiles of 8 RF rows of h
// (as many gate and up rows) of one expert, K split over the wavefronts: the
// expert of a routed pair that is the first to name it (by_pair), or every
// expert in turn.  RF = 1: fragment rows 0 .. 7 are gate rows, 8 .. 15 up rows;
// RF = 2: one fragment each.  A wavefront's stages of all tiles and passes form
// one sequence, so the ring stays full while a tile's sums meet in LDS; the
// first stages' weights are asked for before the routing is looked at.
template <int kW, bool kF16, int kR, int RF, int kWaves, int kDepth>
__global__ __launch_bounds__(kWaves * 64) void gate_up_kernel(const ExpertsArgs p, int by_pair, int run, int down_rows) {
    typedef StageOf<kW, RF, kR, (kW == kWFp8 ? 256 : 512)> St;
    constexpr int kRing = kDepth * St::kBytes, kSums = kWaves * RF * kR * 64;
    constexpr int kSmem = kWaves * kRing + kSums, kIds = kMaxTokens * kMaxTopk * 8;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kSmem > kIds ? kSmem : kIds];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), part = lane >> 4, r = lane & 15;
    if (blockIdx.x == 0) {
        write_passes<kWaves>(p, down_rows, reinterpret_cast<int*>(smem), reinterpret_cast<float*>(smem) + kMaxTokens * kMaxTopk);
        return;
    }
    const int tiles = p.I / (8 * RF), runs = (tiles + run - 1) / run, at = (int)blockIdx.x - 1, owner = at / runs;
    const int tile0 = (at - owner * runs) * run, ntiles = min(run, tiles - tile0), i0 = tile0 * 8 * RF;
    const int e = __builtin_amdgcn_readfirstlane(by_pair ? expert_of(p, owner) : owner);
    if (e < 0) return;

    // the expert's rows from the first gate row to the last up row
    const int ldw = kW == kWFp8 ? p.H : p.H / 2, lds = p.H / 32;
    const int units = (p.H + St::kK - 1) / St::kK, from = units * wave / kWaves, S = units * (wave + 1) / kWaves - from;
    const int64_t row0 = (int64_t)e * 2 * p.I + i0;
    const v4i dW = make_desc(p.w13 + row0 * ldw, (int64_t)(p.I + ntiles * 8 * RF) * ldw);
    const v4i dS = make_desc(static_cast<const uint8_t*>(p.s13) + row0 * lds, (int64_t)(p.I + ntiles * 8 * RF) * lds);
    const v4i dX = make_desc(p.x, ((int64_t)(p.T - 1) * p.ld_x + p.H) * 2);
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem + (uint32_t)wave * kRing;
    const uint8_t* const ring = smem + wave * kRing;

    // weight load j: rows 8 j .. 8 j + 7 of the stage's 16 RF, the gate's then the up's
    int voff[St::kWLoads];
#pragma unroll
    for (int j = 0; j < St::kWLoads; ++j) {
        const int q = 8 * j + (lane >> 3);
        voff[j] = (q < 8 * RF ? q : p.I + q - 8 * RF) * ldw + (((lane & 7) ^ swz(q)) << 4);
    }
    const int sq = lane >> 1;   // scale bytes: two lanes a row
    const int svoff = sq >= 16 * RF ? kOob : (sq < 8 * RF ? sq : p.I + sq - 8 * RF) * lds + (lane & 1) * 4;
    // this lane's chunks lie in the upper half of the stage: behind H at the end
    // of an H that is an odd multiple of 128 (MXFP4)
    const bool behind0 = ((lane & 7) ^ swz(lane >> 3)) >= 4, behind1 = ((lane & 7) ^ swz(8 + (lane >> 3))) >= 4;
    auto load_w = [&](uint32_t base, int tile, int s, bool none) KBN_INLINE {
        v4i w = dW, sc = dS;
        if (none) w[2] = sc[2] = 0;   // an empty load keeps the count of loads in flight
        const bool half = kW == kWMxfp4 && (from + s + 1) * St::kK > p.H;
        static_for<St::kWLoads>([&](auto j_) {
            constexpr int j = decltype(j_)::value;
            dma_b128<j * 1024, true>(w, base, half && (j & 1 ? behind1 : behind0) ? kOob : voff[j],
                                     tile * 8 * RF * ldw + (from + s) * 128);
        });
        if constexpr (St::kScaleLoads) dma_b32<St::kScaleAt>(sc, base, svoff, tile * 8 * RF * lds + (from + s) * 8);
    };
    const bool early = S >= kDepth;
    if (early)
        for (int s = 0; s < kDepth; ++s) load_w(lds0 + (uint32_t)s * St::kBytes, 0, s, false);

    // lane t: token t's first slot that names e
    int slot = -1;
    if (lane < p.T)
        for (int j = p.topk - 1; j >= 0; --j)
            if (expert_of(p, lane * p.topk + j) == e) slot = j;
    const uint64_t mask = __ballot(slot >= 0);
    const int first = mask ? __ffsll((unsigned long long)mask) - 1 : 0;
    const bool owned = mask != 0 && (!by_pair || first * p.topk + __shfl(slot, first) == owner);
    if (!owned) {      // nobody names e, or an earlier pair's workgroup has it
        wait_dma();    // loads in flight write to this workgroup's LDS
        return;
    }
    const int rows = __popcll(mask);
    // lane c: the token and slot of the expert's c-th row
    int token = 0;
    {
        uint64_t m = mask;
        for (int c = 0; c < lane && c < rows - 1; ++c) m &= m - 1;
        token = __ffsll((unsigned long long)m) - 1;
    }
    const int pair = token * p.topk + __shfl(slot, token);

    // the stage that is loaded next: tile lt, rows lr .. lr + kR - 1, stage ls
    int lt = 0, lr = 0, ls = 0;
    constexpr int kChunks = St::kK / 8;   // 16-byte chunks of an activation row
    int xoff[St::kXLoads];
    bool xbehind[St::kXLoads];
    auto set_rows = [&]() {
#pragma unroll
        for (int j = 0; j < St::kXLoads; ++j) {
            const int i = 64 * j + lane, q = i / kChunks, c = (i % kChunks) ^ q;
            const int t = __shfl(token, lr + q < rows ? lr + q : 0);
            xoff[j] = lr + q < rows ? t * (int)p.ld_x * 2 + c * 16 : kOob;
            xbehind[j] = c >= kChunks / 2;
        }
    };
    auto load_x = [&](uint32_t base, int s, bool none) KBN_INLINE {
        v4i x = dX;
        if (none) x[2] = 0;
        const int k = (from + s) * St::kK;
        const bool half = kW == kWMxfp4 && k + St::kK > p.H;
        static_for<St::kXLoads>([&](auto j_) {
            constexpr int j = decltype(j_)::value;
            dma_b128<St::kXAt + j * 1024, false>(x, base, half && xbehind[j] ? kOob : xoff[j], k * 2);
        });
    };
    auto advance = [&]() {
        if (++ls < S) return;
        ls = 0;
        lr += kR;
        if (lr >= rows) {
            lr = 0;
            ++lt;
        }
        if (rows > kR) set_rows();
    };
    auto issue = [&](int buf) KBN_INLINE {
        const uint32_t base = lds0 + (uint32_t)buf * St::kBytes;
        load_w(base, lt, ls, lt >= ntiles);
        load_x(base, ls, lt >= ntiles);
        advance();
    };
    set_rows();
    if (early) {
        for (int s = 0; s < kDepth; ++s) {
            load_x(lds0 + (uint32_t)s * St::kBytes, s, false);
            advance();
        }
    } else if (S) {
        for (int s = 0; s < kDepth; ++s) issue(s);
    }
    wait_dma_n<(kDepth - 1) * St::kXLoads>();   // the first stage, in either order

    int buf = 0, sums_at = 0;
    for (int tile = 0; tile < ntiles; ++tile) {
        const int i = i0 + tile * 8 * RF;
        const float* const s_gate = static_cast<const float*>(p.s13) + ((int64_t)e * 2 * p.I + i) / 128 * (p.H / 128);
        const float* const s_up = static_cast<const float*>(p.s13) + ((int64_t)e * 2 * p.I + p.I + i) / 128 * (p.H / 128);
        for (int r0 = 0; r0 < rows; r0 += kR) {
            v4f acc[RF] = {};
            for (int s = 0; s < S; ++s, buf = buf == kDepth - 1 ? 0 : buf + 1) {
                wait_dma_n<(kDepth - 1) * St::kLoads>();
                const uint8_t* const at = ring + buf * St::kBytes;
                u32x4 w[RF][2], x[2][St::kParts];
                uint32_t byte[RF][2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int f = 0; f < RF; ++f) {
                        w[f][j] = St::w(at, f, j, r, part);
                        byte[f][j] = St::scale(at, f, j, r, part);
                        // bytes behind H are another row's, perhaps a NaN's
                        if (kW == kWMxfp4 && j == 1 && (from + s + 1) * St::kK > p.H) byte[f][j] = 0;
                    }
#pragma unroll
                    for (int q = 0; q < St::kParts; ++q)   // k = 64 j + 16 part + 8 q, MXFP4 128 j + 32 part + 8 q
                        x[j][q] = St::x(at, r, (kW == kWFp8 ? 8 * j + 2 * part : 16 * j + 4 * part) + q);
                }
                const float f0 = kW == kWFp8 ? scalar_load(s_gate, from + s) : 0.0f, f1 = kW == kWFp8 ? scalar_load(s_up, from + s) : 0.0f;
                wait_lds();   // all of the stage is read: its buffer may be filled again
                issue(buf);
                constexpr bool kHalf = kF16 && kW == kWFp8, kPair = kF16 && !kHalf;
                bf16x8 hi[2][St::kParts], lo[2][St::kParts];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int q = 0; q < St::kParts; ++q) {
                        if constexpr (kPair) split8(__builtin_bit_cast(f16x8, x[j][q]), hi[j][q], lo[j][q]);
                        else hi[j][q] = __builtin_bit_cast(bf16x8, x[j][q]);
                    }
#pragma unroll
                for (int f = 0; f < RF; ++f) {
                    v4f t = kW == kWFp8 ? v4f{} : acc[f];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int q = 0; q < St::kParts; ++q) {
                            if constexpr (kHalf) {
                                t = mfma(widen_half(w[f][j], q), __builtin_bit_cast(f16x8, x[j][q]), t);
                            } else {
                                const bf16x8 a = widen_w<kW>(w[f][j], q, byte[f][j]);
                                t = mfma(a, hi[j][q], t);
                                if constexpr (kPair) t = mfma(a, lo[j][q], t);
                            }
                        }
                    if constexpr (kW == kWFp8) acc[f] += t * (RF == 1 ? (part < 2 ? f0 : f1) : f ? f1 : f0);
                    else acc[f] = t;
                }
            }
            // the wavefronts' sums meet: [wavefront][fragment][part][column] of
            // four rows each
            float* const sums = reinterpret_cast<float*>(smem + kWaves * kRing);
            if (r < kR) {
#pragma unroll
                for (int f = 0; f < RF; ++f)
                    *reinterpret_cast<v4f*>(sums + (((wave * RF + f) * 4 + part) * kR + r) * 4) = acc[f];
            }
            __syncthreads();
            // thread: column c, row q of h
            const int c = tid & 15, q = tid >> 4, row = __shfl(pair, min(r0 + c, 63));
            if (q < 8 * RF && r0 + c < rows && c < kR) {
                const int g_at = (q / 4 * kR + c) * 4 + q % 4, u_at = g_at + (RF == 1 ? 2 : 4) * kR * 4;
                float gate = 0.0f, up = 0.0f;
#pragma unroll
                for (int v = 0; v < kWaves; ++v) {
                    gate += sums[v * RF * kR * 16 + g_at];
                    up += sums[v * RF * kR * 16 + u_at];
                }
                const float y = gate / (1.0f + __expf(-gate)) * up;
                const __bf16 hi = (__bf16)y;
                uint16_t* h = p.h + ((int64_t)row * (p.I / 128) + (i + q) / 128) * 256 + (i + q) % 128;
                h[0] = __builtin_bit_cast(uint16_t, hi);
                h[128] = __builtin_bit_cast(uint16_t, low_part(y, hi));
            }
            __syncthreads();   // the sums are read
        }
    }
    wait_dma();
}

// Workgroup: `cols` output columns (at most 16 RF, a multiple of 4) of every
// token.  The stages of all passes form
// one sequence, cut into a run for each wavefront; a pass's sums are weighted
// and added to the wavefront's [T][16 RF] sums in LDS when the run leaves it, and
// the wavefronts' are added in their order at the end.
template <int kW, bool kF16, int kR, int RF, int kWaves, int kDepth>
__global__ __launch_bounds__(kWaves * 64) void down_kernel(const ExpertsArgs p, int cols) {
    typedef StageOf<kW, RF, kR, (kW == kWFp8 ? 512 : 1024)> St;
    constexpr int kRing = kDepth * St::kBytes, kCols = 16 * RF;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];   // rings, sums [kWaves][T][kCols], passes, rows
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), part = lane >> 4, r = lane & 15;
    float* const sums = reinterpret_cast<float*>(smem + kWaves * kRing);
    Pass* const passes = reinterpret_cast<Pass*>(sums + kWaves * p.T * kCols);
    Row* const rows = reinterpret_cast<Row*>(passes + p.T * p.topk);
    const int count = *p.count;
    for (int i = tid; i < p.T * p.topk; i += kWaves * 64) {
        passes[i] = p.passes[i];   // those behind the last hold anything and are not read
        rows[i] = p.rows[i];
    }
    for (int i = tid; i < kWaves * p.T * kCols; i += kWaves * 64) sums[i] = 0.0f;
    __syncthreads();
    float* const own = sums + wave * p.T * kCols;

    const int n0 = blockIdx.x * cols, n = min(cols, p.H - n0), units = (p.I + St::kK - 1) / St::kK;   // stages of a pass
    const int total = count * units;
    const int from = (int)((int64_t)total * wave / kWaves), S = (int)((int64_t)total * (wave + 1) / kWaves) - from;
    const int ldw = kW == kWFp8 ? p.I : p.I / 2, lds = p.I / 32;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem + (uint32_t)wave * kRing;
    const uint8_t* const ring = smem + wave * kRing;
    const v4i dH = make_desc(p.h, (int64_t)p.T * p.topk * p.I * 4);
    int voff[St::kWLoads];   // rows past the last are zeros
#pragma unroll
    for (int j = 0; j < St::kWLoads; ++j) {
        const int q = 8 * j + (lane >> 3);
        voff[j] = q < n ? q * ldw + (((lane & 7) ^ swz(q)) << 4) : kOob;
    }
    const int svoff = (lane >> 1) < n ? (lane >> 1) * lds + (lane & 1) * 4 : kOob;
    const bool behind0 = ((lane & 7) ^ swz(lane >> 3)) >= 4, behind1 = ((lane & 7) ^ swz(8 + (lane >> 3))) >= 4;

    // the stage that is loaded next: pass lp, stage lk of it
    int lp = from / units, lk = from - lp * units;
    v4i dW = {}, dS = {};
    int hoff[St::kXLoads];
    bool hbehind[St::kXLoads];
    constexpr int kChunks = St::kXLoads * 64 / kR;   // 16-byte chunks of an h row's stage
    auto enter = [&]() KBN_INLINE {
        const Pass v = passes[lp < count ? lp : count - 1];
        const int e = __builtin_amdgcn_readfirstlane(v.expert);
        const int64_t row0 = (int64_t)e * p.H + n0;
        dW = make_desc(p.w2 + row0 * ldw, (int64_t)n * ldw);
        if constexpr (kW == kWMxfp4) dS = make_desc(static_cast<const uint8_t*>(p.s2) + row0 * lds, (int64_t)n * lds);
#pragma unroll
        for (int j = 0; j < St::kXLoads; ++j) {
            const int i = 64 * j + lane, q = i / kChunks, c = (i % kChunks) ^ q;
            hoff[j] = q < v.rows ? rows[v.first_row + (q < v.rows ? q : 0)].pair * p.I * 4 + c * 16 : kOob;
            hbehind[j] = c >= kChunks / 2;
        }
    };
    auto issue = [&](auto buf_, int s) KBN_INLINE {
        constexpr int b = decltype(buf_)::value * St::kBytes;
        v4i w = dW, x = dH, sc = dS;
        if (s >= S) w[2] = x[2] = sc[2] = 0;
        const bool half = kW == kWMxfp4 && (lk + 1) * St::kK > p.I;
        static_for<St::kWLoads>([&](auto j_) {
            constexpr int j = decltype(j_)::value;
            dma_b128<b + j * 1024, true>(w, lds0, half && (j & 1 ? behind1 : behind0) ? kOob : voff[j], lk * 128);
        });
        static_for<St::kXLoads>([&](auto j_) {
            constexpr int j = decltype(j_)::value;
            dma_b128<b + St::kXAt + j * 1024, false>(x, lds0, half && hbehind[j] ? kOob : hoff[j], lk * St::kK * 4);
        });
        if constexpr (St::kScaleLoads) dma_b32<b + St::kScaleAt>(sc, lds0, svoff, lk * 8);
        if (s >= S) return;
        if (++lk == units) {
            lk = 0;
            ++lp;
            if (s + 1 < S) enter();
        }
    };

    // the stage in use: pass up, stage uk of it
    int up = lp, uk = lk;
    v4f acc[RF] = {};
    auto leave = [&]() {   // the pass's sums, weighted, to their tokens
        const Pass v = passes[up];
        if (r < v.rows) {
            const Row row = rows[v.first_row + r];
#pragma unroll
            for (int f = 0; f < RF; ++f) *reinterpret_cast<v4f*>(own + row.token * kCols + 16 * f + 4 * part) += acc[f] * row.weight;
        }
#pragma unroll
        for (int f = 0; f < RF; ++f) acc[f] = v4f{};
    };
    auto use = [&](auto buf_, int s) KBN_INLINE {
        constexpr int b = decltype(buf_)::value * St::kBytes;
        if (s >= S) return;
        const uint8_t* const at = ring + b;
        u32x4 w[RF][2], hi[2][St::kParts], lo[2][St::kParts];
        uint32_t byte[RF][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int f = 0; f < RF; ++f) {
                w[f][j] = St::w(at, f, j, r, part);
                byte[f][j] = St::scale(at, f, j, r, part);
                if (kW == kWMxfp4 && j == 1 && (uk + 1) * St::kK > p.I) byte[f][j] = 0;
            }
#pragma unroll
            for (int i = 0; i < St::kParts; ++i) {
                // 128 K of h: 16 chunks of high parts, then 16 of low ones
                const int c = kW == kWFp8 ? 8 * j + 2 * part + i : 32 * j + 4 * part + i;
                hi[j][i] = St::x(at, r, c);
                lo[j][i] = St::x(at, r, c + 16);
            }
        }
        float s0 = 1.0f, s1 = 1.0f;   // the scales of the first column's block and the last one's
        if constexpr (kW == kWFp8) {
            const int64_t row = (int64_t)__builtin_amdgcn_readfirstlane(passes[up].expert) * (p.H / 128);
            s0 = scalar_load(static_cast<const float*>(p.s2), (row + n0 / 128) * units + uk);
            if constexpr (RF == 2) s1 = scalar_load(static_cast<const float*>(p.s2), (row + (n0 + n - 1) / 128) * units + uk);
        }
        wait_lds();
        issue(buf_, s + kDepth);
#pragma unroll
        for (int f = 0; f < RF; ++f) {
            v4f t = kW == kWFp8 ? v4f{} : acc[f];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < St::kParts; ++i) {
                    const bf16x8 a = widen_w<kW>(w[f][j], i, byte[f][j]);
                    t = mfma(a, __builtin_bit_cast(bf16x8, hi[j][i]), t);
                    t = mfma(a, __builtin_bit_cast(bf16x8, lo[j][i]), t);
                }
            if constexpr (kW == kWFp8) acc[f] += t * (RF == 1 || n0 % 128 + 16 * f + 4 * part < 128 ? s0 : s1);
            else acc[f] = t;
        }
        if (++uk == units) {
            leave();
            uk = 0;
            ++up;
        }
    };
    if (S > 0) {
        enter();
        static_for<kDepth>([&](auto b_) { issue(b_, decltype(b_)::value); });
        for (int s = 0; s < S; s += kDepth)
            static_for<kDepth>([&](auto b_) {
                wait_dma_n<(kDepth - 1) * St::kLoads>();
                use(b_, s + decltype(b_)::value);
            });
        if (uk) leave();
    }
    wait_dma();
    __syncthreads();
    for (int i = tid; i < p.T * kCols; i += kWaves * 64) {
        if (i % kCols >= n) continue;
        float y = 0.0f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) y += sums[v * p.T * kCols + i];
        uint16_t* o = static_cast<uint16_t*>(p.out) + (int64_t)(i / kCols) * p.ld_out + n0 + i % kCols;
        if constexpr (kF16) *o = __builtin_bit_cast(uint16_t, (_Float16)y);
        else *o = __builtin_bit_cast(uint16_t, (__bf16)y);
    }
}

constexpr int kDepth = 2;   // stages in flight: more takes LDS that further workgroups use better (T = 5, MXFP4, 72 -> 79 us with 3)

template <int kW, int kR, int RF, int kWaves>
static size_t down_smem(const ExpertsArgs& p) {
    typedef StageOf<kW, RF, kR, (kW == kWFp8 ? 512 : 1024)> St;
    return kWaves * (kDepth * St::kBytes + p.T * 64 * RF) + p.T * p.topk * (sizeof(Pass) + sizeof(Row));
}
template <int kW, bool kF16, int kR, int RF, int kWaves>
static int launch_down(const ExpertsArgs& p, int cols, hipStream_t st) {
    down_kernel<kW, kF16, kR, RF, kWaves, kDepth>
        <<<(p.H + cols - 1) / cols, kWaves * 64, down_smem<kW, kR, RF, kWaves>(p), st>>>(p, cols);
    KBN_CHECK_LAUNCH("few_token_experts");
    return 0;
}

// active: experts named, on average over uniform routing.  Sixteen gate and
// sixteen up rows a workgroup, in runs of up to four such tiles where that
// leaves five workgroups a CU (a run's stages stream without a break: T = 5,
// MXFP4, runs of 1 / 2 / 4 80 / 75 / 74 us; T = 1 on an eighth 17 / 23 / 34); eight and
// eight where there would be fewer workgroups than 1.5 a CU (T = 1 on an eighth
// 16.5 us, T = 5 82.6), then with eight wavefronts if there is at most one a CU
// (15.6; T = 2 on a quarter 24.6 against 20.7 with four).
template <int kW, bool kF16, int kR>
static int launch_gate_up(const ExpertsArgs& p, double active, int down_rows, hipStream_t st) {
    const int pairs = p.T * p.topk, by_pair = pairs <= p.E, owners = by_pair ? pairs : p.E, cus = cu_count();
    const bool many = active * (p.I / 16) >= 1.5 * cus;
    if constexpr (kR == 16) {
        if (!many) return launch_gate_up<kW, kF16, 8>(p, active, down_rows, st);
    }
    if (many) {
        const int run = (int)std::max(1.0, std::min(4.0, std::round(active * (p.I / 16) / (5.0 * cus))));
        gate_up_kernel<kW, kF16, kR, 2, 4, kDepth><<<1 + owners * ((p.I / 16 + run - 1) / run), 256, 0, st>>>(p, by_pair, run, down_rows);
    } else if constexpr (kR < 16) {
        if (owners * (p.I / 8) > cus)
            gate_up_kernel<kW, kF16, kR, 1, 4, kDepth><<<1 + owners * (p.I / 8), 256, 0, st>>>(p, by_pair, 1, down_rows);
        else
            gate_up_kernel<kW, kF16, kR, 1, 8, kDepth><<<1 + owners * (p.I / 8), 512, 0, st>>>(p, by_pair, 1, down_rows);
    }
    KBN_CHECK_LAUNCH("few_token_experts");
    return 0;
}

// Rows of a pass: more hold more tokens of an expert, fewer leave LDS for more
// workgroups.  us of the layer, gate/up with 2 / 4 / 8 / 16: rows an expert 1.1
// (MXFP4) 75 / 77 / 80, 1.6 (MXFP4) 179 / 172 / 177, 2.3 (FP8) - / 1610 / 1532, 4 (MXFP4)
// 458 / 341 / 294 / 348, 4 (FP8) 439 with 8, 434 with 16, 8 (FP8) 357 and 290, (MXFP4)
// 270 and 236, 16 (FP8) 642 and 522, (MXFP4) 452 and 384.  Down with 2 / 4 / 8 / 16:
// 1.1 rows 70 / 71 / 78, 1.6 (FP8) 266 / 259 / 295, 2.3 (FP8) 1702 / 1475 / 1461 and,
// with an eighth of h's columns, 239 / 221 / 238, 4 (MXFP4) 362 / 313 / 294, (FP8) 439
// with 8, 439 with 16, 8 (FP8) 347 and 326, (MXFP4) 285 and 262, 16 (FP8) 642 and
// 560, (MXFP4) 452 and 411.
//
// Pass sizes go by uniform routing with every id inside [0, E).  Other routings give the
// same results from kernels for more or fewer rows than they have, us of 64 tokens,
// 8 a token, (7168, 2048), FP8 / MXFP4: 32 of 256 experts here and the other ids
// outside, 77 to 80 rows, 225 / 206 (16 rows a pass where an expert has two or
// three); all tokens on the same 8 of 256 experts 651 / 495, on 64 of them 810 / 577.
//
// Columns of a down workgroup: 16, but for an H between 16 and 32 columns a CU
// as many as give every CU one workgroup, in two fragments: with 16 columns
// H = 7168 has 448 workgroups, of which LDS lets a CU hold one, and reads h as
// often (64 tokens over 256 experts 1590 -> 1532 us, in MXFP4 1083 -> 976, over 64
// experts 402 -> 362; H = 5120 165 -> 148; H = 10240 the same 65 either way).
template <int kW, bool kF16>
static int launch_for(const ExpertsArgs& p, hipStream_t st) {
    const double active = p.E * (1.0 - pow(1.0 - std::min(1.0, (double)p.topk / p.E), p.T)), rows = p.T * p.topk / active;
    const int cus = cu_count();
    const bool wide = p.H > 16 * cus && p.H <= 32 * cus;
    const int cols = wide ? (p.H + 4 * cus - 1) / (4 * cus) * 4 : 16;
    constexpr size_t kLds = 160 * 1024;
    const bool fits4 = down_smem<kW, 4, 1, 8>(p) <= kLds || (wide && down_smem<kW, 4, 2, 6>(p) <= kLds);
    const int down = rows < 1.5 ? 2 : fits4 && rows < 3.0 ? 4 : rows < 6.0 ? 8 : 16;
    const int rc = rows < 2.0 ? launch_gate_up<kW, kF16, (kW == kWMxfp4 ? 2 : 4)>(p, active, down, st)
                   : rows < (kW == kWMxfp4 ? 6.0 : 3.0) ? launch_gate_up<kW, kF16, 8>(p, active, down, st)
                                                        : launch_gate_up<kW, kF16, 16>(p, active, down, st);
    if (rc) return rc;
    if (down == 2) {
        if (wide && down_smem<kW, 2, 2, 8>(p) <= kLds) return launch_down<kW, kF16, 2, 2, 8>(p, cols, st);
        return launch_down<kW, kF16, 2, 1, 8>(p, 16, st);
    }
    if (down == 4) {
        if (wide && down_smem<kW, 4, 2, 6>(p) <= kLds) return launch_down<kW, kF16, 4, 2, 6>(p, cols, st);
        return launch_down<kW, kF16, 4, 1, 8>(p, 16, st);
    }
    if (down == 8) {
        if (wide && down_smem<kW, 8, 2, 4>(p) <= kLds) return launch_down<kW, kF16, 8, 2, 4>(p, cols, st);
        return launch_down<kW, kF16, 8, 1, 4>(p, 16, st);
    }
    if constexpr (kW == kWFp8) {
        return wide ? launch_down<kW, kF16, 16, 2, 4>(p, cols, st) : launch_down<kW, kF16, 16, 1, 4>(p, 16, st);
    } else {
        if (wide && down_smem<kW, 16, 2, 3>(p) <= kLds) return launch_down<kW, kF16, 16, 2, 3>(p, cols, st);
        if (down_smem<kW, 16, 1, 4>(p) <= kLds) return launch_down<kW, kF16, 16, 1, 4>(p, 16, st);
        return launch_down<kW, kF16, 16, 1, 3>(p, 16, st);
    }
}

static int64_t list_bytes(int64_t T, int64_t topk) { return 256 + T * topk * (int64_t)(sizeof(Pass) + sizeof(Row)); }

}  // namespace kbn

using namespace kbn;

extern "C" int64_t kbn_few_token_experts_workspace_bytes(int64_t T, int64_t topk, int64_t I) {
    if (T < 0 || T > kMaxTokens || topk < 1 || topk > kMaxTopk || I < 0 || I >= (1LL << 31)) return 0;
    return list_bytes(T, topk) + T * topk * I * 4;
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
    KBN_CHECK_ARG(H > 0 && I > 0 && H % 128 == 0 && I % 128 == 0, "%s: H=%lld and I=%lld must be multiples of 128", what,
                  (long long)H, (long long)I);
    // offsets within an expert, within the activations and within h are 32-bit
    KBN_CHECK_ARG(H < (1 << 24) && I < (1 << 24) && (I + 128) * H < (1LL << 31) && T * topk * I * 4 < (1LL << 31) &&
                      E * (I / 8) < (1LL << 31),
                  "%s: H=%lld and I=%lld are too large", what, (long long)H, (long long)I);
    if (T == 0) return 0;
    KBN_CHECK_ARG(ld_x >= H && ld_x % 8 == 0 && x && aligned16(x), "%s: input rows must be 16-byte aligned", what);
    KBN_CHECK_ARG(ld_x < (1 << 24), "%s: input row stride %lld is too large", what, (long long)ld_x);
    KBN_CHECK_ARG(ld_out >= H && out && reinterpret_cast<uintptr_t>(out) % 2 == 0, "%s: output row stride %lld below H=%lld", what,
                  (long long)ld_out, (long long)H);
    KBN_CHECK_ARG(w13 && w2 && s13 && s2 && topk_weights && topk_ids, "%s: null pointer", what);
    KBN_CHECK_ARG(aligned16(w13) && aligned16(w2), "%s: weights must be 16-byte aligned", what);
    KBN_CHECK_ARG(reinterpret_cast<uintptr_t>(s13) % 4 == 0 && reinterpret_cast<uintptr_t>(s2) % 4 == 0,
                  "%s: weight scales must be 4-byte aligned", what);
    const int64_t need = kbn_few_token_experts_workspace_bytes(T, topk, I);
    KBN_CHECK_ARG(workspace_bytes >= need && aligned16(workspace) && workspace, "%s: workspace of %lld bytes needed, got %lld",
                  what, (long long)need, (long long)workspace_bytes);
    uint8_t* const ws = (uint8_t*)workspace;
    const ExpertsArgs p{x, ld_x, (const uint8_t*)w13, (const uint8_t*)w2, s13, s2, topk_ids, id_bytes == 8, topk_weights,
                        (int)T, (int)H, (int)I, (int)E, (int)topk, (int*)ws, (Pass*)(ws + 256),
                        (Row*)(ws + 256 + T * topk * sizeof(Pass)), (uint16_t*)(ws + list_bytes(T, topk)), out, ld_out};
    const hipStream_t st = (hipStream_t)stream;
    if (w_format == kWFp8) return x_dtype == kMxF16 ? launch_for<kWFp8, true>(p, st) : launch_for<kWFp8, false>(p, st);
    return x_dtype == kMxF16 ? launch_for<kWMxfp4, true>(p, st) : launch_for<kWMxfp4, false>(p, st);
}
