// Low-rank adapters of many requests beside a shared projection:
//
//   out[t, :] = base[t, :] + scaling[a] * B_a (A_a x[t]),   a = ids[t]
//   out[t, :] = base[t, :]                                  for ids outside [0, L)
//
// A [L, R, K], B [L, N, R].  Two launches: h = A_a x (a long sum, K split over
// workgroups, fp32 partial sums [S, T, R]) and out (the partial sums added in
// order, so results do not depend on which workgroup ends first).
//
// Tokens go by windows of 64.  In a window, slot s is its s-th adapter in
// order of appearance, and a workgroup works on the tokens of one slot: a
// decode batch in which every request has its own adapter reads each adapter
// once, a window inside one prompt has one slot of 64 tokens.  Nothing has to
// be known of the ids on the host.
//
// h enters the second product as the sum of two bf16 numbers (16 bits of its
// significand, 2^-16 of the value lost, far below the output's own rounding).
#include "kbn_common.h"

#include <algorithm>

namespace kbn {
namespace {

constexpr int kWindow = 64;       // tokens
constexpr int kLoraWaves = 4;
constexpr int kRankChunk = 64;    // ranks of one shrink workgroup
constexpr int kUnit = 64;         // K of one step
constexpr int kMaxSplits = 16;

enum : int { kLBf16 = 0, kLF16 = 1 };

struct LoraArgs {
    const void* x;
    int64_t ld_x;
    const void* base;
    int64_t ld_b;
    const void* a;       // [L, R, K]
    const void* b;       // [L, N, R]
    const void* ids;
    int id64;
    const float* scaling;   // nullptr: 1
    int T, N, K, L, R;
    void* out;
    int64_t ld_o;
    float* h;            // [splits, T, R]
    int splits, slots;   // slots: workgroups a window
    int vec;             // rows of base and out take 16-byte accesses
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, (int)kRsrcWord3);
}
__device__ __forceinline__ f32x4 mma_bf16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma_f16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A window's tokens: lane i's adapter (-1: none), and the adapters in order of appearance.
struct Window {
    int t0, n;
    int64_t id;
    uint64_t left;   // tokens whose adapter was not yet taken
    __device__ __forceinline__ Window(const LoraArgs& a, int w, int lane) {
        t0 = w * kWindow;
        n = min(kWindow, a.T - t0);
        id = -1;
        if (lane < n)
            id = a.id64 ? static_cast<const int64_t*>(a.ids)[t0 + lane] : (int64_t)static_cast<const int32_t*>(a.ids)[t0 + lane];
        if (id >= a.L) id = -1;
        left = __ballot(id >= 0);
    }
    // The next adapter and its tokens; false if there is none.
    __device__ __forceinline__ bool next(int& adapter, uint64_t& tokens) {
        if (!left) return false;
        adapter = __builtin_amdgcn_readlane((int)id, (int)__builtin_ctzll(left));
        tokens = __ballot((int)id == adapter && id >= 0);
        left &= ~tokens;
        return true;
    }
};
// Writes the positions of the set bits in order.
__device__ __forceinline__ void list_tokens(uint64_t tokens, int lane, uint8_t* list) {
    if (tokens >> lane & 1) list[__builtin_popcountll(tokens & ((1ull << lane) - 1))] = (uint8_t)lane;
}

// h[split, t, r0 ..] of one slot's tokens: kTM tiles of 16 tokens, kTR of 16 ranks.
template <int kD, int kTM, int kTR>
__device__ __forceinline__ void shrink_tile(const LoraArgs& a, int t0, int n, const uint8_t* list, int adapter, int r0,
                                            int split, f32x4* part) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = lane & 15, q = lane >> 4;
    const int nr = min(16 * kTR, a.R - r0);
    const __amdgpu_buffer_rsrc_t xr = rsrc(static_cast<const uint8_t*>(a.x) + (int64_t)t0 * a.ld_x * 2,
                                           (int)(((int64_t)(min(kWindow, a.T - t0) - 1) * a.ld_x + a.K) * 2));
    const __amdgpu_buffer_rsrc_t ar =
        rsrc(static_cast<const uint8_t*>(a.a) + ((int64_t)adapter * a.R + r0) * a.K * 2, (int)((int64_t)nr * a.K * 2));
    int xo[kTM], ao[kTR];
#pragma unroll
    for (int i = 0; i < kTM; ++i) xo[i] = 16 * i + row < n ? (list[16 * i + row] * (int)a.ld_x + 16 * q) * 2 : kOob;
#pragma unroll
    for (int j = 0; j < kTR; ++j) ao[j] = 16 * j + row < nr ? ((16 * j + row) * a.K + 16 * q) * 2 : kOob;
    constexpr int kDepth = 2;
    u32x4 xb[kDepth][kTM][2], ab[kDepth][kTR][2];
    auto load = [&](int d, int u) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const bool in = u * kUnit + 16 * q + 8 * s < a.K;
#pragma unroll
            for (int i = 0; i < kTM; ++i)
                xb[d][i][s] = __builtin_amdgcn_raw_buffer_load_b128(xr, in && xo[i] >= 0 ? xo[i] + (u * kUnit + 8 * s) * 2 : kOob, 0, 0);
#pragma unroll
            for (int j = 0; j < kTR; ++j)
                ab[d][j][s] = __builtin_amdgcn_raw_buffer_load_b128(ar, in && ao[j] >= 0 ? ao[j] + (u * kUnit + 8 * s) * 2 : kOob, 0, 0);
        }
    };
    f32x4 acc[kTM][kTR];
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
        for (int j = 0; j < kTR; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int units = (a.K + kUnit - 1) / kUnit, per = (units + a.splits - 1) / a.splits;
    const int end = min(units, (split + 1) * per);
    // units past this split's end read zeros
    auto load_in = [&](int d, int u) { load(d, u < end ? u : units); };
#pragma unroll
    for (int d = 0; d < kDepth; ++d) load_in(d, split * per + wave + d * kLoraWaves);
    for (int u = split * per + wave; u < end; u += kLoraWaves * kDepth) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < kTM; ++i)
#pragma unroll
                    for (int j = 0; j < kTR; ++j)
                        acc[i][j] = kD == kLBf16 ? mma_bf16(xb[d][i][s], ab[d][j][s], acc[i][j])
                                                 : mma_f16(xb[d][i][s], ab[d][j][s], acc[i][j]);
            load_in(d, u + (d + kDepth) * kLoraWaves);
        }
    }
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
        for (int j = 0; j < kTR; ++j) part[((wave * kTM + i) * kTR + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    float* h = a.h + (int64_t)split * a.T * a.R;
    for (int s = threadIdx.x; s < kTM * kTR * 64; s += 64 * kLoraWaves) {
        f32x4 v = part[s];
#pragma unroll
        for (int w = 1; w < kLoraWaves; ++w) v += part[w * kTM * kTR * 64 + s];
        const int l = s & 63, tile = s >> 6;
        const int r = 16 * (tile % kTR) + (l & 15), t = 16 * (tile / kTR) + 4 * (l >> 4);
        if (r < nr) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (t + i < n) h[(int64_t)(t0 + list[t + i]) * a.R + r0 + r] = v[i];
        }
    }
    __syncthreads();   // part and list are used again by the next slot
}

// grid (splits, windows, slots x rank chunks)
template <int kD, int kTR>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_shrink_kernel(const LoraArgs a) {
    __shared__ f32x4 part[kLoraWaves * 4 * kTR * 64];
    __shared__ uint8_t list[kWindow];
    const int lane = threadIdx.x & 63;
    const int chunks = (a.R + kRankChunk - 1) / kRankChunk;
    const int first = blockIdx.z / chunks, r0 = blockIdx.z % chunks * kRankChunk;
    Window win(a, blockIdx.y, lane);
    int adapter;
    uint64_t tokens;
    for (int slot = 0; win.next(adapter, tokens); ++slot) {
        if (slot % a.slots != first) continue;
        if (threadIdx.x < 64) list_tokens(tokens, lane, list);
        __syncthreads();
        const int n = __builtin_popcountll(tokens);
        if (n <= 16) shrink_tile<kD, 1, kTR>(a, win.t0, n, list, adapter, r0, blockIdx.x, part);
        else if (n <= 32) shrink_tile<kD, 2, kTR>(a, win.t0, n, list, adapter, r0, blockIdx.x, part);
        else shrink_tile<kD, 4, kTR>(a, win.t0, n, list, adapter, r0, blockIdx.x, part);
    }
}

__device__ __forceinline__ float value_of(int d, uint16_t v) {
    return d == kLBf16 ? __uint_as_float((uint32_t)v << 16) : (float)__builtin_bit_cast(_Float16, v);
}
__device__ __forceinline__ uint16_t value_to(int d, float f) {
    if (d == kLBf16) return __builtin_bit_cast(uint16_t, (__bf16)f);
    return __builtin_bit_cast(uint16_t, (_Float16)f);
}

// Eight fp32 values as two bf16 numbers each, cut off (their sum is off by 2^-16 at most).
__device__ __forceinline__ void split8(const float (&f)[8], u32x4& hi, u32x4& lo) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = __float_as_uint(f[2 * i]), b = __float_as_uint(f[2 * i + 1]);
        hi[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        const bool fa = (a & 0x7F800000u) != 0x7F800000u, fb = (b & 0x7F800000u) != 0x7F800000u;
        const uint32_t la = fa ? __float_as_uint(f[2 * i] - __uint_as_float(a & 0xFFFF0000u)) : 0u;
        const uint32_t lb = fb ? __float_as_uint(f[2 * i + 1] - __uint_as_float(b & 0xFFFF0000u)) : 0u;
        lo[i] = __builtin_amdgcn_perm(lb, la, 0x07060302u);
    }
}

constexpr int kStrip = 64;                          // output columns of a wavefront
constexpr int kColumns = kLoraWaves * kStrip;       // of a workgroup
constexpr int kMaxRank = 256;

// grid (column blocks, windows, slots + 1): the last slot copies the rows that
// have no adapter (where out is not base itself).
template <int kD>
__global__ __launch_bounds__(64 * kLoraWaves) void lora_expand_kernel(const LoraArgs a) {
    __shared__ uint8_t list[kWindow];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * kColumns + wave * kStrip;
    const uint16_t* const base = static_cast<const uint16_t*>(a.base);
    uint16_t* const out = static_cast<uint16_t*>(a.out);
    Window win(a, blockIdx.y, lane);
    if ((int)blockIdx.z == a.slots) {
        if (a.base == a.out) return;
        uint64_t rows = ~win.left & (win.n == 64 ? ~0ull : (1ull << win.n) - 1);
        const int n = n0 + lane;
        for (; rows; rows &= rows - 1) {
            const int64_t t = win.t0 + __builtin_ctzll(rows);
            if (n < a.N) out[t * a.ld_o + n] = base[t * a.ld_b + n];
        }
        return;
    }
    const int row = lane & 15, q = lane >> 4;
    int adapter;
    uint64_t tokens;
    for (int slot = 0; win.next(adapter, tokens); ++slot) {
        if (slot % a.slots != (int)blockIdx.z) continue;
        __syncthreads();
        if (threadIdx.x < 64) list_tokens(tokens, lane, list);
        __syncthreads();
        const int n = __builtin_popcountll(tokens);
        const float sc = a.scaling ? a.scaling[adapter] : 1.f;
        const uint8_t* bp = static_cast<const uint8_t*>(a.b) + (int64_t)adapter * a.N * a.R * 2;
        const __amdgpu_buffer_rsrc_t br = rsrc(bp, (int)((int64_t)a.N * a.R * 2));
        for (int i = 0; 16 * i < n; ++i) {
            const int at = 16 * i + row;
            const int64_t t = win.t0 + list[min(at, n - 1)];   // this lane's token
            f32x4 acc[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < a.R; k += 32) {
                const int r = k + 8 * q;
                float hv[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) hv[j] = 0.f;
                if (r < a.R && at < n) {
                    const float* hp = a.h + t * a.R + r;
                    for (int s = 0; s < a.splits; ++s, hp += (int64_t)a.T * a.R) {
                        const f32x4 u = *reinterpret_cast<const f32x4*>(hp), v = *reinterpret_cast<const f32x4*>(hp + 4);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            hv[j] += u[j];
                            hv[4 + j] += v[j];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) hv[j] *= sc;
                }
                u32x4 hh, hl;
                split8(hv, hh, hl);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // row m of tile j is column 16 (m / 4) + 4 j + m % 4 of the strip,
                    // so that a lane's results are 16 columns in a row
                    const int col = n0 + 16 * (row >> 2) + 4 * j + (row & 3);
                    const int off = r < a.R && col < a.N ? (col * a.R + r) * 2 : kOob;
                    u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(br, off, 0, 0);
                    if constexpr (kD == kLBf16) {
                        acc[j] = mma_bf16(w, hl, acc[j]);
                        acc[j] = mma_bf16(w, hh, acc[j]);
                    } else {   // fp16 as two bf16 numbers (exact): h may pass fp16's range
                        float wf[8];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            wf[2 * e] = value_of(kLF16, (uint16_t)w[e]);
                            wf[2 * e + 1] = value_of(kLF16, (uint16_t)(w[e] >> 16));
                        }
                        u32x4 wl;
                        split8(wf, w, wl);
                        acc[j] = mma_bf16(wl, hh, acc[j]);
                        acc[j] = mma_bf16(w, hl, acc[j]);
                        acc[j] = mma_bf16(w, hh, acc[j]);
                    }
                }
            }
            if (at < n) {
                const int c0 = n0 + 16 * q;
                const uint16_t* bi = base + t * a.ld_b + c0;
                uint16_t* o = out + t * a.ld_o + c0;
#pragma unroll
                for (int g = 0; g < 2; ++g) {   // eight columns each
                    if (a.vec && c0 + 8 * g + 8 <= a.N) {
                        const u32x4 v = *reinterpret_cast<const u32x4*>(bi + 8 * g);
                        u32x4 y;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float lo = value_of(kD, (uint16_t)v[e]) + acc[2 * g + e / 2][2 * (e & 1)];
                            const float hi = value_of(kD, (uint16_t)(v[e] >> 16)) + acc[2 * g + e / 2][2 * (e & 1) + 1];
                            y[e] = (uint32_t)value_to(kD, lo) | (uint32_t)value_to(kD, hi) << 16;
                        }
                        *reinterpret_cast<u32x4*>(o + 8 * g) = y;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (c0 + 8 * g + e < a.N)
                                o[8 * g + e] = value_to(kD, value_of(kD, bi[8 * g + e]) + acc[2 * g + e / 4][e & 3]);
                    }
                }
            }
        }
    }
}

// K splits and slots a window of a batch.
struct LoraPlan {
    int windows, splits, slots;
};
LoraPlan lora_plan(int64_t T, int64_t K, int64_t L, int64_t R) {
    LoraPlan p;
    p.windows = (int)((T + kWindow - 1) / kWindow);
    p.slots = (int)std::min<int64_t>({L, T, kWindow});
    if (p.windows > 4) p.slots = std::min(p.slots, 2);
    const int64_t chunks = (R + kRankChunk - 1) / kRankChunk;
    const int64_t units = (K + kUnit - 1) / kUnit;
    const int64_t want = std::max<int64_t>(1, 512 / (p.windows * chunks));
    p.splits = (int)std::min<int64_t>({want, kMaxSplits, std::max<int64_t>(1, units / kLoraWaves)});
    return p;
}

template <int kD>
void launch_lora(const LoraArgs& a, int windows, hipStream_t st) {
    const int chunks = (a.R + kRankChunk - 1) / kRankChunk;
    const dim3 grid((unsigned)a.splits, (unsigned)windows, (unsigned)(a.slots * chunks)), block(64 * kLoraWaves);
    if (a.R <= 16) lora_shrink_kernel<kD, 1><<<grid, block, 0, st>>>(a);
    else if (a.R <= 32) lora_shrink_kernel<kD, 2><<<grid, block, 0, st>>>(a);
    else lora_shrink_kernel<kD, 4><<<grid, block, 0, st>>>(a);
    const dim3 egrid((unsigned)((a.N + kColumns - 1) / kColumns), (unsigned)windows, (unsigned)(a.slots + 1));
    lora_expand_kernel<kD><<<egrid, block, 0, st>>>(a);
}

}  // namespace
}  // namespace kbn

using namespace kbn;

extern "C" int64_t kbn_lora_add_workspace_bytes(int64_t T, int64_t K, int64_t L, int64_t R) {
    if (T < 0 || T > 65535LL * kWindow || K < 8 || K % 8 || L < 1 || R < 8 || R % 8 || R > kMaxRank) return -1;
    if (T == 0) return 0;
    return (int64_t)lora_plan(T, K, L, R).splits * T * R * 4;
}

extern "C" int kbn_lora_add(const void* x, int dtype, int64_t ld_x, const void* base, int64_t ld_base, const void* lora_a,
                            const void* lora_b, const void* ids, int id_bytes, const float* scaling, int64_t T, int64_t N,
                            int64_t K, int64_t L, int64_t R, void* out, int64_t ld_out, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    const char* what = "lora_add";
    KBN_CHECK_ARG(dtype == kLBf16 || dtype == kLF16, "%s: dtype code %d (0 bf16, 1 fp16)", what, dtype);
    KBN_CHECK_ARG(id_bytes == 4 || id_bytes == 8, "%s: ids of %d bytes (4 or 8)", what, id_bytes);
    KBN_CHECK_ARG(T >= 0 && T <= 65535LL * kWindow && N >= 1 && L >= 1 && L <= 0x7FFFFFFF, "%s: bad sizes T=%lld, N=%lld, L=%lld",
                  what, (long long)T, (long long)N, (long long)L);
    KBN_CHECK_ARG(K >= 8 && K % 8 == 0 && K <= (1 << 22), "%s: K=%lld must be a multiple of 8 in [8, 2^22]", what, (long long)K);
    KBN_CHECK_ARG(R >= 8 && R % 8 == 0 && R <= kMaxRank, "%s: rank %lld must be a multiple of 8 in [8, %d]", what, (long long)R,
                  kMaxRank);
    KBN_CHECK_ARG(N * R * 2 < 0x7FFFFFFFLL && N <= 65535LL * kColumns, "%s: an adapter's B [%lld, %lld] is too large", what,
                  (long long)N, (long long)R);
    if (T == 0) return 0;
    KBN_CHECK_ARG(x && base && lora_a && lora_b && ids && out, "%s: null pointer", what);
    KBN_CHECK_ARG(aligned16(x) && aligned16(lora_a) && aligned16(lora_b) && ld_x >= K && ld_x % 8 == 0,
                  "%s: rows and adapters must be 16-byte aligned, the rows' stride at least K", what);
    KBN_CHECK_ARG(ld_x < (1 << 23), "%s: row stride must be below 2^23 elements", what);
    KBN_CHECK_ARG(ld_base >= N && ld_out >= N, "%s: base and output rows' strides must be at least N", what);
    KBN_CHECK_ARG(base != out || ld_base == ld_out, "%s: in place, base and output must have one stride", what);
    const LoraPlan p = lora_plan(T, K, L, R);
    KBN_CHECK_ARG(workspace && workspace_bytes >= (int64_t)p.splits * T * R * 4 && aligned16(workspace),
                  "%s: workspace of %lld bytes, 16-byte aligned, needed", what, (long long)((int64_t)p.splits * T * R * 4));
    LoraArgs a{};
    a.x = x;
    a.ld_x = ld_x;
    a.base = base;
    a.ld_b = ld_base;
    a.a = lora_a;
    a.b = lora_b;
    a.ids = ids;
    a.id64 = id_bytes == 8;
    a.scaling = scaling;
    a.T = (int)T;
    a.N = (int)N;
    a.K = (int)K;
    a.L = (int)L;
    a.R = (int)R;
    a.out = out;
    a.ld_o = ld_out;
    a.h = static_cast<float*>(workspace);
    a.splits = p.splits;
    a.slots = p.slots;
    a.vec = aligned16(base) && aligned16(out) && ld_base % 8 == 0 && ld_out % 8 == 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == kLBf16) launch_lora<kLBf16>(a, p.windows, st);
    else launch_lora<kLF16>(a, p.windows, st);
    KBN_CHECK_LAUNCH(what);
    return 0;
}
