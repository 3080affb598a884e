// Low-rank adapters of many requests beside a shared projection:
//
//   out[t, :] = base[t, :] + scaling[a] * B_a (A_a x[t]),   a = ids[t]
//   out[t, :] = base[t, :]                                  for ids outside [0, L)
//
// A [L, R, K], B [L, N, R].  Two launches: h = A_a x (a long sum, K split over
// workgroups, fp32 partial sums [S, T, R]) and out (the partial sums added in
// order, so results do not depend on which workgroup ends first).
//
// Tokens go by windows, of 256 (of 64 where there are more than 63 adapters, so
// that few tokens share one).  A workgroup works on chunks of one adapter's tokens
// in a window, which need not be neighbours: a decode batch reads each adapter once
// a window, a window inside one prompt has one adapter and full chunks.  It finds its
// chunks by counting each adapter's tokens, a lane an adapter (adapter after adapter
// in order of appearance, each waits for the last: 5 us of 15 for 32 tokens of 24
// adapters), or in order of appearance where adapters are more than lanes.  Nothing
// has to be known of the ids on the host.
//
// Bound by rows, base and out for prompts: 4096 tokens of 8 adapters in runs, 7168 x
// 16384, rank 32: 25 to 43 us (134 MB of x at 3.1 to 5.4 TB/s, by what of it the
// memory-side cache holds) and 32 to 34 us (3.5 TB/s: the products of a strip are not all
// hidden behind the next one's loads).  A decode batch is bound by the chain of two
// launches (ids, list, rows; ids, list, h, B): 32 tokens of 24 adapters, 8192 x 8192,
// rank 16, 6 to 6.6 + 5.4 to 7 us.
//
// h enters the second product as the sum of two bf16 numbers, each rounded to nearest:
// off by 2^-17 at most, far below the output's own rounding (cut off instead, by up to
// 2^-15, always towards 0).  fp16 B is the sum of two as well, exactly, and all four
// products are added.
#include "row_stream.h"

#include <algorithm>

namespace kbn {
namespace {

constexpr int kChunk = 64;        // most tokens of one workgroup of the first launch
constexpr int kRankChunk = 64;    // ranks of one workgroup of the first launch
constexpr int kMaxSplits = 4;     // more gain nothing: the second launch reads them all back

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
    int splits;
    int slots1, slots2;  // workgroups a window that share its chunks, in each launch
    int blocks;          // 256-column blocks of a workgroup of the second launch
};

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ int lanes_up_to(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(v, d, 64);
        v += lane >= d ? o : 0;
    }
    return v;
}

// A window of kWords x 64 tokens (lane i has the adapter of token i of each 64; -1:
// none, -2: no token), and its chunks of at most kSize tokens of one adapter, by
// number.  kNone: the tokens without an adapter come too, as those of adapter -1.
// kMode 0: chunks in order of their adapters' appearance; 1 (64 tokens) and 2 (256):
// at most 63 adapters, in order of their numbers.
constexpr int kIndexed = 63;
constexpr int words_of(int mode) { return mode == 2 ? 4 : 1; }
template <int kMode, int kSize, bool kNone>
struct Window {
    static constexpr int kWords = words_of(kMode);
    int t0;
    int id[kWords];
    int count, end;           // by number: this lane's adapter's tokens, chunks up to it
    uint64_t left;            // by appearance: tokens whose adapter was not yet passed
    int passed;               // chunks of those that were
    uint64_t now[kWords];     // tokens of the chunk's adapter
    int adapter, from, n;     // it, and the chunk's tokens among them
    __device__ __forceinline__ Window(const LoraArgs& a, int w, int lane) {
        t0 = w * 64 * kWords;
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
            const int64_t t = t0 + 64 * k + lane;
            int64_t v = -1;
            if (t < a.T) v = a.id64 ? static_cast<const int64_t*>(a.ids)[t] : (int64_t)static_cast<const int32_t*>(a.ids)[t];
            id[k] = t >= a.T ? -2 : v >= 0 && v < a.L ? (int)v : -1;
        }
        if constexpr (kMode > 0) {
            count = 0;
#pragma unroll 4
            for (int l = kNone ? -1 : 0; l < a.L; ++l) {
                const int c = tokens_of(l);
                count = (lane == (l & 63)) ? c : count;   // (none: the last lane)
            }
            end = lanes_up_to((count + kSize - 1) / kSize, lane);
        } else {
            left = __ballot(id[0] >= (kNone ? -1 : 0));
            passed = 0;
        }
    }
    __device__ __forceinline__ int tokens_of(int l) const {
        int c = 0;
#pragma unroll
        for (int k = 0; k < kWords; ++k) c += (int)__builtin_popcountll(__ballot(id[k] == l));
        return c;
    }
    // Chunk p, numbers rising from call to call; false if there is none.
    __device__ __forceinline__ bool seek(int p) {
        int all;
        if constexpr (kMode > 0) {
            const uint64_t at = __ballot(end > p);
            if (!at) return false;
            const int l = (int)__builtin_ctzll(at);
            all = __builtin_amdgcn_readlane(count, l);
            from = (p - (__builtin_amdgcn_readlane(end, l) - (all + kSize - 1) / kSize)) * kSize;
            adapter = l == 63 ? -1 : l;
        } else {
            for (;;) {
                if (!left) return false;
                adapter = __builtin_amdgcn_readlane(id[0], (int)__builtin_ctzll(left));
                const uint64_t m = __ballot(id[0] == adapter);
                all = (int)__builtin_popcountll(m);
                const int chunks = (all + kSize - 1) / kSize;
                from = (p - passed) * kSize;
                if (p < passed + chunks) break;
                passed += chunks;
                left &= ~m;
            }
        }
        n = min(kSize, all - from);
#pragma unroll
        for (int k = 0; k < kWords; ++k) now[k] = __ballot(id[k] == adapter);
        return true;
    }
    // Writes the chunk's tokens as places in the window (one wavefront).
    __device__ __forceinline__ void list(int lane, uint8_t* to) const {
        int before = -from;
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
            const int at = before + (int)__builtin_popcountll(now[k] & ((1ull << lane) - 1));
            if ((now[k] >> lane & 1) && at >= 0 && at < n) to[at] = (uint8_t)(64 * k + lane);
            before += (int)__builtin_popcountll(now[k]);
        }
    }
};

// h[split, t, r0 ..] of n tokens of one adapter (lane i has the i-th's place in
// the window): kTM tiles of 16 tokens, kTR of 16 ranks.
template <int kD, int kTM, int kTR>
__device__ __forceinline__ void shrink_tile(const LoraArgs& a, int t0, int places, int n, int list, int adapter,
                                            int r0, int split, uint8_t* smem) {
    typedef Stream<kTM, kTR, 2, kD, kD> St;
    const int nr = min(16 * kTR, a.R - r0);
    const v4i dX = make_desc(static_cast<const uint8_t*>(a.x) + (int64_t)t0 * a.ld_x * 2,
                             ((int64_t)(min(places, a.T - t0) - 1) * a.ld_x + a.K) * 2);
    const v4i dA = make_desc(static_cast<const uint8_t*>(a.a) + ((int64_t)adapter * a.R + r0) * a.K * 2, (int64_t)nr * a.K * 2);
    const int units = (a.K + kStreamK - 1) / kStreamK;
    St::run(dX, dA, [&](int q) { const int t = __shfl(list, q, 64);
                        return q < n ? t * (int)a.ld_x * 2 : kOob; }, [&](int q) { return q < nr ? q * a.K * 2 : kOob; },
            a.K, units * split / a.splits, units * (split + 1) / a.splits, smem);
    float* h = a.h + (int64_t)split * a.T * a.R;
    for (int s = threadIdx.x; s < kTM * kTR * 64; s += 64 * kStreamWaves) {
        const f32x4 v = St::sum(smem, s);
        const int l = s & 63, tile = s >> 6;
        const int r = 16 * (tile % kTR) + (l & 15), t = 16 * (tile / kTR) + 4 * (l >> 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int token = __shfl(list, t + i, 64);
            if (r < nr && t + i < n) h[(int64_t)(t0 + token) * a.R + r0 + r] = v[i];
        }
    }
    __syncthreads();   // smem is used again by the next chunk
}

// grid (splits, windows, slots x rank chunks); chunks of kSize tokens
template <int kD, int kTR, int kMode, int kSize>
__global__ __launch_bounds__(64 * kStreamWaves) void lora_shrink_kernel(const LoraArgs a) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[Stream<kSize / 16, kTR, 2, kD, kD>::kSmem];
    const int lane = threadIdx.x & 63;
    const int parts = (a.R + kRankChunk - 1) / kRankChunk;
    const int r0 = blockIdx.z % parts * kRankChunk;
    Window<kMode, kSize, false> win(a, blockIdx.y, lane);
    for (int p = blockIdx.z / parts; win.seek(p); p += a.slots1) {
        if (threadIdx.x < 64) win.list(lane, smem);
        __syncthreads();
        const int n = win.n, list = smem[min(lane, n - 1)];
        __syncthreads();
        if (n <= 16) shrink_tile<kD, 1, kTR>(a, win.t0, 64 * words_of(kMode), n, list, win.adapter, r0, blockIdx.x, smem);
        else if (kSize == 32 || n <= 32) shrink_tile<kD, 2, kTR>(a, win.t0, 64 * words_of(kMode), n, list, win.adapter, r0, blockIdx.x, smem);
        else shrink_tile<kD, kSize / 16, kTR>(a, win.t0, 64 * words_of(kMode), n, list, win.adapter, r0, blockIdx.x, smem);
    }
}

__device__ __forceinline__ float value_of(int d, uint16_t v) {
    return d == kG16b ? __uint_as_float((uint32_t)v << 16) : (float)__builtin_bit_cast(_Float16, v);
}
__device__ __forceinline__ uint16_t value_to(int d, float f) {
    if (d == kG16b) return __builtin_bit_cast(uint16_t, (__bf16)f);
    return __builtin_bit_cast(uint16_t, (_Float16)f);
}

// Eight values of an fp16 row as two bf16 numbers each, cut off: 8 and 3 bits, exact.
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

// Eight fp32 values as two bf16 numbers each, rounded to nearest: what the first leaves
// is 2^-8 of the value at most, what the second leaves 2^-9 of that.  (The first is cut off
// where rounding would make an infinity of it.)
__device__ __forceinline__ void round8(const float (&f)[8], u32x4& hi, u32x4& lo) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x2 near = __builtin_convertvector((f32x2{f[2 * i], f[2 * i + 1]}), bf16x2);
        const uint32_t both = __builtin_bit_cast(uint32_t, near);
        float left[2];
        uint32_t first[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float v = f[2 * i + j];
            const uint32_t u = __float_as_uint(v), size = u & 0x7FFFFFFFu;
            first[j] = size < 0x7F7F8000u ? (j ? both & 0xFFFF0000u : both << 16) : u & 0xFFFF0000u;
            left[j] = size < 0x7F800000u ? v - __uint_as_float(first[j]) : 0.f;
        }
        hi[i] = __builtin_amdgcn_perm(first[1], first[0], 0x07060302u);
        lo[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{left[0], left[1]}), bf16x2));
    }
}

constexpr int kStrip = 64;                          // output columns of a wavefront
constexpr int kColumns = kStreamWaves * kStrip;     // of a workgroup's block
constexpr int kRows = 32;                           // tokens of one workgroup of the second launch
constexpr int kMaxRank = 256;

// A wavefront's LDS writes come before its reads that follow.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Four columns' values as they lie in memory with the adapter's added.
template <int kD>
__device__ __forceinline__ u32x2 added(const u32x2& was, float v0, float v1, float v2, float v3) {
    if constexpr (kD == kG16b) {
        const bf16x2 lo = __builtin_convertvector((f32x2{bf16lo(was.x) + v0, bf16hi(was.x) + v1}), bf16x2);
        const bf16x2 hi = __builtin_convertvector((f32x2{bf16lo(was.y) + v2, bf16hi(was.y) + v3}), bf16x2);
        return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const uint32_t a = was.x, b = was.y;
        const h2 wa = __builtin_bit_cast(h2, a), wb = __builtin_bit_cast(h2, b);
        const h2 lo{(_Float16)((float)wa.x + v0), (_Float16)((float)wa.y + v1)};
        const h2 hi{(_Float16)((float)wb.x + v2), (_Float16)((float)wb.y + v3)};
        return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
    }
}

// grid (column blocks, windows, slots).  Rows without an adapter are chunks too,
// and are copied (where out is not base itself).  A wavefront owns 64 columns
// of a block and all tokens of the chunk.  Tile j of its second operand holds
// columns 4 c + j, c = 0 .. 15, so a lane's results are four neighbouring columns
// of four tokens, and 16 lanes read and write whole lines of base and out; B's
// rows come straight into the matrix instruction's layout, once for all tokens;
// h comes from LDS, summed over the splits and cut in two by the workgroup.
// kKS: steps of 32 ranks whose rows of B are asked for ahead of h (0: any rank).
// kVec: base and out go four columns at a time.
template <int kD, int kKS, int kMode, bool kVec>
__global__ __launch_bounds__(64 * kStreamWaves) void lora_expand_kernel(const LoraArgs a) {
    constexpr int kRow = (kKS ? 32 * kKS : kMaxRank) + 8;   // values of a row of h: an odd number of 16-byte slots
    constexpr int kTM = kRows / 16;
    __shared__ __attribute__((aligned(16))) uint16_t part[2][kRows * kRow];
    __shared__ uint8_t places[kStreamWaves][kRows];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = lane & 15, q = lane >> 4;
    constexpr int kWords = words_of(kMode);
    Window<kMode, kRows, true> win(a, blockIdx.y, lane);
    const uint16_t* const base = static_cast<const uint16_t*>(a.base) + (int64_t)win.t0 * a.ld_b;
    uint16_t* const out = static_cast<uint16_t*>(a.out) + (int64_t)win.t0 * a.ld_o;
    const int rows = (int)min((int64_t)64 * kWords, (int64_t)a.T - win.t0);
    const __amdgpu_buffer_rsrc_t bi = rsrc(base, kVec ? (int)(((int64_t)(rows - 1) * a.ld_b + a.N) * 2) : 0);
    const __amdgpu_buffer_rsrc_t bo = rsrc(out, kVec ? (int)(((int64_t)(rows - 1) * a.ld_o + a.N) * 2) : 0);
    const int first = blockIdx.x * a.blocks * kColumns + wave * kStrip;
    // B: rows past N lie behind the descriptor, ranks past R are not asked for
    int wo[kKS ? kKS : 1];
#pragma unroll
    for (int k = 0; k < (kKS ? kKS : 1); ++k) wo[k] = 32 * k + 8 * q < a.R ? (4 * row * a.R + 32 * k + 8 * q) * 2 : kOob;
    uint8_t* const mine = places[wave];
    for (int p = blockIdx.z; win.seek(p); p += a.slots2) {
        const int n = win.n, tiles = (n + 15) / 16;
        const bool copy = win.adapter < 0;
        if (copy && a.base == a.out) continue;
        win.list(lane, mine);   // each wavefront for itself
        wave_lds_fence();
        const __amdgpu_buffer_rsrc_t br = rsrc(static_cast<const uint8_t*>(a.b) + (int64_t)win.adapter * a.N * a.R * 2,
                                               copy ? 0 : (int)((int64_t)a.N * a.R * 2));
        // h of the chunk's tokens, eight ranks of one a thread: asked for first,
        // as everything waits for it
        const int octets = (a.R + 31) / 32 * 4;
        const float sc = a.scaling && !copy ? a.scaling[win.adapter] : 1.f;
        f32x4 u[kMaxSplits][2];
        auto load_h = [&](int s) {
            const int i = s / octets, r = s % octets * 8;
            const bool in = i < n && r < a.R && !copy;
            const float* hp = a.h + (in ? (int64_t)(win.t0 + mine[i & (kRows - 1)]) * a.R + r : 0);
#pragma unroll
            for (int k = 0; k < kMaxSplits; ++k) {
                u[k][0] = u[k][1] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (k < a.splits && in) {
                    u[k][0] = *reinterpret_cast<const f32x4*>(hp + (int64_t)k * a.T * a.R);
                    u[k][1] = *reinterpret_cast<const f32x4*>(hp + (int64_t)k * a.T * a.R + 4);
                }
            }
        };
        // summed over the splits, scaled, cut in two; zeros past the rank and past the tokens
        auto put_h = [&](int s) {
            const int i = s / octets, r = s % octets * 8;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = u[0][j / 4][j & 3];
#pragma unroll
            for (int k = 1; k < kMaxSplits; ++k)
                if (k < a.splits) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] += u[k][j / 4][j & 3];
                }
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= sc;
            u32x4 hi, lo;
            round8(v, hi, lo);
            if (i < 16 * tiles) {
                *reinterpret_cast<u32x4*>(&part[0][i * kRow + r]) = hi;
                *reinterpret_cast<u32x4*>(&part[1][i * kRow + r]) = lo;
            }
        };
        if constexpr (kKS > 0) load_h(threadIdx.x);   // 32 tokens x 8 octets at most
        // a lane's tokens in base and out: 4 q + i of each 16 of the chunk
        int bo_at[kTM][4], oo_at[kTM][4];
#pragma unroll
        for (int m = 0; m < kTM; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 16 * m + 4 * q + i, t = mine[min(at, n - 1)];
                bo_at[m][i] = at < n ? (t * (int)a.ld_b + 4 * row) * 2 : kOob;
                oo_at[m][i] = at < n ? (t * (int)a.ld_o + 4 * row) * 2 : kOob;
            }
        struct Strip {
            u32x2 was[kTM][4];
            u32x4 w[kKS ? kKS : 1][4];
        };
        auto load_b = [&](int n0, int k, u32x4 (&to)[4]) __attribute__((always_inline)) {
            const int off = kKS ? wo[kKS ? k : 0] : 32 * k + 8 * q < a.R ? (4 * row * a.R + 32 * k + 8 * q) * 2 : kOob;
#pragma unroll
            for (int j = 0; j < 4; ++j) to[j] = __builtin_amdgcn_raw_buffer_load_b128(br, off, (n0 + j) * a.R * 2, 0);
        };
        auto ask = [&](int n0, Strip& t) __attribute__((always_inline)) {
            if constexpr (kKS > 0) {
#pragma unroll
                for (int k = 0; k < kKS; ++k) load_b(n0, k, t.w[k]);
            }
            // (past N a row's columns are the next row's: the last strip masks them.  No
            // non-temporal hints: base is mostly just written, x read by other products too;
            // 2048 tokens of 8 adapters, 10240 x 8192, warm 50.2 us, base with the hint 55.1)
            if constexpr (kVec) {
                const bool in = n0 + 4 * row < a.N;
#pragma unroll
                for (int m = 0; m < kTM; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        t.was[m][i] = __builtin_amdgcn_raw_buffer_load_b64(bi, in ? bo_at[m][i] : kOob, n0 * 2, 0);
            }
        };
        auto finish = [&](int n0, Strip& t) __attribute__((always_inline)) {
            f32x4 acc[kTM][4];
#pragma unroll
            for (int m = 0; m < kTM; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            auto step = [&](int kk, u32x4 (&b)[4]) __attribute__((always_inline)) {
                u32x4 bl[4];
                if constexpr (kD == kG16f) {   // as two bf16 numbers (exact): h may pass fp16's range
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float wf[8];
                        to_floats<kG16f>(Raw8<kG16f>{{b[j]}}, wf);
                        split8(wf, b[j], bl[j]);
                    }
                }
#pragma unroll
                for (int m = 0; m < kTM; ++m) {
                    if (m >= tiles) continue;
                    const u32x4 hh = *reinterpret_cast<const u32x4*>(&part[0][(16 * m + row) * kRow + 32 * kk + 8 * q]);
                    const u32x4 hl = *reinterpret_cast<const u32x4*>(&part[1][(16 * m + row) * kRow + 32 * kk + 8 * q]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if constexpr (kD == kG16f) {   // the smallest products first
                            acc[m][j] = mma<false>(hl, bl[j], acc[m][j]);
                            acc[m][j] = mma<false>(hh, bl[j], acc[m][j]);
                        }
                        acc[m][j] = mma<false>(hl, b[j], acc[m][j]);
                        acc[m][j] = mma<false>(hh, b[j], acc[m][j]);
                    }
                }
            };
            if constexpr (kKS > 0) {
#pragma unroll
                for (int kk = 0; kk < kKS; ++kk) step(kk, t.w[kk]);
            } else if (!copy) {
                for (int kk = 0; 32 * kk < a.R; ++kk) {
                    load_b(n0, kk, t.w[0]);
                    step(kk, t.w[0]);
                }
            }
            const int c = n0 + 4 * row;
#pragma unroll
            for (int m = 0; m < kTM; ++m) {
                if (m >= tiles) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (kVec) {
                        const u32x2 y = copy ? t.was[m][i] : added<kD>(t.was[m][i], acc[m][0][i], acc[m][1][i], acc[m][2][i], acc[m][3][i]);
                        __builtin_amdgcn_raw_buffer_store_b64(y, bo, c < a.N ? oo_at[m][i] : kOob, n0 * 2, 0);
                    } else if (16 * m + 4 * q + i < n) {
                        const int64_t at = mine[16 * m + 4 * q + i];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c + e < a.N) {
                                const uint16_t v = base[at * a.ld_b + c + e];
                                out[at * a.ld_o + c + e] = copy ? v : value_to(kD, value_of(kD, v) + acc[m][e][i]);
                            }
                    }
                }
            }
        };
        Strip one, two;
        ask(first, one);
        __syncthreads();   // part of the last chunk is done with
        if constexpr (kKS > 0) {
            put_h(threadIdx.x);
        } else {
            for (int s = threadIdx.x; s < 16 * tiles * octets; s += 64 * kStreamWaves) {
                load_h(s);
                put_h(s);
            }
        }
        __syncthreads();
        // the next strip is asked for before this one is done
        const int end = min(a.N, (int)(blockIdx.x + 1) * a.blocks * kColumns);
        for (int n0 = first; n0 < end; n0 += 2 * kColumns) {
            const int n1 = n0 + kColumns;
            if (n1 < end) ask(n1, two);
            finish(n0, one);
            if (n1 >= end) break;
            if (n1 + kColumns < end) ask(n1 + kColumns, one);
            finish(n1, two);
        }
    }
}

// How a window finds its chunks, workgroups a window that share its chunks in each
// launch, tokens of a chunk and K splits of the first and 256-column blocks of a
// workgroup of the second.
struct LoraPlan {
    int mode, windows, slots1, slots2, chunk, splits, blocks;
};
LoraPlan lora_plan(int64_t T, int64_t K, int64_t L, int64_t R, int64_t N) {
    LoraPlan p;
    // (up to eight tokens are passed one by one sooner than 24 adapters are counted)
    p.mode = L > kIndexed || T <= 8 ? 0 : T <= 64 ? 1 : 2;
    const int64_t tokens = 64 * words_of(p.mode);
    const int64_t size = std::min<int64_t>(T, tokens), cus = cu_count();
    p.windows = (int)((T + tokens - 1) / tokens);
    // chunks a window can have: full ones, and a last one of each adapter; in many
    // windows (prompts) mostly the full ones, and the rest waits its turn
    const int64_t adapters = std::min(L, size), last = p.windows > 2 ? std::min<int64_t>(adapters, 2) : adapters;
    const int64_t full1 = size / kChunk, full2 = size / kRows + 1;   // (and the tokens without an adapter)
    p.slots2 = (int)std::max<int64_t>(1, full2 + last);
    const int64_t parts = (R + kRankChunk - 1) / kRankChunk, units = (K + kStreamK - 1) / kStreamK;
    const int64_t busy = p.windows * std::max<int64_t>(std::max<int64_t>(1, full1), p.windows > 2 ? 1 : adapters * 2 / 3) * parts;
    const int64_t few = std::max<int64_t>(1, 65536 / (std::min<int64_t>(T, kRows) * R * 4));   // that a chunk reads back
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(cus + busy - 1) / busy, few, kMaxSplits, units / kStreamWaves}));
    // where chunks of 64 leave half of the CUs idle, chunks of 32 (777 tokens of runs
    // of 90, 4608 x 7168, rank 64: 23.8 us, with 64 26.1; 4096 tokens in runs of 700,
    // 7168 x 16384, rank 32, which 64 fill the CUs with: 72.9 and 69.0)
    p.chunk = p.mode == 2 && p.windows * full1 * parts * p.splits <= cus / 2 ? 32 : kChunk;
    p.slots1 = (int)std::max<int64_t>(1, size / p.chunk + last);
    // of the second launch's workgroups a CU holds two, and one takes about 5 us
    // whatever its columns: one round of them
    const int64_t cols = (N + kColumns - 1) / kColumns;
    const int64_t all = p.windows * std::min<int64_t>(p.slots2, (size + kRows - 1) / kRows + adapters);
    p.blocks = (int)std::max<int64_t>(1, std::min(cols, (all * cols + 2 * cus - 1) / (2 * cus)));
    return p;
}

template <int kD, int kMode, int kSize>
void launch_shrink(const LoraArgs& a, const dim3& grid, hipStream_t st) {
    const dim3 block(64 * kStreamWaves);
    if (a.R <= 16) lora_shrink_kernel<kD, 1, kMode, kSize><<<grid, block, 0, st>>>(a);
    else if (a.R <= 32) lora_shrink_kernel<kD, 2, kMode, kSize><<<grid, block, 0, st>>>(a);
    else lora_shrink_kernel<kD, 4, kMode, kSize><<<grid, block, 0, st>>>(a);
}
template <int kD, int kMode>
void launch_lora(const LoraArgs& a, const LoraPlan& p, bool vec, hipStream_t st) {
    const int parts = (a.R + kRankChunk - 1) / kRankChunk;
    const dim3 grid((unsigned)a.splits, (unsigned)p.windows, (unsigned)(a.slots1 * parts)), block(64 * kStreamWaves);
    if constexpr (kMode == 2) p.chunk == 32 ? launch_shrink<kD, kMode, 32>(a, grid, st) : launch_shrink<kD, kMode, kChunk>(a, grid, st);
    else launch_shrink<kD, kMode, kChunk>(a, grid, st);
    const int cols = kColumns * a.blocks;
    const dim3 egrid((unsigned)((a.N + cols - 1) / cols), (unsigned)p.windows, (unsigned)a.slots2);
    if (!vec) lora_expand_kernel<kD, 0, kMode, false><<<egrid, block, 0, st>>>(a);
    else if (a.R <= 32) lora_expand_kernel<kD, 1, kMode, true><<<egrid, block, 0, st>>>(a);
    else if (a.R <= 64) lora_expand_kernel<kD, 2, kMode, true><<<egrid, block, 0, st>>>(a);
    else lora_expand_kernel<kD, 0, kMode, true><<<egrid, block, 0, st>>>(a);
}

}  // namespace
}  // namespace kbn

using namespace kbn;

extern "C" int64_t kbn_lora_add_workspace_bytes(int64_t T, int64_t K, int64_t L, int64_t R) {
    if (T < 0 || T > 65535LL * 64 || K < 8 || K % 8 || L < 1 || R < 8 || R % 8 || R > kMaxRank) return -1;
    if (T == 0) return 0;
    return (int64_t)lora_plan(T, K, L, R, 1).splits * T * R * 4;
}

extern "C" int kbn_lora_add(const void* x, int dtype, int64_t ld_x, const void* base, int64_t ld_base, const void* lora_a,
                            const void* lora_b, const void* ids, int id_bytes, const float* scaling, int64_t T, int64_t N,
                            int64_t K, int64_t L, int64_t R, void* out, int64_t ld_out, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    const char* what = "lora_add";
    KBN_CHECK_ARG(dtype == kG16b || dtype == kG16f, "%s: dtype code %d (0 bf16, 1 fp16)", what, dtype);
    KBN_CHECK_ARG(id_bytes == 4 || id_bytes == 8, "%s: ids of %d bytes (4 or 8)", what, id_bytes);
    KBN_CHECK_ARG(T >= 0 && T <= 65535LL * 64 && N >= 1 && L >= 1 && L <= 0x7FFFFFFF, "%s: bad sizes T=%lld, N=%lld, L=%lld",
                  what, (long long)T, (long long)N, (long long)L);
    KBN_CHECK_ARG(K >= 8 && K % 8 == 0 && K <= (1 << 22), "%s: K=%lld must be a multiple of 8 in [8, 2^22]", what, (long long)K);
    KBN_CHECK_ARG(R >= 8 && R % 8 == 0 && R <= kMaxRank, "%s: rank %lld must be a multiple of 8 in [8, %d]", what, (long long)R,
                  kMaxRank);
    KBN_CHECK_ARG((N + kColumns) * R * 2 < 0x7FFFFFFFLL, "%s: an adapter's B [%lld, %lld] is too large", what,
                  (long long)N, (long long)R);
    if (T == 0) return 0;
    KBN_CHECK_ARG(x && base && lora_a && lora_b && ids && out, "%s: null pointer", what);
    KBN_CHECK_ARG(aligned16(x) && aligned16(lora_a) && aligned16(lora_b) && ld_x >= K && ld_x % 8 == 0,
                  "%s: rows and adapters must be 16-byte aligned, the rows' stride at least K", what);
    KBN_CHECK_ARG(ld_x < (1 << 22), "%s: row stride must be below 2^22 elements", what);
    KBN_CHECK_ARG(ld_base >= N && ld_out >= N, "%s: base and output rows' strides must be at least N", what);
    KBN_CHECK_ARG(base != out || ld_base == ld_out, "%s: in place, base and output must have one stride", what);
    const LoraPlan p = lora_plan(T, K, L, R, N);
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
    a.slots1 = p.slots1;
    a.slots2 = p.slots2;
    a.blocks = p.blocks;
    const auto aligned8 = [](const void* v) { return (reinterpret_cast<uintptr_t>(v) & 7u) == 0; };
    const bool vec = N % 4 == 0 && aligned8(base) && aligned8(out) && ld_base % 4 == 0 && ld_out % 4 == 0 && ld_base < (1 << 22) &&
            ld_out < (1 << 22);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == kG16b) {
        if (p.mode == 0) launch_lora<kG16b, 0>(a, p, vec, st);
        else if (p.mode == 1) launch_lora<kG16b, 1>(a, p, vec, st);
        else launch_lora<kG16b, 2>(a, p, vec, st);
    } else {
        if (p.mode == 0) launch_lora<kG16f, 0>(a, p, vec, st);
        else if (p.mode == 1) launch_lora<kG16f, 1>(a, p, vec, st);
        else launch_lora<kG16f, 2>(a, p, vec, st);
    }
    KBN_CHECK_LAUNCH(what);
    return 0;
}
