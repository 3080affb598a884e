// Products of two sets of rows over a long K by wavefronts that split it: whole
// 128-byte lines stream through private LDS rings by direct loads (no barrier),
// and meet the matrix instruction in 16-bit values, fp32 ones as bf16 pieces.
// Shared by the router's product and the adapters' first one.
#pragma once

#include "gemm_kernel.h"

namespace kbn {
namespace {

enum : int { kG16b = 0, kG16f = 1, kG32 = 2 };   // dtype codes: bf16, fp16, fp32

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
__device__ __forceinline__ Pieces<kP> pieces_of(const Raw8<kD>& r) {
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
                if (k + 1 < kP) {   // (an infinity leaves a NaN here: see joined)
                    f[2 * i] -= __uint_as_float(a & 0xFFFF0000u);
                    f[2 * i + 1] -= __uint_as_float(b & 0xFFFF0000u);
                }
            }
    }
    return o;
}

// A sum of products of leading pieces and the sum of all others, which counts only where
// the first is finite: leading pieces are infinite where the values are, and give the
// formula's infinities and NaN, while lower pieces are 0 or NaN beside them.
__device__ __forceinline__ f32x4 joined(const f32x4& lead, const f32x4& rest) {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool finite = (__float_as_uint(lead[i]) & 0x7F800000u) != 0x7F800000u;
        v[i] = lead[i] + (finite ? rest[i] : 0.f);
    }
    return v;
}

template <bool kHalf>
__device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, const f32x4& c) {
    if constexpr (kHalf)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// What one operand of a stage (64 K) takes in LDS: rows of 128-byte lines, one
// line a row of 16-bit values, two of fp32 (set 0: K 0 .. 31, set 1: 32 .. 63).
// Sixteen-byte chunk c of row r lies in slot c ^ swz(r).
template <int kD, int kTiles>
struct Operand {
    static constexpr int kSets = kD == kG32 ? 2 : 1, kLoads = 2 * kTiles * kSets, kBytes = kLoads * 1024;
    // values 32 s + 8 q .. + 7 of fragment i's row
    static __device__ __forceinline__ Raw8<kD> at(const uint8_t* p, int i, int row, int s, int q) {
        Raw8<kD> r;
        if constexpr (kD == kG32) {
            const uint8_t* const line = p + s * (kTiles * 2048) + (16 * i + row) * 128;
            r.v[0] = *reinterpret_cast<const u32x4*>(line + (((2 * q) ^ swz(row)) << 4));
            r.v[1] = *reinterpret_cast<const u32x4*>(line + (((2 * q + 1) ^ swz(row)) << 4));
        } else {
            r.v[0] = *reinterpret_cast<const u32x4*>(p + (16 * i + row) * 128 + (((4 * s + q) ^ swz(row)) << 4));
        }
        return r;
    }
};

constexpr int kStreamK = 64;       // K of a stage
constexpr int kStreamWaves = 4;

// What a workgroup's wavefronts need of LDS: kDepth stages each, and afterwards
// their sums.
template <int kTM, int kTE, int kDepth, int kX, int kW>
struct Stream {
    typedef Operand<kX, kTM> OX;
    typedef Operand<kW, kTE> OW;
    static constexpr int kLoads = OX::kLoads + OW::kLoads, kStage = OX::kBytes + OW::kBytes, kRing = kDepth * kStage;
    static constexpr int kSums = kTM * kTE * 1024;                 // bytes of a wavefront's sums
    static constexpr int kSmem = kStreamWaves * (kRing > kSums ? kRing : kSums);
    static_assert(kSmem <= 163840 && (kDepth - 1) * kLoads <= 63);

    // part[0 .. kTM kTE 64) = sums over the units [from, end) of 64 K of the
    // products of x rows with w rows, as the matrix instruction lays them out: tile
    // (i, j) at (i kTE + j) 64 + lane, lane's four x rows 4 (lane / 16) .. of w row lane %
    // 16.  x_at(q), w_at(q): byte offsets of row q in its descriptor, kOob for none (it
    // reads zeros).  All wavefronts of the workgroup; part holds every wavefront's
    // sums behind each other on return.
    template <class XAt, class WAt>
    static __device__ __forceinline__ void run(const v4i& dX, const v4i& dW, XAt x_at, WAt w_at, int K, int from, int end,
                                               uint8_t* smem) {
        constexpr int bx = bytes_of<kX>(), bw = bytes_of<kW>();
        // two pieces hold fp16's 11 bits where the other side is bf16 pieces
        constexpr int PX = kX == kG32 ? 3 : (kX == kG16f && kW == kG32) ? 2 : 1;
        constexpr int PW = kW == kG32 ? 3 : 1;
        constexpr bool kHalf = kX == kG16f && kW == kG16f;
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const uint32_t lds = (uint32_t)(uintptr_t)smem + (uint32_t)wave * kRing;
        const uint8_t* const ring = smem + wave * kRing;
        // load j of an operand brings rows 8 j .. 8 j + 7 (of its second set from
        // the middle on); rows that x_at and w_at do not give read zeros
        const int r8 = lane >> 3;
        auto offset = [&](int j, int tiles, int q, int at) {
            return at == kOob ? kOob : at + j / (2 * tiles) * 128 + (((lane & 7) ^ swz(q)) << 4);
        };
        int xo[OX::kLoads], wo[OW::kLoads];
#pragma unroll
        for (int j = 0; j < OX::kLoads; ++j) xo[j] = offset(j, kTM, 8 * (j % (2 * kTM)) + r8, x_at(8 * (j % (2 * kTM)) + r8));
#pragma unroll
        for (int j = 0; j < OW::kLoads; ++j) wo[j] = offset(j, kTE, 8 * (j % (2 * kTE)) + r8, w_at(8 * (j % (2 * kTE)) + r8));
        // Unit u into buffer buf.  Units past the end load nothing (and keep the
        // count of loads in flight); in the last unit of a ragged K the chunks
        // behind K read zeros, not the next row.
        auto issue = [&](int buf, int u) __attribute__((always_inline)) {
            const uint32_t base = lds + (uint32_t)buf * kStage;
            v4i x = dX, w = dW;
            if (u >= end) x[2] = w[2] = 0;
            const int left = K - u * kStreamK;
            if (left >= kStreamK || u >= end) {
                static_for<OX::kLoads>([&](auto j_) __attribute__((always_inline)) {
                    dma_b128<decltype(j_)::value * 1024, false>(x, base, xo[decltype(j_)::value], u * kStreamK * bx);
                });
                static_for<OW::kLoads>([&](auto j_) __attribute__((always_inline)) {
                    dma_b128<OX::kBytes + decltype(j_)::value * 1024, false>(w, base, wo[decltype(j_)::value], u * kStreamK * bw);
                });
            } else {
                auto cut = [&](int j, int tiles, int off, int bytes) {
                    const int q = 8 * (j % (2 * tiles)) + r8;
                    return j / (2 * tiles) * 128 + (((lane & 7) ^ swz(q)) << 4) < left * bytes ? off : kOob;
                };
                static_for<OX::kLoads>([&](auto j_) __attribute__((always_inline)) {
                    constexpr int j = decltype(j_)::value;
                    dma_b128<j * 1024, false>(x, base, cut(j, kTM, xo[j], bx), u * kStreamK * bx);
                });
                static_for<OW::kLoads>([&](auto j_) __attribute__((always_inline)) {
                    constexpr int j = decltype(j_)::value;
                    dma_b128<OX::kBytes + j * 1024, false>(w, base, cut(j, kTE, wo[j], bw), u * kStreamK * bw);
                });
            }
        };
        constexpr int kAcc = PX + PW > 2 ? 2 : 1;   // products of leading pieces, of others
        f32x4 acc[kAcc][kTM][kTE];
#pragma unroll
        for (int c = 0; c < kAcc; ++c)
#pragma unroll
            for (int i = 0; i < kTM; ++i)
#pragma unroll
                for (int j = 0; j < kTE; ++j) acc[c][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int row = lane & 15, q = lane >> 4;
        for (int d = 0; d < kDepth; ++d) issue(d, from + wave + d * kStreamWaves);
        int buf = 0;
        for (int u = from + wave; u < end; u += kStreamWaves) {
            wait_dma_n<(kDepth - 1) * kLoads>();
            const uint8_t* const at = ring + buf * kStage;
            Raw8<kX> xv[2][kTM];
            Raw8<kW> wv[2][kTE];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int i = 0; i < kTM; ++i) xv[s][i] = OX::at(at, i, row, s, q);
#pragma unroll
                for (int j = 0; j < kTE; ++j) wv[s][j] = OW::at(at + OX::kBytes, j, row, s, q);
            }
            wait_lds();   // all of the stage is read: its buffer may be filled again
            issue(buf, u + kDepth * kStreamWaves);
            buf = buf == kDepth - 1 ? 0 : buf + 1;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                Pieces<PX> px[kTM];
                Pieces<PW> pw[kTE];
#pragma unroll
                for (int i = 0; i < kTM; ++i) px[i] = pieces_of<kX, PX>(xv[s][i]);
#pragma unroll
                for (int j = 0; j < kTE; ++j) pw[j] = pieces_of<kW, PW>(wv[s][j]);
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
                            for (int j = 0; j < kTE; ++j) {
                                f32x4& to = acc[sum > 0 ? 1 : 0][i][j];
                                to = mma<kHalf>(px[i].p[m], pw[j].p[n], to);
                            }
                    }
                }
            }
        }
        wait_dma();         // no load writes to LDS any more
        __syncthreads();    // no wavefront reads its ring any more
        f32x4* const part = reinterpret_cast<f32x4*>(smem);
#pragma unroll
        for (int i = 0; i < kTM; ++i)
#pragma unroll
            for (int j = 0; j < kTE; ++j) {
                f32x4 v = acc[0][i][j];
                if constexpr (kAcc == 2) v = joined(v, acc[1][i][j]);
                part[((wave * kTM + i) * kTE + j) * 64 + lane] = v;
            }
        __syncthreads();
    }

    // Slot s of the sums over the wavefronts, in their order.
    static __device__ __forceinline__ f32x4 sum(const uint8_t* smem, int s) {
        const f32x4* const part = reinterpret_cast<const f32x4*>(smem);
        f32x4 v = part[s];
#pragma unroll
        for (int n = 1; n < kStreamWaves; ++n) v += part[n * kTM * kTE * 64 + s];
        return v;
    }
};

}  // namespace
}  // namespace kbn
