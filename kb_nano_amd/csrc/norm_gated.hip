// The step between two blocks of a layer whose blocks are normed on both sides:
//
//   p  = x / sqrt(mean(x^2) + eps) * post      (x itself without a post norm)
//   r' = residual_scale * r + gate * p         (rounded to the rows' type and kept)
//   n  = r' / sqrt(mean(r'^2) + eps) * w       (of the rounded r': what a later reader sees)
//
// n leaves as rows of the type, or (and) as 1x128 FP8 codes with UE8M0 scales,
// quantized from its unrounded fp32 values as the RMSNorm + quant kernels do.
// gate: none, one value for each channel, for each token or for each element.
//
// Bound by the rows: x, r (and a full gate) are read once and stay in
// registers over both norms, r' and n are written once.  A workgroup of kW
// wavefronts has one token; chunk c of its row is the 512 elements c*512 ..
// c*512+511 (eight a lane), wavefront w owns chunks w, w + kW, ...  Sums of
// squares are fp32: over a lane's elements in order, by butterfly over the
// wavefront, over the wavefronts in order.  A wavefront a chunk up to 4096 columns
// (4096 x 1024 9.2 us, 12.1 before that and the packing of values in pairs).
//
// 4096 x 7168 bf16 with a post norm, a full gate and codes out: 47 us, 264 MB, 5.6
// TB/s (a copy of 1 GiB: 5.1); 777 x 8192 fp16, a gate for each channel, 14.7 us (3 TB/s:
// with one round of workgroups the loads, sums and stores of the rows follow each
// other); one token of 7168 3.9 us, of which 2.4 are a launch.
#include "norm_common.h"

namespace kbn {
namespace {

struct GatedArgs {
    const void* x;
    int64_t ld_x;
    const void* r;
    int64_t ld_r;
    const void* w;
    const void* post;      // nullptr: no post norm
    const void* gate;      // nullptr: no gate
    int64_t gate_row, gate_col;   // element strides; gate_col 0 or 1
    float residual_scale, eps;
    int T, H;
    void* r_out;
    int64_t ld_ro;
    void* n;               // nullptr: no rows out
    int64_t ld_n;
    uint8_t* q;            // nullptr: no codes out
    int64_t ld_q;
    float* s;
    int64_t s_m, s_g;
    int s_bytes;
};

// Sum over the workgroup, in every lane; `part` has a slot for each wavefront.
template <int kW>
__device__ __forceinline__ float group_sum(float p, float* part, int wave, int lane) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) p = p + __shfl_xor(p, d, 64);
    if (lane == 0) part[wave] = p;
    __syncthreads();
    p = part[0];
#pragma unroll
    for (int w = 1; w < kW; ++w) p = p + part[w];
    return p;
}

// Eight elements of a row as they lie in memory (zeros past the range).
template <int kT>
struct Eight {
    u32x4 w[kT == kNormF32 ? 2 : 1];
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, int off, int nt) {
        if (nt) {
            w[0] = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, kNtLoad);
            if constexpr (kT == kNormF32) w[1] = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 16, 0, kNtLoad);
        } else {
            w[0] = __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0);
            if constexpr (kT == kNormF32) w[1] = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 16, 0, 0);
        }
    }
    __device__ __forceinline__ void floats(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t word = w[0][j];
            if constexpr (kT == kNormF32) {
                v[j] = __uint_as_float(word);
                v[4 + j] = __uint_as_float(w[1][j]);
            } else if constexpr (kT == kNormBf16) {
                v[2 * j] = bf16lo(word);
                v[2 * j + 1] = bf16hi(word);
            } else {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const h2 h = __builtin_bit_cast(h2, word);
                v[2 * j] = (float)h.x;
                v[2 * j + 1] = (float)h.y;
            }
        }
    }
    // v rounded to the type
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (kT == kNormF32) {
                w[0][j] = __float_as_uint(v[j]);
                w[1][j] = __float_as_uint(v[4 + j]);
            } else {
                w[0][j] = pack2<kT>(v[2 * j], v[2 * j + 1]);
            }
        }
    }
    __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t rs, int off) const {
        __builtin_amdgcn_raw_buffer_store_b128(w[0], rs, off, 0, 0);
        if constexpr (kT == kNormF32) __builtin_amdgcn_raw_buffer_store_b128(w[1], rs, off + 16, 0, 0);
    }
};

// What a token's elements have in common.
struct Step {
    float inv;          // of the post norm
    float scale;        // residual's
    float gate;         // the token's gate (1 without one)
};
// A lane's eight elements of the new residual, rounded.
template <int kT>
__device__ __forceinline__ Eight<kT> new_residual(const Step& st, bool post, bool gated, const float (&x)[8], const Eight<kT>& r,
                                                  const Eight<kT>& wp, const Eight<kT>& g) {
    float p[8], f[8], o[8];
    if (post) {
        wp.floats(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = (x[j] * st.inv) * f[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = x[j];
    }
    if (gated) {
        g.floats(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = f[j] * p[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = st.gate * p[j];
    }
    r.floats(f);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = fmaf(st.scale, f[j], p[j]);
    Eight<kT> out;
    out.set(o);
    return out;
}

// Rows or codes of a lane's eight normalized values at element e0 of token m.
template <int kT>
__device__ __forceinline__ void put(const GatedArgs& a, int m, int e0, int lane, const float (&v)[8]) {
    constexpr int kB = elt_bytes<kT>();
    if (a.n) {
        const __amdgpu_buffer_rsrc_t nw = row_rsrc(static_cast<uint8_t*>(a.n) + (int64_t)m * a.ld_n * kB, kB * a.H);
        store8<kT>(nw, kB * e0, v);
    }
    if (a.q) {
        const __amdgpu_buffer_rsrc_t qw = row_rsrc(a.q + (int64_t)m * a.ld_q, a.H);
        const __amdgpu_buffer_rsrc_t sw = row_rsrc(a.s, a.s_bytes);
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[j]));
        amax = __uint_as_float(row16_max_u32(__float_as_uint(amax)));
        amax = fmaxf(amax, kGroupEps);
        const float sc = ue8m0_ceil_div448(amax), is = inv_scale(sc);
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = clamp448(v[j] * is);
        __builtin_amdgcn_raw_buffer_store_b64(
            u32x2{pack4_e4m3(t[0], t[1], t[2], t[3]), pack4_e4m3(t[4], t[5], t[6], t[7])}, qw, e0, 0, 0);
        const bool owner = (lane & 15) == 0 && e0 < a.H;
        __builtin_amdgcn_raw_buffer_store_b32(
            __float_as_uint(sc), sw, owner ? (int)(4 * ((int64_t)m * a.s_m + (int64_t)(e0 >> 7) * a.s_g)) : kOob, 0, 0);
    }
}

// kCW > 0: the row stays in registers, kCW chunks a wavefront.  kCW == 0: any
// length, its values computed again in each of three passes (no pass reads
// what another wrote, so r' may replace r).
template <int kW, int kCW, int kT>
__global__ __launch_bounds__(64 * kW, kCW == 2 && kT != kNormF32 ? 4 : 1) void gated_norm_kernel(const GatedArgs a) {
#pragma clang fp contract(off)
    __shared__ float part[2][kW];
    constexpr int kB = elt_bytes<kT>();
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = blockIdx.x;
    const int bytes = kB * a.H;
    auto row = [&](const void* p, int64_t ld) {
        return row_rsrc(p ? static_cast<const uint8_t*>(p) + (int64_t)m * ld * kB : nullptr, p ? bytes : 0);
    };
    const bool post = a.post != nullptr, gated = a.gate != nullptr && a.gate_col != 0;
    const __amdgpu_buffer_rsrc_t xr = row(a.x, a.ld_x), rr = row(a.r, a.ld_r), ro = row(a.r_out, a.ld_ro);
    const __amdgpu_buffer_rsrc_t wr = row(a.w, 0), pr = row(a.post, 0), gr = row(gated ? a.gate : nullptr, a.gate_row);
    Step st{1.f, a.residual_scale, 1.f};
    if (a.gate && !gated) {
        const int64_t at = (int64_t)m * a.gate_row;
        if constexpr (kT == kNormF32) st.gate = static_cast<const float*>(a.gate)[at];
        else if constexpr (kT == kNormF16) st.gate = (float)static_cast<const _Float16*>(a.gate)[at];
        else st.gate = __uint_as_float((uint32_t)static_cast<const uint16_t*>(a.gate)[at] << 16);
    }
    if constexpr (kCW > 0) {
        // all that the token takes is asked for at once: one wait for the memory
        // instead of three (the weights mostly come from L2)
        Eight<kT> x[kCW], r[kCW], g[kCW], wp[kCW], wv[kCW];
#pragma unroll
        for (int i = 0; i < kCW; ++i) {
            const int off = kB * ((kW * i + wave) * 512 + 8 * lane);
            x[i].load(xr, off, kNtLoad);
            if (post) wp[i].load(pr, off, 0);
            r[i].load(rr, off, kNtLoad);
            if (gated) g[i].load(gr, off, a.gate_row ? kNtLoad : 0);
            wv[i].load(wr, off, 0);
        }
        float v[kCW][8];   // x, then r'
        float p = 0.f;
#pragma unroll
        for (int i = 0; i < kCW; ++i) {
            x[i].floats(v[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) p = fmaf(v[i][j], v[i][j], p);
        }
        if (post) st.inv = 1.0f / sqrtf(group_sum<kW>(p, part[0], wave, lane) / (float)a.H + a.eps);
        p = 0.f;
#pragma unroll
        for (int i = 0; i < kCW; ++i) {
            const int off = kB * ((kW * i + wave) * 512 + 8 * lane);
            const Eight<kT> o = new_residual<kT>(st, post, gated, v[i], r[i], wp[i], g[i]);
            o.store(ro, off);
            o.floats(v[i]);
            if (off >= bytes) {   // past the row: 0 * inf may have come out
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) p = fmaf(v[i][j], v[i][j], p);
        }
        const float inv = 1.0f / sqrtf(group_sum<kW>(p, part[1], wave, lane) / (float)a.H + a.eps);
#pragma unroll
        for (int i = 0; i < kCW; ++i) {
            const int e0 = (kW * i + wave) * 512 + 8 * lane;
            float w8[8], n[8];
            wv[i].floats(w8);
            // (past the row weights are 0 and a NaN of 0 * inf is passed over by the group's maximum)
#pragma unroll
            for (int j = 0; j < 8; ++j) n[j] = (v[i][j] * inv) * w8[j];
            put<kT>(a, m, e0, lane, n);
        }
    } else {
        const int chunks = (a.H + 511) / 512;
        float p = 0.f;
        if (post) {
            for (int c = wave; c < chunks; c += kW) {
                float x[8];
                load8<kT>(xr, kB * (c * 512 + 8 * lane), x);
#pragma unroll
                for (int j = 0; j < 8; ++j) p = fmaf(x[j], x[j], p);
            }
            st.inv = 1.0f / sqrtf(group_sum<kW>(p, part[0], wave, lane) / (float)a.H + a.eps);
        }
        auto residual = [&](int c, float (&o)[8]) {
            const int off = kB * (c * 512 + 8 * lane);
            Eight<kT> x, r, wp, g;
            x.load(xr, off, 0);
            r.load(rr, off, 0);
            if (post) wp.load(pr, off, 0);
            if (gated) g.load(gr, off, 0);
            float xf[8];
            x.floats(xf);
            const Eight<kT> out = new_residual<kT>(st, post, gated, xf, r, wp, g);
            out.floats(o);
            if (off >= bytes) {
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = 0.f;
            }
            return out;
        };
        p = 0.f;
        for (int c = wave; c < chunks; c += kW) {
            float o[8];
            residual(c, o);
#pragma unroll
            for (int j = 0; j < 8; ++j) p = fmaf(o[j], o[j], p);
        }
        const float inv = 1.0f / sqrtf(group_sum<kW>(p, part[1], wave, lane) / (float)a.H + a.eps);
        for (int c = wave; c < chunks; c += kW) {
            const int e0 = c * 512 + 8 * lane;
            float o[8], w8[8], n[8];
            residual(c, o).store(ro, kB * e0);
            load8<kT>(wr, kB * e0, w8);
#pragma unroll
            for (int j = 0; j < 8; ++j) n[j] = (o[j] * inv) * w8[j];
            put<kT>(a, m, e0, lane, n);
        }
    }
}

template <int kW, int kCW, int kT>
void launch_cfg(const GatedArgs& a, hipStream_t st) {
    gated_norm_kernel<kW, kCW, kT><<<dim3((unsigned)a.T), dim3(64 * kW), 0, st>>>(a);
}

template <int kT>
void launch_gated(const GatedArgs& a, hipStream_t st) {
    const int chunks = (a.H + 511) / 512;
    if (chunks <= 1) launch_cfg<1, 1, kT>(a, st);
    else if (chunks <= 2) launch_cfg<2, 1, kT>(a, st);
    else if (chunks <= 4) launch_cfg<4, 1, kT>(a, st);
    else if (chunks <= 8) launch_cfg<8, 1, kT>(a, st);
    else if (chunks <= 16) launch_cfg<8, 2, kT>(a, st);
    else if (chunks <= 32) launch_cfg<8, 4, kT>(a, st);
    else launch_cfg<8, 0, kT>(a, st);
}

}  // namespace
}  // namespace kbn

using namespace kbn;

extern "C" int kbn_gated_add_rmsnorm(const void* x, int dtype, int64_t ld_x, const void* r, int64_t ld_r, const void* w,
                                     const void* post, const void* gate, int64_t gate_row, int64_t gate_col,
                                     float residual_scale, float eps, int64_t T, int64_t H, void* r_out, int64_t ld_ro,
                                     void* n_out, int64_t ld_n, void* q_fp8, int64_t ld_q, float* scale,
                                     int64_t s_stride_m, int64_t s_stride_g, void* stream) {
    const char* what = "gated_add_rmsnorm";
    KBN_CHECK_ARG(dtype >= 0 && dtype <= 2, "%s: dtype code %d (0 bf16, 1 fp16, 2 fp32)", what, dtype);
    KBN_CHECK_ARG(T >= 0 && T <= 0x7FFFFFFFLL, "%s: bad T=%lld", what, (long long)T);
    KBN_CHECK_ARG(H > 0 && H % 8 == 0 && H <= (1 << 26), "%s: hidden size %lld must be a positive multiple of 8, at most 2^26",
                  what, (long long)H);
    if (T == 0) return 0;
    KBN_CHECK_ARG(x && r && w && r_out && (n_out || q_fp8), "%s: null pointer", what);
    const int64_t b = dtype == kNormF32 ? 4 : 2;
    auto rows = [&](const void* p, int64_t ld) { return aligned16(p) && ld >= H && ld * b % 16 == 0; };
    KBN_CHECK_ARG(rows(x, ld_x) && rows(r, ld_r) && rows(r_out, ld_ro) && (!n_out || rows(n_out, ld_n)),
                  "%s: rows must be 16-byte aligned with strides of at least the hidden size", what);
    KBN_CHECK_ARG(aligned16(w) && aligned16(post), "%s: weights must be 16-byte aligned", what);
    KBN_CHECK_ARG(!gate || (gate_row >= 0 && (gate_col == 0 || (gate_col == 1 && aligned16(gate) && gate_row * b % 16 == 0))),
                  "%s: the gate's values must be contiguous, its rows 16-byte aligned", what);
    GatedArgs a{};
    if (q_fp8) {
        KBN_CHECK_ARG(scale && (reinterpret_cast<uintptr_t>(scale) & 3u) == 0 && s_stride_m >= 0 && s_stride_g >= 0,
                      "%s: scales must be 4-byte aligned with strides that are not negative", what);
        KBN_CHECK_ARG(ld_q >= H && ld_q % 8 == 0 && (reinterpret_cast<uintptr_t>(q_fp8) & 7u) == 0,
                      "%s: code rows must be 8-byte aligned with a stride of at least the hidden size", what);
        const int64_t s_bytes = ((T - 1) * s_stride_m + ((H + 127) / 128 - 1) * s_stride_g + 1) * 4;
        KBN_CHECK_ARG(s_bytes < 0x7FFFFFFFLL, "%s: the scales span 2 GiB or more", what);
        a.s_bytes = (int)s_bytes;
    }
    a.x = x;
    a.ld_x = ld_x;
    a.r = r;
    a.ld_r = ld_r;
    a.w = w;
    a.post = post;
    a.gate = gate;
    a.gate_row = gate_row;
    a.gate_col = gate_col;
    a.residual_scale = residual_scale;
    a.eps = eps;
    a.T = (int)T;
    a.H = (int)H;
    a.r_out = r_out;
    a.ld_ro = ld_ro;
    a.n = n_out;
    a.ld_n = ld_n;
    a.q = static_cast<uint8_t*>(q_fp8);
    a.ld_q = ld_q;
    a.s = scale;
    a.s_m = s_stride_m;
    a.s_g = s_stride_g;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == kNormBf16) launch_gated<kNormBf16>(a, st);
    else if (dtype == kNormF16) launch_gated<kNormF16>(a, st);
    else launch_gated<kNormF32>(a, st);
    KBN_CHECK_LAUNCH(what);
    return 0;
}
