// Routing of tokens to experts: scores, choice, weights.
//
//   l       logits [T, E]; NaN counts as -inf, +inf as the largest float
//   score   softmax(l) or 1 / (1 + exp(-l))
//   c       choice: l without a bias (scores order as the logits do, and l has
//           no rounding of its own), score + bias with one; -inf where l is
//   groups  E / G consecutive experts each; a group's rank is the largest c in
//           it, or with a bias the sum of its two largest; experts outside the
//           best topk_groups groups count as -inf
//   ids     the top_k experts of largest c, descending
//   weight  score of each (0 where c is -inf), over their sum if renormalised
//           (all 0 where that is 0), times scale
// Equal values go to the lower index, in groups and in experts.
//
// Scores next to a border decide which expert is taken, and in fp32 two experts
// of 256 come out in the other order once in some 10^4 tokens: whatever a choice
// depends on is computed in 64 bits, and so are the few weights.
//
// Reads and writes are small (16384 x 256 fp32 logits, top 8 with groups and a bias:
// 18 MB, 4 us at the rate of a copy).  That case takes 18 us (1 TB/s): 14 the four-token
// way, some 1100 instructions a wavefront, and 4 to 5 the last way of the 1 to 7 tokens
// that need it, which ends after all others.  Few tokens take the latency of their
// instructions (one token 5.4; 777 x 128, no groups, 3.8).
//
// The general path: one wavefront a token, expert e = lane * V + j in register j, so the lowest
// index of equal keys is the first lane's first register.  Keys are the values'
// bits mapped to unsigned integers of the same order, 0 for taken or absent.
#include "kbn_common.h"

#include <type_traits>
#include <utility>

namespace kbn {
namespace {

constexpr int kMaxRouted = 1024;   // experts (16 a lane)
constexpr int kWaves = 4;          // tokens a workgroup

enum : int { kL16b = 0, kL16f = 1, kL32 = 2 };   // logit dtype codes: bf16, fp16, fp32

struct TopkArgs {
    const void* l;
    int64_t ld;
    const float* bias;
    int T, E, k;
    int G, kept, per;        // groups, groups kept, experts a group
    uint32_t per_magic;      // ceil(2^32 / per): e / per for e < 1024 and per > 1
    int sigmoid, renorm;
    float scale;
    float* w;
    void* ids;
    int id64;
    int vec, vec_bias;       // rows, bias take loads of four
};

// Bits in the values' order; -0 and 0 are one value.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
    return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
template <typename K> struct Masked;   // the key of -inf
template <> struct Masked<uint32_t> { static constexpr uint32_t key = 0x007FFFFFu; };
template <> struct Masked<uint64_t> { static constexpr uint64_t key = 0x000FFFFFFFFFFFFFull; };

// Largest value over the wavefront, the same in every lane (a scalar).
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = row16_max_u32(v);
    const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
    const uint32_t c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
    const uint32_t ab = a > b ? a : b, cd = c > d ? c : d;
    return ab > cd ? ab : cd;
}
// First lane that holds the largest key.
__device__ __forceinline__ int wave_argmax(uint32_t key) {
    return (int)__builtin_ctzll(__ballot(key == wave_max(key)));
}
__device__ __forceinline__ int wave_argmax(uint64_t key) {
    const uint32_t hi = (uint32_t)(key >> 32), top = wave_max(hi);
    const uint64_t at = __ballot(hi == top);
    if ((at & (at - 1)) == 0) return (int)__builtin_ctzll(at);   // the upper words decide nearly always
    const uint32_t lo = hi == top ? (uint32_t)key : 0u, low = wave_max(lo);
    return (int)__builtin_ctzll(__ballot(hi == top && lo == low));
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

template <int kL>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
    if constexpr (kL == kL32) return static_cast<const float*>(p)[i];
    else if constexpr (kL == kL16b) return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
    else return (float)static_cast<const _Float16*>(p)[i];
}

// Token t by the whole wavefront; `mine`: 64 V words of LDS of its own.
// K: uint32_t where c is the logit, uint64_t where it is score + bias.
template <int V, int kL, typename K>
__device__ __forceinline__ void route_token(const TopkArgs& a, int t, int lane, uint64_t* mine) {
    constexpr bool kBias = sizeof(K) == 8;
    const float low = -__builtin_inff();
    float l[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = lane * V + j;
        float v = low;
        if (e < a.E) v = load_logit<kL>(a.l, (int64_t)t * a.ld + e);
        l[j] = v != v ? low : fminf(v, 3.4028234663852886e38f);
    }
    // softmax over the row, where its sum is needed
    double top = 0.0, sum = 1.0;
    if (!a.sigmoid && (kBias || !a.renorm)) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) m = max(m, order_key(l[j]));
        m = wave_max(m);
        const float fm = __uint_as_float(m & 0x80000000u ? m ^ 0x80000000u : ~m);
        top = fm == low ? 0.0 : (double)fm;
        sum = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) sum += exp((double)l[j] - top);
        sum = wave_sum(sum);
    }
    auto score = [&](float v) -> double {
        if (v == low) return 0.0;
        if (a.sigmoid) return 1.0 / (1.0 + exp(-(double)v));
        return exp((double)v - top) / sum;
    };
    K key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = lane * V + j;
        if constexpr (kBias) {
            const double c = l[j] == low ? (double)low : score(l[j]) + (double)a.bias[e < a.E ? e : 0];
            key[j] = c != c ? Masked<K>::key : order_key(c);
        } else {
            key[j] = order_key(l[j]);
        }
        if (e >= a.E) key[j] = 0;
    }
    if (a.G > 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) mine[lane * V + j] = key[j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        uint64_t rank = 0;
        if (lane < a.G) {
            uint64_t best = 0, second = 0;
            // eight at a time: one by one each read waits for the last
            for (int i0 = 0; i0 < a.per; i0 += 8) {
                uint64_t v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = i0 + i < a.per ? mine[lane * a.per + i0 + i] : 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    second = v[i] > best ? best : (v[i] > second ? v[i] : second);
                    best = v[i] > best ? v[i] : best;
                }
            }
            rank = best;
            if (kBias && a.per > 1) {
                auto value = [](uint64_t u) {
                    return __longlong_as_double((long long)(u >> 63 ? u ^ 0x8000000000000000ull : ~u));
                };
                const double s = value(best) + value(second);
                rank = s != s ? Masked<uint64_t>::key : order_key(s);
            }
        }
        uint64_t keep = 0;
        for (int i = 0; i < a.kept; ++i) {
            const int g = wave_argmax(rank);
            keep |= 1ull << g;
            if (lane == g) rank = 0;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = lane * V + j;
            const int g = a.per == 1 ? e : (int)__umulhi((uint32_t)e, a.per_magic);
            if (e < a.E && !(keep >> g & 1)) key[j] = Masked<K>::key;
        }
    }
    // the best of the lane's own, its register and logit
    K best;
    int at;
    float logit;
    auto own_best = [&] {
        best = key[0];
        at = 0;
        logit = l[0];
#pragma unroll
        for (int j = 1; j < V; ++j)
            if (key[j] > best) {
                best = key[j];
                at = j;
                logit = l[j];
            }
    };
    own_best();
    int id = 0;
    float picked = low;   // this lane's slot: its expert's logit, -inf if it counts for nothing
    for (int i = 0; i < a.k; ++i) {
        const int src = wave_argmax(best);
        const int e = src * V + __builtin_amdgcn_readlane(at, src);
        const float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(best == Masked<K>::key ? low : logit), src));
        if (lane == i) {
            id = e;
            picked = v;
        }
        if (lane == src) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j == at) key[j] = 0;
            own_best();
        }
    }
    double s;
    if (a.renorm) {
        if (!a.sigmoid) {   // the row's sum falls out: over the largest of the chosen
            const uint32_t m = wave_max(order_key(lane < a.k ? picked : low));
            const float fm = __uint_as_float(m & 0x80000000u ? m ^ 0x80000000u : ~m);
            s = lane < a.k && picked != low ? exp((double)picked - (double)fm) : 0.0;
        } else {
            s = lane < a.k ? score(picked) : 0.0;
        }
        const double all = wave_sum(s);
        s = all > 0.0 ? s / all : 0.0;
    } else {
        s = lane < a.k ? score(picked) : 0.0;
    }
    if (lane < a.k) {
        const int64_t o = (int64_t)t * a.k + lane;
        a.w[o] = (float)(s * (double)a.scale);
        if (a.id64) static_cast<int64_t*>(a.ids)[o] = id;
        else static_cast<int32_t*>(a.ids)[o] = id;
    }
}

template <int V, int kL, typename K>
__global__ __launch_bounds__(64 * kWaves) void router_topk_kernel(const TopkArgs a) {
    __shared__ uint64_t choice[kWaves][64 * V];   // used with groups only
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * kWaves + wave;
    if (t >= a.T) return;   // no barrier follows: each wavefront uses its own part of the LDS
    route_token<V, kL, K>(a, t, lane, choice[wave]);
}

// ---- Four tokens a wavefront ------------------------------------------------
// Sixteen lanes a token, lane n holding experts 4 (n + 16 jj) + i in register 4 jj
// + i (coalesced loads; V = 16 experts a lane at 256).  A key is a choice value in
// its upper bits and the expert's number in its lower kIB: a value and its owner at
// once, never equal to another, and sorting is maxima and minima.  Each lane sorts
// its best eight; four exchanges across the 16 lanes keep the best eight of the
// token, in order, in every lane, and the best of what was left out.
//
// 16-bit logits (no bias) leave the lower bits of a float empty: nothing is lost.
// Other values go as places between the row's smallest and largest, 24 bits of
// them, from fp32 scores.  Where neighbours in the order are further apart than the
// errors of both, the order is the exact one.  Where some are not, the eight and the
// best one left out are ordered by their 64-bit values, a lane each; that is exact
// if the last one taken is above whatever else was left out.  A token for which
// that does not hold either, or whose last kept and first dropped group are too
// close, is routed again by the whole wavefront in 64 bits (route_token).  (Cut
// floats in the keys, 2^-15 of the value: 0.5% of tokens took the last way, and at
// some 7 us a wavefront 1000 tokens 14 us.)
constexpr int kFastK = 8;

// Exchange with another of the row's 16 lanes: 0 x ^ 1, 1 x ^ 2, 2 the other half of
// eight, 3 the other eight (after the first two and three all lanes of four and
// eight hold the same, so mirrors serve).
template <int kStep>
__device__ __forceinline__ uint32_t from_other(uint32_t v) {
    constexpr int ctrl = kStep == 0 ? 0xB1 : kStep == 1 ? 0x4E : kStep == 2 ? 0x141 : 0x128;   // row_half_mirror, row_ror:8
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xF, 0xF, false);
}
template <int kStep>
__device__ __forceinline__ float from_other(float v) { return __uint_as_float(from_other<kStep>(__float_as_uint(v))); }

template <class F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) { each_of(f, std::make_integer_sequence<int, N>{}); }

__device__ __forceinline__ void order2(uint32_t& a, uint32_t& b) {   // a >= b
    const uint32_t hi = max(a, b), lo = min(a, b);
    a = hi;
    b = lo;
}
// Descending order of eight keys (19 exchanges).
__device__ __forceinline__ void sort8(uint32_t (&k)[8]) {
    order2(k[0], k[1]); order2(k[2], k[3]); order2(k[4], k[5]); order2(k[6], k[7]);
    order2(k[0], k[2]); order2(k[1], k[3]); order2(k[4], k[6]); order2(k[5], k[7]);
    order2(k[1], k[2]); order2(k[5], k[6]); order2(k[0], k[4]); order2(k[3], k[7]);
    order2(k[1], k[5]); order2(k[2], k[6]);
    order2(k[1], k[4]); order2(k[3], k[6]);
    order2(k[2], k[4]); order2(k[3], k[5]);
    order2(k[3], k[4]);
}
// The best eight of two descending eights, descending, and the best of the rest.
__device__ __forceinline__ void merge8(uint32_t (&k)[8], const uint32_t (&o)[8], uint32_t& rest) {
#pragma unroll
    for (int i = 0; i < 8; ++i) rest = max(rest, min(k[i], o[7 - i]));
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = max(k[i], o[7 - i]);
    // the maxima rise and then fall (or the other way round): halves, quarters, pairs
    order2(k[0], k[4]); order2(k[1], k[5]); order2(k[2], k[6]); order2(k[3], k[7]);
    order2(k[0], k[2]); order2(k[1], k[3]); order2(k[4], k[6]); order2(k[5], k[7]);
    order2(k[0], k[1]); order2(k[2], k[3]); order2(k[4], k[5]); order2(k[6], k[7]);
}

// Largest number of groups: a lane has one.
constexpr int kFastGroups = 16;

template <int V, int kL, bool kBias>
__global__ __launch_bounds__(64 * kWaves) void router_topk_rows_kernel(const TopkArgs a) {
    constexpr int Q = V / 4;                                   // quads of experts a lane
    constexpr int kIB = V == 4 ? 6 : V == 8 ? 7 : V == 16 ? 8 : 9;
    constexpr uint32_t kIds = (1u << kIB) - 1;
    // 16-bit logits leave the cut bits empty: nothing is lost
    constexpr bool kExact = !kBias && kL != kL32;
    // upper parts of keys: 0 no expert; -inf; values
    constexpr uint32_t kMaskedPart = kExact ? Masked<uint32_t>::key >> kIB : 1u;
    constexpr float kPlaces = kIB == 9 ? 8388604.f : 16777212.f;   // 2^(32 - kIB), 2^24 at most, less four
    // The row's smallest value is meant to lie here; the rounding of the origin below (terms
    // up to 64 kPlaces < 2^30: two of 32 at most) moves the whole row by up to 64 places,
    // so no value reaches the place of -inf, and none the end: 0.0001 kPlaces > 838 are left.
    constexpr float kFirstPlace = 68.f;
    __shared__ uint64_t scratch[kWaves][16 * V];               // quads of four tokens, or one token's choice
    const int lane = threadIdx.x & 63, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t0 = (blockIdx.x * kWaves + wave) * 4;
    if (t0 >= a.T) return;                                     // no barrier follows
    const int t = min(t0 + (lane >> 4), a.T - 1);              // past the end: the last token again, not stored
    const float low = -__builtin_inff();
    float f[V];
#pragma unroll
    for (int jj = 0; jj < Q; ++jj) {
        const int e = 4 * (n + 16 * jj);
        const int64_t at = (int64_t)t * a.ld + e;
        if (a.vec) {
            if constexpr (kL == kL32) {
                typedef float f4 __attribute__((ext_vector_type(4)));
                f4 v{low, low, low, low};
                if (e < a.E) v = *reinterpret_cast<const f4*>(static_cast<const float*>(a.l) + at);
#pragma unroll
                for (int i = 0; i < 4; ++i) f[4 * jj + i] = v[i];
            } else {
                u32x2 v{0u, 0u};
                if (e < a.E) v = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(a.l) + at);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint16_t h = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
                    const float x = kL == kL16b ? __uint_as_float((uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
                    f[4 * jj + i] = e < a.E ? x : low;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[4 * jj + i] = e + i < a.E ? load_logit<kL>(a.l, at + i) : low;
        }
    }
    // (the larger of a NaN and -inf is -inf; as a median of three the compiler drops the -inf)
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = fminf(fmaxf(f[j], low), 3.4028234663852886e38f);
    // Choice values in fp32 and how far they may be from the exact ones: err + 2^-23
    // of the value.  exp2(x) of |x| < 128 with x off by 2^-24 of itself and the
    // instruction by 2^-23, u / (1 + u)^2 (1 + |x|) < 0.6, a sum and a reciprocal of
    // 2^-24 and 2^-23: a sigmoid is off by less than 2^-21.  A softmax adds its sum's
    // V + 4 roundings: 2^-18.
    float err = 0.f;
    if constexpr (kBias) {
        constexpr float kLog2e = 1.4426950408889634f;
        float bias[V];
        if (a.vec_bias) {
            typedef float f4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int jj = 0; jj < Q; ++jj) {
                const f4 v = *reinterpret_cast<const f4*>(a.bias + min(4 * (n + 16 * jj), a.E - 4));
#pragma unroll
                for (int i = 0; i < 4; ++i) bias[4 * jj + i] = v[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) bias[j] = a.bias[min(4 * (n + 16 * (j / 4)) + (j & 3), a.E - 1)];
        }
        if (a.sigmoid) {
            err = 0x1p-21f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * f[j]));
                f[j] = f[j] == low ? low : s + bias[j];
            }
        } else {
            err = 0x1p-18f;
            float top = low, sum = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) top = fmaxf(top, f[j]);
            top = fmaxf(top, from_other<0>(top));
            top = fmaxf(top, from_other<1>(top));
            top = fmaxf(top, from_other<2>(top));
            top = fmaxf(top, from_other<3>(top));
            top = top == low ? 0.f : top;
            float u[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                u[j] = __builtin_amdgcn_exp2f(kLog2e * (f[j] - top));
                sum += u[j];
            }
            sum += from_other<0>(sum);
            sum += from_other<1>(sum);
            sum += from_other<2>(sum);
            sum += from_other<3>(sum);
            const float over = __builtin_amdgcn_rcpf(sum);
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = f[j] == low ? low : u[j] * over + bias[j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = fmaxf(f[j], low);   // a NaN counts as -inf
    }
    bool groups = true, sure = true;   // the kept groups, the order are the exact ones
    if (a.G > 1) {
        // a quad's best, and its two best with a bias; lane g then ranks group g
        float* const quads = reinterpret_cast<float*>(scratch[wave]) + (lane >> 4) * (16 * Q * 2);
#pragma unroll
        for (int jj = 0; jj < Q; ++jj) {
            const float b1 = fmaxf(f[4 * jj], f[4 * jj + 1]), s1 = fminf(f[4 * jj], f[4 * jj + 1]);
            const float b2 = fmaxf(f[4 * jj + 2], f[4 * jj + 3]), s2 = fminf(f[4 * jj + 2], f[4 * jj + 3]);
            *reinterpret_cast<f32x2*>(&quads[2 * (n + 16 * jj)]) = f32x2{fmaxf(b1, b2), fmaxf(fminf(b1, b2), fmaxf(s1, s2))};
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const int quads_of = a.per / 4;   // quads a group
        float best = low, second = low;
        for (int i0 = 0; i0 < quads_of; i0 += 4) {
            f32x2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = *reinterpret_cast<const f32x2*>(&quads[2 * min(n * quads_of + min(i0 + i, quads_of - 1), 16 * Q - 1)]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i0 + i < quads_of) {
                    second = fmaxf(fminf(best, v[i].x), fmaxf(second, v[i].y));
                    best = fmaxf(best, v[i].x);
                }
        }
        const float rank = n < a.G ? (kBias ? best + second : best) : low;
        int before = 0;   // groups that come before this lane's
        auto compare = [&](float other, int shift) {
            const int g = (n + 16 - shift) & 15;   // row_ror: lane n gets lane n - shift
            before += (int)(other > rank) | ((int)(other == rank) & (int)(g < n));
        };
        each<15>([&](auto i) {
            constexpr int shift = decltype(i)::value + 1;
            compare(__uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(rank), 0x120 + shift, 0xF, 0xF, false)),
                    shift);
        });
        const bool kept = n < a.G && before < a.kept;
        const uint32_t keep = (uint32_t)(__ballot(kept) >> (lane & 48)) & 0xFFFFu;
        if constexpr (kBias) {   // (a group's rank is exact without one)
            float least = kept ? rank : __builtin_inff(), most = kept || n >= a.G ? low : rank;
            float size = n < a.G ? fmaxf(fabsf(best), fabsf(second)) : 0.f;   // of the sums' terms
            auto both = [&](float l, float m, float z) {
                least = fminf(least, l);
                most = fmaxf(most, m);
                size = fmaxf(size, z);
            };
            both(from_other<0>(least), from_other<0>(most), from_other<0>(size));
            both(from_other<1>(least), from_other<1>(most), from_other<1>(size));
            both(from_other<2>(least), from_other<2>(most), from_other<2>(size));
            both(from_other<3>(least), from_other<3>(most), from_other<3>(size));
            // two sums of two terms, each off by err + 2^-23 of itself, and rounded
            if (a.kept < a.G) groups = least - most > 4.f * err + 0x1p-20f * size;
        }
#pragma unroll
        for (int jj = 0; jj < Q; ++jj) {
            const int quad = n + 16 * jj;
            const int g = a.per == 4 ? quad : (int)__umulhi(4u * (uint32_t)quad, a.per_magic);
            const bool in = g < 16 && (keep >> (g & 15) & 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) f[4 * jj + i] = in ? f[4 * jj + i] : low;
        }
    }
    float lo = __builtin_inff(), hi = low, scale = 0.f, from = 2.f;   // (places 2 and up; 1: -inf)
    if constexpr (!kExact) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            lo = f[j] == low ? lo : fminf(lo, f[j]);
            hi = fmaxf(hi, f[j]);
        }
        lo = fminf(lo, from_other<0>(lo));
        hi = fmaxf(hi, from_other<0>(hi));
        lo = fminf(lo, from_other<1>(lo));
        hi = fmaxf(hi, from_other<1>(hi));
        lo = fminf(lo, from_other<2>(lo));
        hi = fmaxf(hi, from_other<2>(hi));
        lo = fminf(lo, from_other<3>(lo));
        hi = fmaxf(hi, from_other<3>(hi));
        // (one value, none, an infinite one, or values close together far from 0, whose
        // places would be off by more than is left at the end: all in one place)
        const float range = hi - lo;
        const bool fits = range > 0x1p-100f && range < __builtin_inff() && fmaxf(fabsf(lo), fabsf(hi)) < 64.f * range;
        scale = fits ? kPlaces * 0.9999f / range : 0.f;
        from = fits ? kFirstPlace - lo * scale : 2.f;
    }
    auto part = [&](float v) -> uint32_t {
        if constexpr (kExact) return order_key(v) >> kIB;
        return (uint32_t)fmaxf(fmaf(v, scale, from), 1.f);   // (-inf, and its NaN with a scale of 0, in place 1)
    };
    uint32_t k[8], rest = 0;
#pragma unroll
    for (int b = 0; b < (V + 7) / 8; ++b) {
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (8 * b + j >= V) {
                o[j] = 0;
                continue;
            }
            const int jj = 2 * b + j / 4, e = 4 * (n + 16 * jj) + (j & 3);
            o[j] = (part(f[8 * b + j]) << kIB | (kIds - (uint32_t)e)) & (e < a.E ? ~0u : 0u);
        }
        sort8(o);
        if (b == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) k[j] = o[j];
        } else {
            merge8(k, o, rest);
        }
    }
    auto join = [&](auto step) {
        constexpr int S = decltype(step)::value;
        uint32_t o[8];
        rest = max(rest, from_other<S>(rest));
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = from_other<S>(k[j]);
        merge8(k, o, rest);
    };
    join(std::integral_constant<int, 0>{});
    join(std::integral_constant<int, 1>{});
    join(std::integral_constant<int, 2>{});
    join(std::integral_constant<int, 3>{});
    float off = 0.f;   // of a fp32 choice value
    if constexpr (!kExact) {
        if constexpr (kBias) off = err + 0x1p-22f * fmaxf(fabsf(lo), fabsf(hi));
        // a place is off by less than three: the sum, the scale, the cut (all of a row by
        // their origin's rounding too, the same)
        const uint32_t apart = 4u + (uint32_t)fminf(2.f * off * scale, 0x1p30f);
        int far = 1, values = 1;   // neighbours are far enough apart; all taken are values
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t mine = k[i] >> kIB, next = (i < 7 ? k[i + 1] : rest) >> kIB;
            // (a value comes before -inf and before nothing)
            far &= (int)(i >= a.k) | (int)(next <= kMaskedPart) | (int)(mine > next + apart);
            values &= (int)(i >= a.k) | (int)(mine > kMaskedPart);
        }
        // one exact value on the whole row is in order of the numbers; -inf is left to route_token
        sure = values & (far | ((int)!kBias & (int)(hi == lo)));
    }
    // lane n's expert: the n-th of the order, lane 8 the best one left out
    uint32_t key = n < 8 ? k[0] : n == 8 ? rest : 0u;
#pragma unroll
    for (int i = 1; i < 8; ++i) key = n == i ? k[i] : key;
    const int id = min((int)(kIds - (key & kIds)), a.E - 1);
    const bool valid = kExact ? (key >> kIB) != 0 && (key >> kIB) != kMaskedPart : (key >> kIB) > kMaskedPart;
    const float l = fminf(load_logit<kL>(a.l, (int64_t)t * a.ld + id), 3.4028234663852886e38f);
    double s = 0.0;   // a sigmoid
    if (a.sigmoid && valid) s = 1.0 / (1.0 + exp(-(double)l));
    int place = n;
    if constexpr (!kExact) {
        if (__any(!sure) && (!kBias || a.sigmoid)) {
            double c = -__builtin_inf();
            if (valid) c = kBias ? s + (double)a.bias[id] : (double)l;
            const int mine = valid ? id : 0x7FFFFFFF;
            int better = 0;
            auto compare = [&](auto ctrl) {
                constexpr int kCtrl = 0x120 + decltype(ctrl)::value;   // row_ror
                const uint64_t b = (uint64_t)__double_as_longlong(c);
                const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, kCtrl, 0xF, 0xF, false);
                const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), kCtrl, 0xF, 0xF, false);
                const int other = __builtin_amdgcn_update_dpp(0, mine, kCtrl, 0xF, 0xF, false);
                const double v = __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
                better += (int)(v > c) | ((int)(v == c) & (int)(other < mine));
            };
            each<15>([&](auto i) { compare(std::integral_constant<int, decltype(i)::value + 1>{}); });
            place = valid ? better : 15;
            double last = valid && better == a.k - 1 ? c : -__builtin_inf();
#pragma unroll
            for (int d = 1; d < 16; d *= 2) last = fmax(last, __shfl_xor(last, d, 64));
            // nothing else that was left out is above this
            const double most = ((double)(rest >> kIB) + 4.0 - (double)from) / (double)scale + (double)off;
            const bool above = (rest >> kIB) <= kMaskedPart ? last > -__builtin_inf() : scale > 0.f && last > most;
            sure = sure || above;
        }
        sure = sure && groups;
    }
    const bool taken = place < a.k && n <= 8;
    const bool counts = taken && valid;
    if (!a.sigmoid) {
        float top = counts ? l : low;
        top = fmaxf(top, from_other<0>(top));
        top = fmaxf(top, from_other<1>(top));
        top = fmaxf(top, from_other<2>(top));
        top = fmaxf(top, from_other<3>(top));
        if (counts) s = exp((double)l - (double)top);
    }
    s = counts ? s : 0.0;
    if (a.renorm) {
        double all = s;
#pragma unroll
        for (int d = 1; d < 16; d *= 2) all += __shfl_xor(all, d, 64);
        s = all > 0.0 ? s / all : 0.0;
    }
    if (taken && sure && t0 + (lane >> 4) < a.T) {
        const int64_t o = (int64_t)t * a.k + place;
        a.w[o] = (float)(s * (double)a.scale);
        if (a.id64) static_cast<int64_t*>(a.ids)[o] = id;
        else static_cast<int32_t*>(a.ids)[o] = id;
    }
    if constexpr (!kExact) {
        const uint64_t unsure = __ballot(!sure);
        for (int i = 0; i < 4; ++i)
            if ((unsure >> (16 * i) & 1) && t0 + i < a.T) {
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                route_token<Q, kL, std::conditional_t<kBias, uint64_t, uint32_t>>(a, t0 + i, lane, scratch[wave]);
            }
    }
}

template <int V, typename K>
void launch(const TopkArgs& a, int dtype, hipStream_t st) {
    const dim3 grid((unsigned)((a.T + kWaves - 1) / kWaves)), block(64 * kWaves);
    if (dtype == kL16b) router_topk_kernel<V, kL16b, K><<<grid, block, 0, st>>>(a);
    else if (dtype == kL16f) router_topk_kernel<V, kL16f, K><<<grid, block, 0, st>>>(a);
    else router_topk_kernel<V, kL32, K><<<grid, block, 0, st>>>(a);
}

template <typename K>
void launch_for(const TopkArgs& a, int dtype, hipStream_t st) {
    if (a.E <= 64) launch<1, K>(a, dtype, st);
    else if (a.E <= 128) launch<2, K>(a, dtype, st);
    else if (a.E <= 256) launch<4, K>(a, dtype, st);
    else if (a.E <= 512) launch<8, K>(a, dtype, st);
    else launch<16, K>(a, dtype, st);
}

template <int V, bool kBias>
void launch_rows(const TopkArgs& a, int dtype, hipStream_t st) {
    const dim3 grid((unsigned)((a.T + 4 * kWaves - 1) / (4 * kWaves))), block(64 * kWaves);
    if (dtype == kL16b) router_topk_rows_kernel<V, kL16b, kBias><<<grid, block, 0, st>>>(a);
    else if (dtype == kL16f) router_topk_rows_kernel<V, kL16f, kBias><<<grid, block, 0, st>>>(a);
    else router_topk_rows_kernel<V, kL32, kBias><<<grid, block, 0, st>>>(a);
}

template <bool kBias>
void launch_rows_for(const TopkArgs& a, int dtype, hipStream_t st) {
    if (a.E <= 64) launch_rows<4, kBias>(a, dtype, st);
    else if (a.E <= 128) launch_rows<8, kBias>(a, dtype, st);
    else if (a.E <= 256) launch_rows<16, kBias>(a, dtype, st);
    else launch_rows<32, kBias>(a, dtype, st);
}

// What the four-token kernel covers: up to eight experts a token, quads that lie
// in one group, and weights that need no sum over the row.
bool rows_cover(const TopkArgs& a) {
    return a.k <= kFastK && a.E <= 512 && (a.G == 1 || (a.G <= kFastGroups && a.per % 4 == 0)) && (a.sigmoid || a.renorm);
}

}  // namespace
}  // namespace kbn

using namespace kbn;

extern "C" int kbn_moe_router_topk(const void* logits, int dtype, int64_t ld, const float* bias, int64_t T, int64_t E,
                                   int64_t top_k, int sigmoid, int64_t num_groups, int64_t topk_groups, int renormalize,
                                   float scale, float* weights, void* ids, int id_bytes, void* stream) {
    const char* what = "moe_router_topk";
    KBN_CHECK_ARG(dtype >= 0 && dtype <= 2, "%s: logits dtype code %d (0 bf16, 1 fp16, 2 fp32)", what, dtype);
    KBN_CHECK_ARG(id_bytes == 4 || id_bytes == 8, "%s: ids of %d bytes (4 or 8)", what, id_bytes);
    KBN_CHECK_ARG(T >= 0 && T <= 0x7FFFFFFFLL, "%s: bad T=%lld", what, (long long)T);
    KBN_CHECK_ARG(E >= 1 && E <= kMaxRouted, "%s: E=%lld outside [1, %d]", what, (long long)E, kMaxRouted);
    KBN_CHECK_ARG(num_groups >= 1 && num_groups <= 64 && E % num_groups == 0,
                  "%s: num_groups=%lld must divide E=%lld and be at most 64", what, (long long)num_groups, (long long)E);
    KBN_CHECK_ARG(topk_groups >= 1 && topk_groups <= num_groups, "%s: topk_groups=%lld outside [1, %lld]", what,
                  (long long)topk_groups, (long long)num_groups);
    KBN_CHECK_ARG(top_k >= 1 && top_k <= 64 && top_k <= topk_groups * (E / num_groups),
                  "%s: top_k=%lld outside [1, 64] or more than the %lld experts of the kept groups", what, (long long)top_k,
                  (long long)(topk_groups * (E / num_groups)));
    KBN_CHECK_ARG(T <= 1 || ld >= E, "%s: row stride %lld is less than E=%lld", what, (long long)ld, (long long)E);
    if (T == 0) return 0;
    KBN_CHECK_ARG(logits && weights && ids, "%s: null pointer", what);
    TopkArgs a{};
    a.l = logits;
    a.ld = ld;
    a.bias = bias;
    a.T = (int)T;
    a.E = (int)E;
    a.k = (int)top_k;
    a.G = (int)num_groups;
    a.kept = (int)topk_groups;
    a.per = (int)(E / num_groups);
    a.per_magic = a.per > 1 ? (uint32_t)(((1ull << 32) + a.per - 1) / a.per) : 0;
    a.sigmoid = sigmoid;
    a.renorm = renormalize;
    a.scale = scale;
    a.w = weights;
    a.ids = ids;
    a.id64 = id_bytes == 8;
    const int64_t size = dtype == kL32 ? 4 : 2;
    a.vec = E % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % (4 * size) == 0 && (T == 1 || ld % 4 == 0);
    a.vec_bias = E % 4 == 0 && aligned16(bias);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (rows_cover(a)) bias ? launch_rows_for<true>(a, dtype, st) : launch_rows_for<false>(a, dtype, st);
    else if (bias) launch_for<uint64_t>(a, dtype, st);
    else launch_for<uint32_t>(a, dtype, st);
    KBN_CHECK_LAUNCH(what);
    return 0;
}
