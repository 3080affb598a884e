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
// One wavefront a token, expert e = lane * V + j in register j, so the lowest
// index of equal keys is the first lane's first register.  Keys are the values'
// bits mapped to unsigned integers of the same order, 0 for taken or absent.
#include "kbn_common.h"

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

// K: uint32_t where c is the logit, uint64_t where it is score + bias.
template <int V, int kL, typename K>
__global__ __launch_bounds__(64 * kWaves) void router_topk_kernel(const TopkArgs a) {
    __shared__ uint64_t choice[kWaves][64 * V];   // used with groups only
    constexpr bool kBias = sizeof(K) == 8;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * kWaves + wave;
    if (t >= a.T) return;   // no barrier follows: each wavefront uses its own part of the LDS
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
        uint64_t* mine = choice[wave];
#pragma unroll
        for (int j = 0; j < V; ++j) mine[lane * V + j] = key[j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        uint64_t rank = 0;
        if (lane < a.G) {
            uint64_t best = 0, second = 0;
            for (int i = 0; i < a.per; ++i) {
                const uint64_t v = mine[lane * a.per + i];
                second = v > best ? best : (v > second ? v : second);
                best = v > best ? v : best;
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
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (bias) launch_for<uint64_t>(a, dtype, st);
    else launch_for<uint32_t>(a, dtype, st);
    KBN_CHECK_LAUNCH(what);
    return 0;
}
