// The router's product: logits[t, e] = sum_h x[t, h] w[e, h] in fp32.
//
// Few experts (8 to some hundred) and a long sum: what bounds it is reading w
// (few tokens: 1 x 128 x 4096 2.5 us, of which 2.4 are a launch) or x and w by CUs
// that share neither (many: 4096 x 256 x 7168 bf16 24.1 us, 470 MB through 256 CUs
// at 76 B/ns each, 0.62 PFLOP/s; memory alone 13), with weights in fp32 the
// matrix instructions and the barriers of a stage (2051 x 256 x 7168 with bf16 rows
// 36 us, three products each: 0.63 PFLOP/s).  The wavefronts of a workgroup share one tile of
// logits and split its K, unit by unit; each streams whole 128-byte lines of its
// units through a private LDS ring by direct loads, so there is no barrier until
// their sums meet in LDS, in wavefront order.  (Fragments loaded straight into
// the matrix instruction's layout have neighbouring lanes in different rows: 4096
// x 256 x 7168 took 58 us so.)  Where tiles are too few for the CUs, workgroups
// split K as well and a second launch adds their sums in order: the same bits on
// every run.
//
// fp32 operands go through the 16-bit matrix instruction as well: a float is
// the exact sum of three bf16 numbers (8 + 8 + 8 bits of its significand, cut
// off by clearing low bits: the second is below 2^-7 of it, the third below 2^-15).
// Of two such numbers the products of second and third pieces, up to 2^-22 each, are
// left out, always towards 0: up to 2^-21 of a product, 2^-24.7 on average (an fp32
// product's rounding: up to 2^-24).  Products of leading pieces have a sum of their own,
// which alone counts where it is not finite (an infinity's lower pieces are no numbers):
// 1 to 3% of the time, and half of the error.
#include "row_stream.h"

#include <algorithm>

namespace kbn {
namespace {

struct GateArgs {
    const void* x;
    int64_t ld_x;
    const void* w;
    int64_t ld_w;
    float* out;
    int64_t ld_o;
    int T, E, H;
    int splits;      // of K over workgroups
    float* sums;     // [splits, T, E] where splits > 1
};

// A tile of 16 kTM tokens x 16 kTE experts; kDepth stages a wavefront.
template <int kTM, int kTE, int kDepth, int kX, int kW>
__global__ __launch_bounds__(64 * kStreamWaves) void router_gemm_tile_kernel(const GateArgs a) {
    typedef Stream<kTM, kTE, kDepth, kX, kW> St;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[St::kSmem];
    constexpr int bx = bytes_of<kX>(), bw = bytes_of<kW>();
    // workgroups go to the XCDs in turn: the tiles of one block of tokens run on
    // one XCD, whose L2 then reads x once
    const int te = (a.E + 16 * kTE - 1) / (16 * kTE), tt = (a.T + 16 * kTM - 1) / (16 * kTM), across = te * a.splits;
    const int per = blockIdx.x / (8 * across) * 8, width = min(8, tt - per), in = blockIdx.x - per * across;
    const int tile_t = per + in % width, tile_e = in / width / a.splits, split = in / width % a.splits;
    const int t0 = tile_t * 16 * kTM, e0 = tile_e * 16 * kTE;
    const int nt = min(16 * kTM, a.T - t0), ne = min(16 * kTE, a.E - e0);
    const v4i dX = make_desc(static_cast<const uint8_t*>(a.x) + (int64_t)t0 * a.ld_x * bx, ((int64_t)(nt - 1) * a.ld_x + a.H) * bx);
    const v4i dW = make_desc(static_cast<const uint8_t*>(a.w) + (int64_t)e0 * a.ld_w * bw, ((int64_t)(ne - 1) * a.ld_w + a.H) * bw);
    const int units = (a.H + kStreamK - 1) / kStreamK;
    const int from = (int)((int64_t)units * split / a.splits), end = (int)((int64_t)units * (split + 1) / a.splits);
    St::run(dX, dW, [&](int q) { return q < nt ? q * (int)a.ld_x * bx : kOob; },
            [&](int q) { return q < ne ? q * (int)a.ld_w * bw : kOob; }, a.H, from, end, smem);
    float* const out = a.splits > 1 ? a.sums + (int64_t)split * a.T * a.E : a.out;
    const int64_t ld = a.splits > 1 ? a.E : a.ld_o;
    for (int s = threadIdx.x; s < kTM * kTE * 64; s += 64 * kStreamWaves) {
        const f32x4 v = St::sum(smem, s);
        const int l = s & 63, tile = s >> 6;
        const int e = 16 * (tile % kTE) + (l & 15), t = 16 * (tile / kTE) + 4 * (l >> 4);
        if (e < ne) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (t + i < nt) out[(t0 + t + i) * ld + e0 + e] = v[i];
        }
    }
}

// Many tokens and weights in fp32: 128 tokens x 128 experts a workgroup, whose
// wavefronts (64 x 32 each) meet both operands' pieces in LDS.  Each value is taken
// apart once a workgroup, on its way there: a thread has eight values of a row of
// each operand a stage (32 K) and holds those of the next kAhead stages (one, two or three:
// the same times within 3%; of fp16 rows one, with which two workgroups fit a CU's
// registers).  (In the tiles above each wavefront takes its
// own K's values apart: 2051 x 256 x 7168 with fp32 weights 58 us, here 36.)
constexpr int kWideT = 128, kWideE = 128, kWideK = 32, kWideThreads = 512;

template <int kX>
__global__ __launch_bounds__(kWideThreads, kX == kG32 ? 1 : 4) void router_gemm_wide_kernel(const GateArgs a) {
    constexpr int PX = kX == kG32 ? 3 : kX == kG16f ? 2 : 1, PW = 3;
    constexpr int kAhead = kX == kG16f ? 1 : 2;
    constexpr int bx = bytes_of<kX>();
    __shared__ __attribute__((aligned(16))) u32x4 lx[2][PX][kWideT * 4];   // rows of four 16-byte chunks
    __shared__ __attribute__((aligned(16))) u32x4 lw[2][PW][kWideE * 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int te = (a.E + kWideE - 1) / kWideE;
    const int split = blockIdx.x % a.splits, tile_e = blockIdx.x / a.splits % te, tile_t = blockIdx.x / a.splits / te;
    const int t0 = tile_t * kWideT, e0 = tile_e * kWideE;
    const int nt = min(kWideT, a.T - t0), ne = min(kWideE, a.E - e0);
    // a wavefront's 16 rows of each operand
    const int row = tid >> 2, oct = tid & 3, row0 = 16 * wave;
    const __amdgpu_buffer_rsrc_t xr = rsrc(static_cast<const uint8_t*>(a.x) + (int64_t)(t0 + row0) * a.ld_x * bx,
                                           nt > row0 ? (int)(((int64_t)(min(16, nt - row0) - 1) * a.ld_x + a.H) * bx) : 0);
    const __amdgpu_buffer_rsrc_t wr = rsrc(static_cast<const uint8_t*>(a.w) + (int64_t)(e0 + row0) * a.ld_w * 4,
                                           ne > row0 ? (int)(((int64_t)(min(16, ne - row0) - 1) * a.ld_w + a.H) * 4) : 0);
    const int units = (a.H + kWideK - 1) / kWideK;
    const int from = (int)((int64_t)units * split / a.splits), end = (int)((int64_t)units * (split + 1) / a.splits);
    const int xo = row < nt ? (row - row0) * (int)a.ld_x * bx : kOob, wo = row < ne ? (row - row0) * (int)a.ld_w * 4 : kOob;
    const int put = 4 * row + (oct ^ (row >> 1 & 3));   // chunk c of row r lies in slot c ^ (r / 2) % 4
    Raw8<kX> xs[kAhead];
    Raw8<kG32> ws[kAhead];
    // (a stage past the split's end and values past the row's read zeros)
    auto ask = [&](int u, Raw8<kX>& x, Raw8<kG32>& w) __attribute__((always_inline)) {
        const int k = u * kWideK + 8 * oct;
        const bool in = u < end && k < a.H;
        x = load_raw8<kX>(xr, in && xo != kOob ? xo + k * bx : kOob);
        w = load_raw8<kG32>(wr, in && wo != kOob ? wo + k * 4 : kOob);
    };
    auto give = [&](int buf, const Raw8<kX>& x, const Raw8<kG32>& w) __attribute__((always_inline)) {
        const Pieces<PX> px = pieces_of<kX, PX>(x);
        const Pieces<PW> pw = pieces_of<kG32, PW>(w);
#pragma unroll
        for (int i = 0; i < PX; ++i) lx[buf][i][put] = px.p[i];
#pragma unroll
        for (int i = 0; i < PW; ++i) lw[buf][i][put] = pw.p[i];
    };
    f32x4 acc[2][4][2];   // products of leading pieces, of others
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[c][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int tw = 64 * (wave & 1), ew = 32 * (wave >> 1);
    const int fr = lane & 15, at = 4 * fr + ((lane >> 4) ^ (fr >> 1 & 3));   // (16 rows on, the same slot)
    auto products = [&](int buf) __attribute__((always_inline)) {
        u32x4 w[PW][2];
#pragma unroll
        for (int n = 0; n < PW; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) w[n][j] = lw[buf][n][4 * (ew + 16 * j) + at];
#pragma unroll
        for (int m = PX - 1; m >= 0; --m) {   // the smallest products first
            u32x4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = lx[buf][m][4 * (tw + 16 * i) + at];
#pragma unroll
            for (int n = 2 - m; n >= 0; --n) {
                if (n >= PW) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        f32x4& to = acc[m + n > 0 ? 1 : 0][i][j];
                        to = mma<false>(x[i], w[n][j], to);
                    }
            }
        }
    };
#pragma unroll
    for (int d = 0; d < kAhead; ++d) ask(from + d, xs[d], ws[d]);
    give(0, xs[0], ws[0]);
    ask(from + kAhead, xs[0], ws[0]);
    __syncthreads();
    // stage u lies in buffer (u - from) % 2; its successor is given while it is multiplied
    for (int u = from; u < end;) {
#pragma unroll
        for (int d = 1; d <= 2 * kAhead; ++d) {
            if (u >= end) break;
            give(d & 1, xs[d % kAhead], ws[d % kAhead]);
            ask(u + 1 + kAhead, xs[d % kAhead], ws[d % kAhead]);
            products((d - 1) & 1);
            __syncthreads();
            ++u;
        }
    }
    float* const out = a.splits > 1 ? a.sums + (int64_t)split * a.T * a.E : a.out;
    const int64_t ld = a.splits > 1 ? a.E : a.ld_o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const f32x4 v = joined(acc[0][i][j], acc[1][i][j]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int t = tw + 16 * i + 4 * (lane >> 4) + k, e = ew + 16 * j + fr;
                if (t < nt && e < ne) out[(t0 + t) * ld + e0 + e] = v[k];
            }
        }
}

// out = the sums of the splits, in order; eight of them asked for at a time
// (one by one, each waits for the memory: 5.8 us for 16 sums of 61 x 256).
template <int kV>
__device__ __forceinline__ void sum_splits(const float* p, int64_t n, int splits, float (&v)[kV]) {
    typedef float vec __attribute__((ext_vector_type(kV)));
    for (int s0 = 0; s0 < splits; s0 += 8) {
        vec u[8];
#pragma unroll
        for (int s = 0; s < 8; ++s)
            if (s0 + s < splits) u[s] = *reinterpret_cast<const vec*>(p + (s0 + s) * n);
#pragma unroll
        for (int s = 0; s < 8; ++s)
            if (s0 + s < splits) {
#pragma unroll
                for (int k = 0; k < kV; ++k) v[k] = s0 + s == 0 ? u[s][k] : v[k] + u[s][k];
            }
    }
}
template <int kV>
__global__ __launch_bounds__(64) void router_gemm_sum_kernel(const GateArgs a) {
    const int64_t n = (int64_t)a.T * a.E, i = ((int64_t)blockIdx.x * 64 + threadIdx.x) * kV;
    if (i >= n) return;
    float v[kV];
    sum_splits<kV>(a.sums + i, n, a.splits, v);
    const int64_t t = i / a.E, e = i - t * a.E;   // kV divides E
#pragma unroll
    for (int k = 0; k < kV; ++k) a.out[t * a.ld_o + e + k] = v[k];
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

// Most tokens of the rows kernel: past 8 its time grows with the tokens (us for
// 8, 12, 16 tokens and 61 through tiles: 256 x 7168 bf16 4.6, 6.9, 7.0, 7.1; 128 x
// 4096 3.7, 5.3, 5.4, 6.5; fp32 rows 5.5, 9.7, 11.3, 11.7 and 4.0, 6.0, 6.8, 8.2).
constexpr int kRowTokens = 16, kRowTokens32 = 12;

// Tiles of 16 tm x 16 te logits, K in `splits` parts; tm = 0: the rows kernel, 8: the wide one.
struct GatePlan {
    int tm, te, splits;
};

// The second launch of a split product, in ns.
double sum_price(int64_t T, int64_t E, int s) { return s > 1 ? 2400.0 + 200.0 * ((s + 7) / 8) + 60.0 * s + 8.0 * s * T * E / 4000.0 : 0.0; }

// The cheapest of the tile widths and splits by what one takes in ns: the bytes
// of a CU's workgroups, of which a lone CU takes 100 a ns and each of 256 at
// work 80, a price on wide tiles (one workgroup a CU), and with splits the second
// launch.  Fitted to 13 token counts from 4 to 4096 with (256, 7168), (128, 4096) and
// (16, 2048): 1.3% above the best of up to 30 choices on average, 14% at most (512 x
// 256 x 7168: 12.0 us with 32 experts a tile and four splits, 14.7 with 64 and three;
// 2048 tokens 18.8 with 32 and none, 27.4 with 16).
// With fp32 weights the bytes cost more by the work of taking the values apart, by
// the rows' type and the tile's width; the wide kernel goes by what a stage takes a
// lone workgroup of a CU and each two (of fp32 rows LDS holds one).  Fitted to 10
// token counts from 61 to 4096 with those and three more sizes: 1.2% on average, 15%
// at most (2051 x 256 x 7168, wide and not: bf16 rows 34 and 53 us, fp16 44 and 76,
// fp32 51 and 99; 777 x 128 x 4096 bf16 15 and 12; before leading pieces had sums of
// their own, which cost both alike).
GatePlan gate_plan(int64_t T, int64_t E, int64_t H, int xd, int wd) {
    if (T <= (xd == kG32 ? kRowTokens32 : kRowTokens)) return {0, 0, 1};
    const int64_t units = (H + kStreamK - 1) / kStreamK, cus = cu_count();
    const bool apart = wd == kG32;
    const int tm = xd == kG32 ? 2 : 4, most = apart ? 2 : 4;
    const double bx = xd == kG32 ? 4 : 2, bw = apart ? 4 : 2;
    const double slow[3][2] = {{1.13, 1.44}, {1.97, 2.29}, {1.6, 1.81}};   // bf16, fp16, fp32 rows; 16, 32 experts
    GatePlan best{tm, 1, 1};
    double least = 1e30;
    for (int te = 1, i = 0; te <= most; te *= 2, ++i) {
        if (te > 1 && 8 * te >= E) break;
        const int64_t tiles = (T + 16 * tm - 1) / (16 * tm) * ((E + 16 * te - 1) / (16 * te));
        for (const int s : {1, 2, 3, 4, 8, 16, 32}) {
            if (s > 1 && (s > units / kStreamWaves || tiles * s > 2 * cus)) break;
            const double rate = 80.0 + 20.0 * std::max<double>(0.0, 1.0 - (double)(tiles * s) / cus);
            const double ns = (double)((tiles * s + cus - 1) / cus) * (16 * tm * bx + 16 * te * bw) * H / s / rate *
                    (apart ? slow[xd][i] : 1.0) + (apart ? 3900.0 : 900.0 * i) + sum_price(T, E, s);
            if (ns < least) {
                least = ns;
                best = {tm, te, s};
            }
        }
    }
    if (!apart) return best;
    const double start[] = {1000.0, 2900.0, 3900.0}, one[] = {835.0, 1065.0, 1150.0}, two[] = {1120.0, 1550.0, 2300.0};
    const int64_t tiles = (T + kWideT - 1) / kWideT * ((E + kWideE - 1) / kWideE), stages = (H + kWideK - 1) / kWideK;
    for (int s = 1; s <= 32 && 4 * s <= stages && (s == 1 || tiles * s <= 2 * cus); ++s) {
        const int64_t n = (tiles * s + cus - 1) / cus;
        const double ns = start[xd] + (double)stages / s * ((double)(n / 2) * two[xd] + (double)(n % 2) * one[xd]) + sum_price(T, E, s);
        if (ns < least) {
            least = ns;
            best = {8, 8, s};
        }
    }
    return best;
}

template <int kX, int kW>
void launch(GateArgs a, const GatePlan& p, hipStream_t st) {
    if (p.tm == 0) {
        const dim3 grid((unsigned)a.E), block(64 * kRowWaves);
        if (a.T <= 1) router_gemm_rows_kernel<1, kX, kW><<<grid, block, 0, st>>>(a);
        else if (a.T <= 2) router_gemm_rows_kernel<2, kX, kW><<<grid, block, 0, st>>>(a);
        else if (a.T <= 4) router_gemm_rows_kernel<4, kX, kW><<<grid, block, 0, st>>>(a);
        else if (a.T <= 8) router_gemm_rows_kernel<8, kX, kW><<<grid, block, 0, st>>>(a);
        else router_gemm_rows_kernel<16, kX, kW><<<grid, block, 0, st>>>(a);
        return;
    }
    constexpr int kTM = kX == kG32 ? 2 : 4;
    const int64_t tiles = (int64_t)((a.T + 16 * p.tm - 1) / (16 * p.tm)) * ((a.E + 16 * p.te - 1) / (16 * p.te));
    const dim3 grid((unsigned)(tiles * p.splits)), block(64 * kStreamWaves);
    if (p.tm == 8) {
        if constexpr (kW == kG32) router_gemm_wide_kernel<kX><<<grid, dim3(kWideThreads), 0, st>>>(a);
    } else if (p.te == 1) router_gemm_tile_kernel<kTM, 1, 2, kX, kW><<<grid, block, 0, st>>>(a);
    else if (p.te == 2) router_gemm_tile_kernel<kTM, 2, 2, kX, kW><<<grid, block, 0, st>>>(a);
    else if constexpr (kW != kG32) router_gemm_tile_kernel<kTM, 4, 2, kX, kW><<<grid, block, 0, st>>>(a);
    if (p.splits > 1) {
        const int64_t n = (int64_t)a.T * a.E;
        if (a.E % 2 == 0) router_gemm_sum_kernel<2><<<dim3((unsigned)((n + 127) / 128)), dim3(64), 0, st>>>(a);
        else router_gemm_sum_kernel<1><<<dim3((unsigned)((n + 63) / 64)), dim3(64), 0, st>>>(a);
    }
}

bool gate_sizes(int64_t T, int64_t E, int64_t H) {
    return T >= 0 && T < (1 << 24) && E >= 1 && E <= 65536 && H >= 8 && H % 8 == 0 && H <= (1 << 22);
}

}  // namespace
}  // namespace kbn

using namespace kbn;

extern "C" int64_t kbn_moe_router_gemm_workspace_bytes(int64_t T, int64_t E, int64_t H, int x_dtype, int w_dtype) {
    if (!gate_sizes(T, E, H) || x_dtype < 0 || x_dtype > 2 || (w_dtype != x_dtype && w_dtype != kG32)) return -1;
    const GatePlan p = gate_plan(T, E, H, x_dtype, w_dtype);
    return p.splits > 1 ? (int64_t)p.splits * T * E * 4 : 0;
}

extern "C" int kbn_moe_router_gemm(const void* x, int x_dtype, int64_t ld_x, const void* w, int w_dtype, int64_t ld_w,
                                   float* out, int64_t ld_out, int64_t T, int64_t E, int64_t H, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
    const char* what = "moe_router_gemm";
    KBN_CHECK_ARG(x_dtype >= 0 && x_dtype <= 2 && w_dtype >= 0 && w_dtype <= 2,
                  "%s: dtype codes %d and %d (0 bf16, 1 fp16, 2 fp32)", what, x_dtype, w_dtype);
    KBN_CHECK_ARG(w_dtype == x_dtype || w_dtype == kG32, "%s: weights must have the rows' dtype or be fp32", what);
    KBN_CHECK_ARG(H >= 8 && H % 8 == 0 && H <= (1 << 22), "%s: H=%lld must be a multiple of 8 in [8, 2^22]", what, (long long)H);
    KBN_CHECK_ARG(gate_sizes(T, E, H), "%s: bad sizes T=%lld (below 2^24), E=%lld (1 to 65536)", what, (long long)T, (long long)E);
    if (T == 0) return 0;
    KBN_CHECK_ARG(x && w && out, "%s: null pointer", what);
    const int bx = x_dtype == kG32 ? 4 : 2, bw = w_dtype == kG32 ? 4 : 2;
    KBN_CHECK_ARG(aligned16(x) && aligned16(w) && ld_x >= H && ld_w >= H && ld_x * bx % 16 == 0 && ld_w * bw % 16 == 0,
                  "%s: rows must be 16-byte aligned with strides of at least H", what);
    KBN_CHECK_ARG(ld_x < (1 << 23) && ld_w < (1 << 23), "%s: row strides must be below 2^23 elements", what);
    KBN_CHECK_ARG(ld_out >= E && (reinterpret_cast<uintptr_t>(out) & 3u) == 0, "%s: bad output rows", what);
    const GatePlan p = gate_plan(T, E, H, x_dtype, w_dtype);
    const int64_t need = p.splits > 1 ? (int64_t)p.splits * T * E * 4 : 0;
    KBN_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
                  "%s: workspace of %lld bytes, 16-byte aligned, needed", what, (long long)need);
    GateArgs a{x, ld_x, w, ld_w, out, ld_out, (int)T, (int)E, (int)H, p.splits, static_cast<float*>(workspace)};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (x_dtype == kG16b) w_dtype == kG16b ? launch<kG16b, kG16b>(a, p, st) : launch<kG16b, kG32>(a, p, st);
    else if (x_dtype == kG16f) w_dtype == kG16f ? launch<kG16f, kG16f>(a, p, st) : launch<kG16f, kG32>(a, p, st);
    else launch<kG32, kG32>(a, p, st);
    KBN_CHECK_LAUNCH(what);
    return 0;
}
