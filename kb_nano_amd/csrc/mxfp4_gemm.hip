// Product of two MXFP4 operands,
//   D[m, n] = bf16( sum_g 2^(ea[m,g] + ew[n,g] - 254) sum_{k in g} a[m,k] w[n,k] ),
// on v_mfma_scale_f32_32x32x64_f8f6f4: a lane's operand is one scale group (32
// codes, 16 bytes) of one row and the instruction takes the group's scale byte,
// so scales cost no arithmetic.
//
// Tiled kernel: WM x WN wavefronts compute a BM x BN tile, four of them for the
// small tiles, of which a CU holds two, eight for the others: with four, 777 x
// 4608 x 7168 takes 25.0 us in 128x128 tiles (20.5 with eight) and 47.1 in 256x256
// (41.4), 4096 x 36864 x 7168 556 (534).
// Codes go from memory to LDS by direct loads in a ring of kStages stages of
// 256 K (128 bytes a row: whole lines, as the L2 serves a half line in the time
// of a whole one, 67 against 133 B/ns for each CU when all read shared data).
// Scale bytes have one buffer of 1024 K, 32 bytes a row: a request takes the L2
// the same time whatever it fetches of a line, and at 512 K a load the scales
// were a third of all requests (2 to 8% of the time, 200 x 8192 x 8192 21.3 ->
// 19.7 us with 64x64 tiles, 4096 x 36864 x 7168 577 -> 571 with 256x256).  A
// stage is four steps of 64 K.  Its one barrier comes where all of it has been
// read and frees it for the loads of the stage kStages ahead, which are spread
// over the MFMA slots behind it.
//
// What bounds it.  Large products: power.  4096 x 36864 x 7168 takes 533 us, 4.06
// PFLOP/s, at the 1.6 to 1.8 GHz that the card then holds; the matrix pipes are
// busy 56% of the cycles, the LDS 30%.  The same instructions alone on random
// operands reach 5.6 to 6 PFLOP/s.
// Smaller ones, 2 to 4 times their floor: not known.  A CU receives 45 B/ns at 200
// x 8192 x 8192 (18.5 us, one 64x128 tile a CU) and 41 at 777 x 4608 x 7168 (24.0, one
// 128x128 tile), a third of the 133 above, and no counted unit is at its limit:
// the matrix pipes are busy 24 and 37% of the cycles, the LDS 25 and 38%, the
// load path's address side 53 and 58%, and its return side, which has a load
// pending in 83 and 82%, moves 30 and 31 bytes in such a cycle.  A deeper ring,
// another row stride and the loads' cache scope change nothing.
#include "mxfp4_gemm.h"

#include "gemm_kernel.h"

namespace kbn {

constexpr int kMxStageK = 256, kMxPairK = 512, kMxScaleK = 1024;

template <int BM, int BN, int kStages, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 2) void mxfp4_gemm_kernel(const MxGemmArgs p) {
    constexpr int kRows = BM + BN, kStage = kRows * 128, kScaleAt = kStages * kStage;
    constexpr int kWaves = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
    constexpr int kDma = kRows / (8 * kWaves);                  // loads of a wavefront per stage: 8 rows each
    constexpr int kScaleDma = (kRows + 32 * kWaves - 1) / (32 * kWaves);   // and per 1024 K of scales: 32 rows each
    static_assert(BM * BN * 2 <= kScaleAt, "epilogue");
    static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0, "a load lies in one operand");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kScaleAt + kRows * 32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;

    int tm, tn, trel, split;
    tile_coords<8>(p.tiles_m, p.tiles_n, 0, p.splits, tm, tn, trel, split);
    const int m0 = tm * BM, n0 = tn * BN;
    const int k_from = split * p.groups_per_split * kMxPairK;
    const int k_len = min(p.K, k_from + p.groups_per_split * kMxPairK) - k_from;
    // The loop has no branches (with one the 256x256 tile's accumulators move
    // between register files): it runs pairs of stages, and what lies past
    // k_len reads as codes and scale bytes of 0, which add nothing.
    const int pairs = (k_len + kMxPairK - 1) / kMxPairK, whole = k_len / kMxStageK;

    // rows past the operand's last read as zeros
    const int rows_a = min(p.M - m0, BM), rows_w = min(p.N - n0, BN);
    const v4i dA = make_desc(p.A + (int64_t)m0 * p.lda + k_from / 2, (rows_a - 1) * p.lda + k_len / 2);
    const v4i dW = make_desc(p.W + (int64_t)n0 * p.ldw + k_from / 2, (rows_w - 1) * p.ldw + k_len / 2);
    const v4i dsA = make_desc(p.sA + (int64_t)m0 * p.ld_sa + k_from / 32, (rows_a - 1) * p.ld_sa + k_len / 32);
    const v4i dsW = make_desc(p.sW + (int64_t)n0 * p.ld_sw + k_from / 32, (rows_w - 1) * p.ld_sw + k_len / 32);

    // Load j of this wavefront: rows 8 q .. 8 q + 7 of the stage, q = kWaves j + wave.
    // 16-byte chunk c of row r lies in slot c ^ swz(r) (the swizzle is applied
    // to the address read, a load's LDS side is contiguous).
    int voff[kDma];
#pragma unroll
    for (int j = 0; j < kDma; ++j) {
        const int r = (kWaves * j + wave) * 8 + (lane >> 3), chunk = (lane & 7) ^ swz(r);
        voff[j] = (j < BM / (8 * kWaves) ? r * (int)p.lda : (r - BM) * (int)p.ldw) + chunk * 16;
    }
    int svoff[kScaleDma];
#pragma unroll
    for (int j = 0; j < kScaleDma; ++j) {
        const int r = ((kWaves * j + wave) * 32 + (lane >> 1)) % kRows;   // some may load the same as another wavefront
        svoff[j] = (r < BM ? r * (int)p.ld_sa : (r - BM) * (int)p.ld_sw) + (lane & 1) * 16;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem, lds = lds0 + (uint32_t)wave * 1024u;

    // Loads of stages past the last fall outside an empty range; in a half stage
    // the lanes of the chunks behind k_len (the same for every j, whose rows
    // differ by multiples of 16) fall outside as well.
    const int behind = ((lane & 7) ^ swz(wave * 8 + (lane >> 3))) >= 4 ? kOob : 0;
    auto issue = [&](uint32_t base, auto j_, int s) {
        constexpr int j = decltype(j_)::value;
        v4i d = j < BM / (8 * kWaves) ? dA : dW;
        if (s * kMxStageK >= k_len) d[2] = 0;
        dma_b128<j * 1024 * kWaves, false>(d, base, voff[j] | (s == whole ? behind : 0), s * 128);
    };
    auto issue_scales = [&](int c) {   // 1024 K
        static_for<kScaleDma>([&](auto j_) {
            constexpr int j = decltype(j_)::value;
            // the 32 rows of one load lie in one operand
            const int q = (kWaves * j + wave) % (kRows / 32);
            v4i d = q < BM / 32 ? dsA : dsW;
            if (c * kMxScaleK >= k_len) d[2] = 0;
            dma_b128<kScaleAt, false>(d, lds0 + (uint32_t)q * 1024u, svoff[j], c * 32);
        });
    };

    // fragment f (A: f < FM, W: f - FM) of step ks of the stage at LDS offset `at`
    const int half = lane >> 5, ra = wm * TM + (lane & 31), rw = BM + wn * TN + (lane & 31);
    auto read_frag = [&](int at, int ks, int f) -> u32x4 {
        const int r = f < FM ? ra : rw;   // the swizzle is the same 32 rows on
        return *reinterpret_cast<const u32x4*>(smem + at + r * 128 + (((2 * ks + half) ^ swz(r)) << 4) + (f < FM ? f : f - FM) * 4096);
    };
    auto read_scale = [&](int o, int f) -> u32x4 {
        return *reinterpret_cast<const u32x4*>(smem + kScaleAt + (f < FM ? ra : rw) * 32 + (o & 1) * 16 + (f < FM ? f : f - FM) * 1024);
    };

    // The large tile reads the fragments of one step ahead, under the 8 MFMAs
    // (256 cycles) of a step.  A smaller one's step is over before the reads of
    // the next are back, so it reads a whole stage ahead.
    constexpr bool kWhole = FM + FN <= 4;
    v16f acc[FM][FN] = {};
    constexpr int kR = FM + FN, kT = FM * FN;
    u32x4 f[kWhole ? 8 : 2][kR], raw[kR];
    uint32_t sc[kR][4];   // dword: 128 K of the 512; byte 0 for the first 64 of them, byte 2 for the second
    auto mfma_at = [&](int t, const u32x4 (&f)[kR], auto step_) {   // step of 64 K within the 512
        constexpr int step = decltype(step_)::value, op = (step & 1) * 2;
        const int i = t / FN, j = t % FN;
        const v8i a = {(int)f[i].x, (int)f[i].y, (int)f[i].z, (int)f[i].w}, w = {(int)f[FM + j].x, (int)f[FM + j].y, (int)f[FM + j].z, (int)f[FM + j].w};
        // W as the first operand: a lane then holds runs of four columns of one row
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, acc[i][j], 4, 4, op, (int)sc[FM + j][step >> 1], op,
                                                                      (int)sc[i][step >> 1]);
        keep_here<false>(acc[i][j][0]);
    };

    issue_scales(0);
    static_for<kStages>([&](auto b_) {
        static_for<kDma>([&](auto j_) { issue(lds + decltype(b_)::value * kStage, j_, decltype(b_)::value); });
    });
    wait_dma_n<(kStages - 1) * kDma>();
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kR; ++q) {
#pragma unroll
        for (int ks = 0; ks < (kWhole ? 4 : 1); ++ks) f[ks][q] = read_frag(0, ks, q);
        raw[q] = read_scale(0, q);
    }

    int at = 0;   // LDS offset of the current stage
    // Stage s + 1 has landed; in flight behind it: kStages - 2 stages.  All of
    // stage s is read: its buffer is free.  Returns the LDS address that the
    // stage kStages ahead goes to.  The scales' one buffer is free once the
    // second pair's bytes are in registers: the next 1024 K are asked for in
    // the third stage of four and have landed, ahead of that stage's codes, a
    // stage later.
    auto turn = [&](auto par_, int s) -> uint32_t {
        constexpr int par = decltype(par_)::value;
        wait_dma_n<(par == 1 && kStages > 3 ? 1 : kStages - 2) * kDma>();
        wait_lds();
        __syncthreads();
        if (par == 0 && (s & 2)) issue_scales(s / 4 + 1);
        const uint32_t base = lds + (uint32_t)at;
        at = at == (kStages - 1) * kStage ? 0 : at + kStage;
        return base;
    };
    // loads of the stage kStages ahead that go to slot t of n
    auto refill = [&](uint32_t base, auto t_, auto n_, int s) {
        constexpr int u0 = decltype(t_)::value * kDma / decltype(n_)::value, u1 = (decltype(t_)::value + 1) * kDma / decltype(n_)::value;
        static_for<u1 - u0>([&](auto u_) { issue(base, std::integral_constant<int, u0 + decltype(u_)::value>{}, s + kStages); });
    };
    auto stage = [&](auto par_, int s) {
        constexpr int par = decltype(par_)::value;
        if constexpr (kWhole) {
            const uint32_t base = turn(par_, s);
            constexpr int kReads = 4 * kR, kAt = (kReads + 3 * kT - 1) / (3 * kT);   // all in the first three steps
            static_for<4 * kT>([&](auto t_) {
                constexpr int t = decltype(t_)::value;
                mfma_at(t % kT, f[4 * par + t / kT], std::integral_constant<int, 4 * par + t / kT>{});
#pragma unroll
                for (int q = t * kAt; q < (t + 1) * kAt && q < kReads; ++q) f[4 * (1 - par) + q / kR][q % kR] = read_frag(at, q / kR, q % kR);
                if constexpr (par == 1 && t < kR) raw[t] = read_scale(s / 2 + 1, t);
                refill(base, t_, std::integral_constant<int, 4 * kT>{}, s);
                __builtin_amdgcn_sched_barrier(0);
            });
        } else {
            constexpr int kAt = kT >= 2 * kR ? 1 : (2 * kR + kT - 1) / kT;   // reads in a slot
            static_for<3>([&](auto ks_) {
                constexpr int ks = decltype(ks_)::value;
#pragma unroll
                for (int t = 0; t < kT; ++t) {
                    mfma_at(t, f[ks & 1], std::integral_constant<int, 4 * par + ks>{});
#pragma unroll
                    for (int q = t * kAt; q < (t + 1) * kAt && q < kR; ++q) f[1 - (ks & 1)][q] = read_frag(at, ks + 1, q);
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
            const uint32_t base = turn(par_, s);
            static_for<kT>([&](auto t_) {
                constexpr int t = decltype(t_)::value;
                mfma_at(t, f[1], std::integral_constant<int, 4 * par + 3>{});
#pragma unroll
                for (int q = t * kAt; q < (t + 1) * kAt && q < kR; ++q) {
                    f[0][q] = read_frag(at, 0, q);
                    if constexpr (par == 1) raw[q] = read_scale(s / 2 + 1, q);
                }
                refill(base, t_, std::integral_constant<int, kT>{}, s);
                __builtin_amdgcn_sched_barrier(0);
            });
        }
    };
    for (int o = 0; o < pairs; ++o) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // bytes behind k_len are another row's, perhaps a NaN's
            const uint32_t m = o * kMxPairK + i * 128 < k_len ? ~0u : 0u;
#pragma unroll
            for (int q = 0; q < kR; ++q) sc[q][i] = (raw[q][i] & m) >> (8 * half);
        }
        stage(std::integral_constant<int, 0>{}, 2 * o);
        stage(std::integral_constant<int, 1>{}, 2 * o + 1);
    }
    wait_dma();        // the loads past the end still write to this workgroup's LDS
    __syncthreads();

    if (p.splits > 1) {
        float* slab = p.P + ((int64_t)split * p.tiles_m * p.tiles_n + trel) * (BM * BN);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int r = wm * TM + i * 32 + (lane & 31);
            if (m0 + r >= p.M) continue;
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = wn * TN + j * 32 + 8 * q + 4 * half;
                    *reinterpret_cast<u32x4*>(slab + r * BN + c) =
                        u32x4{__float_as_uint(acc[i][j][4 * q]), __float_as_uint(acc[i][j][4 * q + 1]),
                              __float_as_uint(acc[i][j][4 * q + 2]), __float_as_uint(acc[i][j][4 * q + 3])};
                }
        }
        return;
    }
    // bf16 through LDS, so that rows leave as whole lines: each wavefront parks
    // its block row-major, 16-byte chunks rotated by the row (no two of the 32
    // rows written at once then share more than their fair share of banks)
    constexpr int kCh = TN / 8, kRowsPer = 64 / kCh;
    uint8_t* reg = smem + wave * (TM * TN * 2);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int r = i * 32 + (lane & 31);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<u32x2*>(reg + r * (TN * 2) + ((4 * j + q + r) % kCh) * 16 + 8 * half) =
                    u32x2{pack_bf16(acc[i][j][4 * q], acc[i][j][4 * q + 1]), pack_bf16(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3])};
        __builtin_amdgcn_sched_barrier(0);   // one fragment row's registers at a time
    }
    wait_lds();
    const bool lines = p.N % 8 == 0 && p.ldd % 8 == 0 && (reinterpret_cast<uintptr_t>(p.D) & 15) == 0;
    const int cl = lane % kCh, n = n0 + wn * TN + cl * 8;
#pragma unroll 4
    for (int it = 0; it < TM / kRowsPer; ++it) {
        const int r = it * kRowsPer + lane / kCh, m = m0 + wm * TM + r;
        if (m >= p.M) continue;
        const u32x4 v = *reinterpret_cast<const u32x4*>(reg + r * (TN * 2) + ((cl + r) % kCh) * 16);
        uint16_t* d = p.D + (int64_t)m * p.ldd + n;
        if (lines) {
            if (n < p.N) *reinterpret_cast<u32x4*>(d) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < p.N) d[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
        }
    }
}

// D = bf16 of the splits' partial sums, added in their order; a lane takes four columns.
template <int BM, int BN>
__global__ __launch_bounds__(256) void mxfp4_sum_kernel(const MxGemmArgs p) {
    const int tiles = p.tiles_m * p.tiles_n;
    constexpr int kRuns = BN / 4;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;   // (tile row of a tile, run of four columns)
    const int run = (int)(at % kRuns), r = (int)(at / kRuns % BM);
    const int64_t t = at / (kRuns * BM);
    if (t >= tiles) return;
    // the tile order of the product's workgroups, without their XCD placement
    const int group = 8 * p.tiles_n, g = (int)t / group, first = g * 8, gm = min(p.tiles_m - first, 8), w = (int)t - g * group;
    const int m = (first + w % gm) * BM + r, n = (w / gm) * BN + run * 4;
    if (m >= p.M || n >= p.N) return;
    const float* s = p.P + (t * BM + r) * BN + run * 4;
    float v[4] = {};
    for (int i = 0; i < p.splits; ++i) {
        const u32x4 q = *reinterpret_cast<const u32x4*>(s + (int64_t)i * tiles * (BM * BN));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += __uint_as_float(q[e]);
    }
    uint16_t* d = p.D + (int64_t)m * p.ldd + n;
    if (n + 4 <= p.N && p.ldd % 4 == 0 && (reinterpret_cast<uintptr_t>(p.D) & 7) == 0) {
        *reinterpret_cast<u32x2*>(d) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < p.N) d[e] = (uint16_t)pack_bf16(v[e], 0.0f);
    }
}

template <int BM, int BN, int kStages, int WM, int WN>
static int launch_tiled(MxGemmArgs& p, const MxPlan& plan, float* slabs, hipStream_t st) {
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + BN - 1) / BN;
    const int groups = (p.K + kMxPairK - 1) / kMxPairK;
    p.groups_per_split = (groups + plan.splits - 1) / plan.splits;
    p.splits = (groups + p.groups_per_split - 1) / p.groups_per_split;
    p.P = slabs;
    mxfp4_gemm_kernel<BM, BN, kStages, WM, WN><<<p.tiles_m * p.tiles_n * p.splits, WM * WN * 64, 0, st>>>(p);
    KBN_CHECK_LAUNCH("mxfp4_gemm_nt");
    if (p.splits > 1) {
        const int64_t lanes = (int64_t)p.tiles_m * p.tiles_n * BM * (BN / 4);
        mxfp4_sum_kernel<BM, BN><<<(unsigned)((lanes + 255) / 256), 256, 0, st>>>(p);
        KBN_CHECK_LAUNCH("mxfp4_gemm_nt");
    }
    return 0;
}

// Prices, in us, of the tiles: fixed cost, a further round of workgroups, a
// stage of 256 K where each CU has one workgroup, one where it has several (a
// workgroup's share), fitted to 96 shapes (M 20 .. 4096, eight weights) and four
// split counts timed in graphs; 14% off each, but the tile picked is 0.3%
// slower than the best one on average, 6% at most.  Those are the shapes it was
// fitted to; on 47 random ones of other weights (M 17 .. 4096, N 300 .. 40000, K 256
// .. 19200) 0.5% on average and 11% at most, where K is 256 or 512 (1832 x 2478 x 256
// 16.5 / 14.8).  Known to be off by more: 64 x 10240 x 8192 takes 64x64 tiles, 18.1
// against 15.4 with 48 weight rows a workgroup.  Each tile carries shapes (us
// with 64x64, 64x128, 128x128, 128x256, 256x256): 320 x 1000 x 4096 7.19 / 8.94 / 11.2 / 16.9 / 24.9, 65 x 24576 x
// 1536 9.58 / 8.61 / 8.24 / 10 / 13.5, 777 x 4608 x 7168 28.7 / 23.3 / 20.1 / 26.1 / 41.8, 777 x 8192 x 8192 60.4 / 50 / 43.1 / 35.5 / 49.8, 4096 x 36864 x
// 7168 1.17e+03 / 919 / 824 / 667 / 547.
struct TilePrice {
    int bm, bn, per_cu;
    double fixed, round, stage_one, stage_many;
};
static const TilePrice kTiles[] = {
    {64, 64, 2, 3.07, 0.975, 0.275, 0.275},
    {64, 128, 2, 3.03, 1.45, 0.458, 0.407},
    {128, 128, 1, 3.37, 1.81, 0.555, 0.655},
    {128, 256, 1, 4.6, 4.3, 0.758, 0.835},
    {256, 256, 1, 6.74, 4.43, 1.25, 1.42},
};
// the sum's launch, and each MB of partial sums, which go through memory
constexpr double kSplitFixed = 3.0, kSplitMb = 0.35;

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

MxPlan mxfp4_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t groups = ceil_div(K, kMxPairK), cus = cu_count();
    MxPlan best{};
    double price = 1e30;
    if (M <= 64) {
        // The few-rows kernel is bound by what each CU reads: 16 (rf + cg) rows
        // a workgroup, K in pairs of stages of each wavefront; fitted to 70
        // shapes, 12% off, the variant picked 0.5% slower than the best one on
        // average.  us with rf 1 / 2 / 3 / 4: M = 64, 2048 x 2048 4.4 / 5.2 / 6.0 / 6.9,
        // 8192 x 8192 18.4 / 13.0 / 14.6 / 16.5, 10240 x 8192 25.6 / 20.8 / 15.0 / 17.0;
        // M = 1, 2.8 / 3.1 / 3.5 / 4.4, 8.3 / 8.5 / 9.8 / 11.4, 11.0 / 11.9 / 10.6 / 10.9,
        // 36864 x 7168 25.6 / 27.1 / 23.7 / 30.4.  Against the best tile, M = 20 and 64:
        // 8192 x 8192 9.7 and 13.0 (12.4 and 13.4), 8192 x 28672 29.1 and 38.7
        // (28.1 and 30.4).
        const int64_t cg = ceil_div(M, 16), stages = 8 * ceil_div(ceil_div(K, 256), 8);
        for (int rf = 1; rf <= (cg < 4 ? 4 : 3); ++rf) {
            const int64_t rounds = ceil_div(ceil_div(N, 16 * rf), cus);
            const double t = 2.5 + 0.33 * (rounds - 1) + (0.06 * rf + 0.044 * cg) * stages * rounds;
            if (t < price) {
                price = t;
                best = {0, 0, 1, rf};
            }
        }
        if (M <= 16) return best;
    }
    for (const TilePrice& t : kTiles) {
        const int64_t tiles_m = ceil_div(M, t.bm), tiles = tiles_m * ceil_div(N, t.bn);
        const double cold = tiles_m == 1 ? 1.1 : 1.0;   // one row of tiles: every weight line comes from memory
        for (int splits = 1; splits <= 4 && splits <= groups; ++splits) {
            const int64_t per = ceil_div(groups, splits), used = ceil_div(groups, per);
            if (used != splits) continue;
            const int64_t q = ceil_div(tiles * splits, cus), stages = 2 * per;
            double us = t.fixed + t.round * (ceil_div(q, t.per_cu) - 1) +
                        cold * (q == 1 ? t.stage_one * stages : t.stage_many * stages * q);
            if (splits > 1) us += kSplitFixed + kSplitMb * 4e-6 * (double)(tiles * t.bm * t.bn * splits);
            if (us < price) {
                price = us;
                best = {t.bm, t.bn, splits, 0};
            }
        }
    }
    return best;
}

int64_t mxfp4_plan_bytes(const MxPlan& p, int64_t M, int64_t N) {
    return p.rf || p.splits == 1 ? 0 : ceil_div(M, p.bm) * ceil_div(N, p.bn) * p.bm * p.bn * 4 * p.splits;
}

int mxfp4_gemm_launch(MxGemmArgs& p, float* slabs, hipStream_t st) {
    const MxPlan plan = mxfp4_plan(p.M, p.N, p.K);
    if (plan.rf) return mxfp4_rows_launch(p, plan.rf, kMxBf16, st);
    if (plan.bm == 256) return launch_tiled<256, 256, 2, 2, 4>(p, plan, slabs, st);
    if (plan.bn == 256) return launch_tiled<128, 256, 3, 2, 4>(p, plan, slabs, st);
    if (plan.bm == 128) return launch_tiled<128, 128, 4, 4, 2>(p, plan, slabs, st);
    if (plan.bn == 128) return launch_tiled<64, 128, 3, 2, 2>(p, plan, slabs, st);
    return launch_tiled<64, 64, 4, 2, 2>(p, plan, slabs, st);
}

}  // namespace kbn
