// The experts' products over rows sorted by expert, with group sizes known only on the GPU:
//     forward   y[r]  = W[e] x[r]             m = rows of e, n = out, k = in
//     dgrad     dx[r] = W[e]^T dy[r]          m = rows of e, n = in,  k = out
//     wgrad     dw[e] = sum_r dy[r] x[r]^T    m = out,       n = in,  k = rows of e
// as T x T tiles of the bf16 MFMA with fp32 accumulators.  The grid is an upper bound that depends
// on the number of rows alone; each work-group finds its group and tile from the offsets.
//
// Row-major operands: x and dy of the row products, W of the forward one; K-major: W of dgrad, both operands of
// wgrad (slabs.hpp).  Groups end anywhere: what a slab has beyond the group's rows or beyond K reads as zeros, so no
// element of another group, of a spare row or of what follows a tensor meets a product.
#include "slabs.hpp"
#include "../../include/muon_sr_amd.h"

namespace msr {

enum : int { EX_FWD = 0, EX_DGRAD = 1, EX_WGRAD = 2 };

struct ExpertArgs {
    const uint16_t *P;           // x (forward), dy (dgrad, wgrad): the operand of m
    int64_t ldp;
    const uint16_t *Q;           // W (forward, dgrad), x (wgrad): the operand of n
    int64_t ldq;                 // row length of one expert's W, or x's row stride
    uint16_t *D;                 // y, dx [rows][n], or dw / acc [experts][m][n]
    const int32_t *offsets;
    int32_t rows, experts, M, N, K;    // M: wgrad only; K: not wgrad
    int32_t tiles_n, zero_init, by_size;
    Noise ns;
};

// First row of group e: experts, then the rows without one (e = experts).
__device__ __forceinline__ int group_row(const ExpertArgs &a, int e) {
    return e <= 0 ? 0 : e > a.experts ? a.rows : min(max(a.offsets[e], 0), a.rows);
}

constexpr int X_SORT = 512;                  // rows per expert from which the order of experts pays for finding it
// Tile rows that share a walk over the columns (forward, 16384 rows over 8 experts of 4096 x 4096, 256-wide tiles:
// 555 us with 4, 531 with 8; the smaller tiles and the weight gradients lose 0 to 5 % with 8).
constexpr int x_group(int kind, int T) { return kind != EX_WGRAD && T == 256 ? 8 : 4; }

// The group, first row and column of tile v, over the E + 1 groups' tile rows (false: no such tile).  Every wave finds
// it by itself: lane l adds the tile rows of c consecutive groups, a sum over the lanes gives the number of all and the lane
// that holds the tile, and, where c > 1, the lanes then take that lane's groups one each.  Numbering the tiles without
// sums (group g from lo / T + g on, which needs its own offset only) leaves tiles out that nothing fills: it was 0.7 us
// faster for 8 experts and up to 40 % slower for 64, whose XCDs then differ in work.
template <int T>
__device__ __forceinline__ bool find_rows(const ExpertArgs &a, int v, int &e, int &lo, int &hi, int &m0, int &nt) {
    const int lane = threadIdx.x & 63, c = (a.experts + 64) / 64;
    auto tiles = [](int from, int to) __attribute__((always_inline)) { return (max(0, to - from) + T - 1) / T; };
    int n = 0, at = group_row(a, lane * c);
#pragma unroll 4
    for (int i = 0; i < c; ++i) {
        const int next = group_row(a, lane * c + i + 1);
        n += tiles(at, next);
        at = next;
    }
    int to = wave_scan(n);
    const int mt = __builtin_amdgcn_readlane(to, 63), total = mt * a.tiles_n;
    if (v >= total || mt > a.rows / T + a.experts + 1) return false;   // (offsets that do not ascend: too many)
    // Consecutive work-groups go to the 8 XCDs in turn: each XCD takes a contiguous eighth of the
    // tiles, whose operands its L2 shares
    const int per = total / NXCD;
    if (v < per * NXCD) v = (v % NXCD) * per + v / NXCD;
    constexpr int G = x_group(EX_FWD, T);
    const int pg = G * a.tiles_n, g = v / pg, first = G * g, rows = min(G, mt - first), r = v - g * pg;
    int t = first + r % rows;
    nt = r / rows;
    int l = __builtin_ctzll(__ballot(to > t) | 1ull << 63);
    t -= __builtin_amdgcn_readlane(to - n, l);
    e = l * c;
    if (c > 1) {
        n = lane < c ? tiles(group_row(a, e + lane), group_row(a, e + lane + 1)) : 0;
        to = wave_scan(n);
        l = __builtin_ctzll(__ballot(to > t) | 1ull << 63);
        t -= __builtin_amdgcn_readlane(to - n, l);
        e += l;
    }
    lo = __builtin_amdgcn_readfirstlane(group_row(a, e));
    hi = __builtin_amdgcn_readfirstlane(group_row(a, e + 1));
    m0 = t * T;
    return t >= 0 && (int64_t)t * T < hi - lo;   // (and no tile outside a group)
}

// The expert with the q-th most rows (at most 64 experts): the last tiles to run are then short ones.
__device__ __forceinline__ int by_size(const ExpertArgs &a, int q) {
    const int lane = threadIdx.x & 63;
    const int n = lane < a.experts ? max(0, group_row(a, lane + 1) - group_row(a, lane)) : -1;
    int rank = 0;
    for (int l = 0; l < a.experts; ++l) {
        const int o = __builtin_amdgcn_readlane(n, l);
        rank += o > n || (o == n && l < lane) ? 1 : 0;
    }
    return __builtin_ctzll(__ballot(lane < a.experts && rank == q));
}

// T: tile; MODE: noise mode of the accumulation, or -1 for a plain store; BK: k per slab; S: LDS stages; WPS: waves per SIMD
// that the registers leave room for.
// KG: groups of waves that take consecutive shares of K each, joined through LDS in their order at the end.
template <int KIND, int MODE, int T, int BK, int S_, int WPS, int KG = 1>
__global__ __launch_bounds__(64 * Shape<T>::NW * KG, WPS) void experts_kernel(ExpertArgs a) {
    using S = Shape<T>;
    constexpr int NW = S::NW, FM = S::FM, FN = S::FN;
    constexpr bool PK = KIND == EX_WGRAD, QK = KIND != EX_FWD;
    using PR = Product<T, BK, S_, PK, QK>;
    using SP = typename PR::SP;
    using SQ = typename PR::SQ;
    // one variable per stage and operand, so that the compiler knows that fragment reads of one
    // stage do not alias the loads into the others
    constexpr int PB = SP::BYTES * KG, QB = SQ::BYTES * KG;
    __shared__ __attribute__((aligned(1024))) char p_0[PB], p_1[PB], q_0[QB], q_1[QB];
    __shared__ __attribute__((aligned(1024))) char p_2[S_ > 2 ? PB : 16], q_2[S_ > 2 ? QB : 16];
    __shared__ __attribute__((aligned(1024))) char p_3[S_ > 3 ? PB : 16], q_3[S_ > 3 ? QB : 16];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6), kg = KG > 1 ? wid / NW : 0, wave = KG > 1 ? wid % NW : wid;
    const int wm = wave / S::WN, wn = wave % S::WN;
    int e = 0, lo = 0, hi = 0, m0 = 0, nt = 0, M, K;
    if constexpr (KIND == EX_WGRAD) {
        // Consecutive work-groups go to the 8 XCDs in turn: each XCD takes a contiguous eighth of every
        // expert's tiles, as experts differ in rows and so their tiles in time (16384 rows over 8 experts of
        // 4096 x 4096, 256-wide tiles: 1054 us with an eighth of all tiles, nearly one expert, per XCD, 487 us so)
        const int tiles_m = (a.M + T - 1) / T, tiles = tiles_m * a.tiles_n, per = (tiles + NXCD - 1) / NXCD;
        const int x = blockIdx.x / NXCD;
        e = a.by_size ? by_size(a, x / per) : x / per;
        const int v = (blockIdx.x % NXCD) * per + x % per;
        if (v >= tiles) return;
        constexpr int G = x_group(EX_WGRAD, T);
        const int pg = G * a.tiles_n, g = v / pg, first = G * g, rows = min(G, tiles_m - first), r = v - g * pg;
        m0 = (first + r % rows) * T;
        nt = r / rows;
        lo = __builtin_amdgcn_readfirstlane(group_row(a, e));
        hi = __builtin_amdgcn_readfirstlane(max(lo, group_row(a, e + 1)));
        M = a.M;
        K = hi - lo;
        if (MODE >= 0 && K == 0 && !a.zero_init) return;   // nothing to add
    } else {
        if (!find_rows<T>(a, blockIdx.x, e, lo, hi, m0, nt)) return;
        M = hi - lo;
        K = e < a.experts ? a.K : 0;                       // rows without an expert: zeros
    }
    const int n0 = nt * T;
    const uint16_t *const P = KIND == EX_WGRAD ? a.P + (int64_t)lo * a.ldp + m0 : a.P + (int64_t)(lo + m0) * a.ldp;
    const uint16_t *const Q = KIND == EX_WGRAD  ? a.Q + (int64_t)lo * a.ldq + n0
                              : KIND == EX_FWD ? a.Q + (int64_t)e * a.N * a.K + (int64_t)n0 * a.ldq
                                               : a.Q + (int64_t)e * a.N * a.K + n0;
    const int mrows = min(T, M - m0), nrows = min(T, a.N - n0);

    PR pr;
    pr.init(wave, lane, a.ldp, a.ldq);
    f32x16_t (&acc)[FM][FN] = pr.acc;

    // The accumulator's first PRE row blocks of the wave, as its epilogue takes them: 16 bytes at row crow +
    // RPP y of a block, loaded ahead of the products
    constexpr int WC = S::TN / 8, RPP = 64 / WC, NP = 32 / RPP;   // chunks per row, rows per access, accesses per block
    constexpr int PRE = MODE >= 0 ? FM < 4 ? 1 : 2 : 0;
    u32x4_t old[PRE ? PRE : 1][NP];
    auto fetch = [&](u32x4_t (&c)[NP], int i, int ln) __attribute__((always_inline)) {
        const int n = n0 + wn * S::TN + 8 * (ln % WC);
#pragma unroll
        for (int y = 0; y < NP; ++y) {
            const int m = m0 + wm * S::TM + 32 * i + ln / WC + RPP * y;
            c[y] = u32x4_t{0u, 0u, 0u, 0u};
            if (m < M && n < a.N && !a.zero_init) c[y] = ld_nt4(a.D + ((int64_t)e * M + m) * a.N + n);
        }
    };

    auto lds_p = [&](auto ST) __attribute__((always_inline)) -> char * {
        constexpr int st = decltype(ST)::value;
        return (st == 0 ? p_0 : st == 1 ? p_1 : st == 2 ? p_2 : p_3) + kg * SP::BYTES;
    };
    auto lds_q = [&](auto ST) __attribute__((always_inline)) -> char * {
        constexpr int st = decltype(ST)::value;
        return (st == 0 ? q_0 : st == 1 ? q_1 : st == 2 ? q_2 : q_3) + kg * SQ::BYTES;
    };
    // this group's share of K: `slabs` of them from kb on
    const int slabs = ((K + BK - 1) / BK + KG - 1) / KG, kb = kg * slabs * BK, kend = min(K, kb + slabs * BK);
    if constexpr (PRE > 0) fetch(old[0], 0, lane);
    if constexpr (PRE > 1) fetch(old[1], 1, lane);
    pr.run(lds_p, lds_q, {P, a.ldp, mrows, M - m0, kend}, {Q, a.ldq, nrows, a.N - n0, kend}, kb, K > 0 ? slabs : 0);

    // ---------------- epilogue ----------------
    // Outputs and accumulators pass through once, non-temporal: kept out of the caches they leave room for the
    // operands (weight gradients of 16411 rows over 64 experts of 1024 x 2048: 128 us with plain stores, 103 so;
    // accumulated 171 and 154).  Each wave stages its sub-tile through LDS of its own, one 32-row block at a
    // time (LDS accesses of one wave execute in order).  Lane l holds D[m = l % 32][n = 8 r + 4 (l / 32) + q] of each
    // 32 x 32 block.
    constexpr int EP = S::TN + 8;                              // staging row pitch (16-byte rows)
    constexpr int PER = PB / (32 * EP * 2);                    // waves that stage in one variable
    static_assert(SP::BYTES == SQ::BYTES && PER > 0 && NW <= 4 * PER, "the staging fits the first two stages");
    const int sv = wave / PER;
    char *const wst = (KG > 1 ? p_1 : sv == 0 ? p_0 : sv == 1 ? q_0 : sv == 2 ? p_1 : q_1) + (wave % PER) * (32 * EP * 2);
    auto est = [&](int row) __attribute__((always_inline)) { return reinterpret_cast<uint16_t *>(wst + row * (EP * 2)); };
    // lane indices from an opaque copy of the thread index: the addresses are formed here, not kept
    // through the K loop
    int etid = tid;
    asm volatile("" : "+v"(etid));
    const int elane = etid & 63, r32 = elane & 31, khalf = elane >> 5, crow = elane / WC, cchk = elane % WC;
    const int n = n0 + wn * S::TN + 8 * cchk;
    wait_vm<0>();                                              // no load writes LDS any more
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if constexpr (KG > 1) {
        // groups 1, 2, .. leave their sums in the first stage (16 floats per lane, 16 KiB per group), group 0 adds
        // them in that order and stores
        static_assert(T == 64 && PB >= KG * 8192 && PER >= NW, "the sums fit the first stage, the staging the second");
        auto part = [&](int g, int i) __attribute__((always_inline)) {
            char *const b = (g <= KG / 2 ? p_0 : q_0) + ((g - 1) % (KG / 2)) * 16384;
            return reinterpret_cast<float *>(b) + (i * NW + wave) * 64 + lane;
        };
        if (kg > 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) *part(kg, i) = acc[0][0][i];
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int g = 1; g < KG; ++g)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[0][0][i] = acc[0][0][i] + *part(g, i);
    }
    u32x4_t late[PRE && FM > PRE ? FM - PRE : 1][NP];
    if constexpr (PRE > 0 && FM > PRE) {
        fetch(late[0], PRE, elane);
        if constexpr (FM > PRE + 1) fetch(late[1], PRE + 1, elane);
    }
    auto block = [&](auto I) __attribute__((always_inline)) {
        constexpr int i = decltype(I)::value;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<uint2 *>(est(r32) + j * 32 + 8 * r + 4 * khalf) =
                    make_uint2(rne_bf16x2(acc[i][j][4 * r], acc[i][j][4 * r + 1]), rne_bf16x2(acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]));
        const int mb = m0 + wm * S::TM + 32 * i + crow;
        if constexpr (MODE >= 0) {
            u32x4_t (&c)[NP] = i < PRE ? old[i < PRE ? i : 0] : late[i < PRE ? 0 : i - PRE];
#pragma unroll
            for (int y = 0; y < NP; ++y) {
                const int m = mb + RPP * y;
                const int64_t o0 = ((int64_t)e * M + m) * a.N + n;
                const uint4 w = *reinterpret_cast<const uint4 *>(est(crow + RPP * y) + 8 * cchk);
                if (m < M && n < a.N) {
                    const uint32_t gw[4] = {w.x, w.y, w.z, w.w}, cw[4] = {c[y].x, c[y].y, c[y].z, c[y].w};
                    uint32_t rn[8], o[4];
                    noise8<MODE>(a.ns, o0, 8, rn);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        o[q] = pack2(sr_bf16(bf16_lo(cw[q]) + bf16_lo(gw[q]), rn[2 * q]),
                                     sr_bf16(bf16_hi(cw[q]) + bf16_hi(gw[q]), rn[2 * q + 1]));
                    st_nt4(a.D + o0, u32x4_t{o[0], o[1], o[2], o[3]});
                }
            }
        } else {
#pragma unroll
            for (int y = 0; y < NP; ++y) {
                const int m = mb + RPP * y;
                const u32x4_t w = *reinterpret_cast<const u32x4_t *>(est(crow + RPP * y) + 8 * cchk);
                const int64_t row = KIND == EX_WGRAD ? (int64_t)e * M + m : (int64_t)lo + m;
                if (m < M && n < a.N) st_nt4(a.D + row * a.N + n, w);
            }
        }
    };
    block(std::integral_constant<int, 0>{});
    if constexpr (FM > 1) block(std::integral_constant<int, 1>{});
    if constexpr (FM > 2) {
        block(std::integral_constant<int, 2>{});
        block(std::integral_constant<int, 3>{});
    }
}

// The slabs' k, the LDS stages and the waves per SIMD that a tile runs with.  Times of 8192 and 16384 rows
// over 8 experts of 14336 x 4096 and 4096 x 4096, of 16411 and 32768 over 64 of 1024 and 1408 x 2048 (us, with
// outputs stored through the caches):
//            256: (64, 2)  (32, 4)      128: (64, 2)  (32, 3)  (32, 4)
//   forward   950 561 123 251   974 577 124 254     1127 640 122 271   1357 725 130 293   1309 720 131 294
//   dgrad    1120 546 110 242  1070 527 110 238     1216 634 130 276   1420 688 125 286   1442 696 133 295
//   wgrad     913 489 143 289   867 449 130 274     1138 609 149 347   1054 550 138 279   1092 573 146 316
//   accum    1130 542 188 378  1096 514 182 364     1356 664 198 438   1205 595 169 335   1286 622 182 378
// Half-length slabs cost barriers and row-major reads of 64-byte rows, which the forward product pays most for;
// more of them in flight hide the latency of operands that K-major products load in shorter pieces.
// SPLIT: few tiles over a long K, a work-group to a CU: its time is the latency of one slab after the other, which
// 2 groups with 4 stages (forward) or 4 groups with 2 (dgrad) shorten:
//   rows x experts, out x in          forward: no split, (2, 4), (4, 2)      dgrad
//   300 x 4,  1024 x 8192 (8192 x 1024)        62  26  34                    62  50  39
//   1 x 1,    4096 x 4096                      32  15  18                    32  24  19
//   64 x 8,   (4096 x 1024)                                                  34  28  23
//   16 x 8,   4096 x 4096 (272 tiles)          35  36  41                    36  52  48
// ACC, 128: the accumulation has its noise to compute and its accumulators to wait for, which a fourth work-group per CU
// hides better than a third stage.  us with 2 stages and 4 waves per SIMD (so); 3 and 3; 3, 3 and two row blocks of
// accumulators fetched ahead instead of one, on one card, the same tensors every time and four sets of them in turn (no
// operand left in the last-level cache):
//   16411 x 64, 1024 x 2048   148 153 155   161 162 161
//   32768 x 64, 1408 x 2048   303 311 311   327 331 330
//   8192 x 32,  1024 x 2048    78  79  83    78  79  82
//   16384 x 128, 768 x 2048   176 182 184   189 193 191
//   4096 x 8,   1536 x 1536    37  37  36    40  37  37
template <int KIND, bool ACC, int T, bool SPLIT>
struct Ring {
    static constexpr bool FINE = KIND != EX_FWD && T >= 128;
    static constexpr int KG = !SPLIT ? 1 : KIND == EX_FWD ? 2 : 4;
    static constexpr int BK = FINE ? 32 : 64, S = KG == 2 ? 4 : FINE ? (T == 256 ? 4 : ACC ? 2 : 3) : 2;
    static constexpr int WPS = KG == 4 ? 4 : FINE && T == 128 ? (ACC ? 4 : 3) : 2;
};

// Estimated time (us) of a call in tiles of T, from times per slab of 64 k of a tile: p with every CU busy, u for a
// tile that has its CU to itself; and o for its start and end.  Fitted to the forward and dgrad times above and to
// (stored and accumulated weight gradients with non-temporal outputs):
//   rows x experts, weights      forward 256 128 64   dgrad 256 128 64   wgrad 256 128 64   accum 256 128 64
//   8192 x 8,    1536 x 384            17  20  27           33  20  23         39  25  23         47  42  25
//   4096 x 128,   768 x 2048          126 108 107          116  96  96         83  71 114        193 147 206
//   512 x 64,    1024 x 2048           49  41  40           48  44  42         54  42  67        131  96 131
//   61 x 8,       512 x 256           9.1 5.8 4.7         13.6 7.9 5.7        6.2 4.0 4.0       13.0 6.6 4.2
//   16411 x 64,  1024 x 2048                                                  101  98 154        165 145 214
//   65536 x 64,  1024 x 2048          307 355 533          305 380 584        282 329 587        343 372 623
// A group is taken to end in the middle of its last tile, and the largest expert to have twice the average rows.
static float experts_cost(int kind, bool accum, int T, bool split, const ExpertArgs &a) {
    const int i = T == 256 ? 2 : T == 128 ? 1 : 0;
    constexpr float ROWS_P[3] = {0.25f, 0.62f, 1.9f}, U[3] = {0.5f, 0.75f, 1.2f}, ROWS_O[3] = {1.5f, 3.0f, 5.0f};
    constexpr float W_P[3] = {0.215f, 0.54f, 1.75f}, W_O[3] = {0.4f, 0.8f, 5.0f}, ACC_O[3] = {0.9f, 2.3f, 13.0f};
    const float tn = (float)((a.N + T - 1) / T);
    if (kind == EX_WGRAD) {
        const float n = (float)((a.M + T - 1) / T) * tn * (float)a.experts / 256.0f;   // tiles per CU
        const float ks = (float)a.rows / (float)a.experts / 64.0f + 0.5f, o = accum ? ACC_O[i] : W_O[i];
        return std::max(n * (ks * W_P[i] + o), 2.0f * ks * (accum && T == 128 ? 1.15f : U[i]) + o);   // its two stages alone: 42 us for 1536 x 384
    }
    const float n = ((float)a.rows / (float)T + 0.5f * (float)std::min(a.experts, a.rows)) * tn / 256.0f, ks = (float)a.K / 64.0f;
    if (split) return ceilf(n) * (ks * (kind == EX_FWD ? 0.22f : 0.33f) + 4.0f);
    return ks * std::max(n * ROWS_P[i], U[i]) + std::max(n, 1.0f) * ROWS_O[i];
}

struct ExpertPlan {
    int tile;
    bool split;
};
static ExpertPlan experts_plan(int kind, bool accum, const ExpertArgs &a) {
    ExpertPlan best{64, false};
    float least = experts_cost(kind, accum, 64, false, a);
    for (const ExpertPlan p : {ExpertPlan{128, false}, ExpertPlan{256, false}, ExpertPlan{64, true}}) {
        if (p.split && kind == EX_WGRAD) continue;
        const float c = experts_cost(kind, accum, p.tile, p.split, a);
        if (c < least) {
            least = c;
            best = p;
        }
    }
    return best;
}

template <int KIND, int MODE, int T, bool SPLIT>
static void experts_launch_tile(const ExpertArgs &a, unsigned grid, hipStream_t s) {
    using R = Ring<KIND, (MODE >= 0), T, SPLIT>;
    hipLaunchKernelGGL((experts_kernel<KIND, MODE, T, R::BK, R::S, R::WPS, R::KG>), dim3(grid), dim3(64 * Shape<T>::NW * R::KG), 0, s, a);
}

template <int KIND, int MODE>
static int experts_launch(ExpertArgs a, const char *name, hipStream_t s) {
    const ExpertPlan plan = experts_plan(KIND, MODE >= 0, a);
    const int T = plan.tile;
    a.tiles_n = (a.N + T - 1) / T;
    a.by_size = a.experts <= 64 && a.rows / a.experts >= X_SORT;
    // wgrad: 8 shares of every expert's tiles; the row products: at most one part tile per group more than
    // the rows fill
    const int64_t tiles = KIND == EX_WGRAD ? ((int64_t)((a.M + T - 1) / T) * a.tiles_n + NXCD - 1) / NXCD * NXCD * a.experts
                                           : ((int64_t)a.rows / T + a.experts + 1) * a.tiles_n;
    constexpr int MOST = 64 * Shape<64>::NW * 4;   // threads of a work-group; a launch has fewer than 2^32
    if (tiles > UINT32_MAX / MOST) { set_error("%s: too many tiles for a launch (%lld)", name, (long long)tiles); return MSR_ERR_ARG; }
    if (T == 256) experts_launch_tile<KIND, MODE, 256, false>(a, (unsigned)tiles, s);
    else if (T == 128) experts_launch_tile<KIND, MODE, 128, false>(a, (unsigned)tiles, s);
    else if (!plan.split) experts_launch_tile<KIND, MODE, 64, false>(a, (unsigned)tiles, s);
    else if constexpr (KIND != EX_WGRAD) experts_launch_tile<KIND, MODE, 64, true>(a, (unsigned)tiles, s);
    return check_launch(name);
}

static int experts_check(const char *name, int64_t rows, int32_t experts, int64_t in_f, int64_t out_f) {
    if (rows < 0 || rows >= (1 << 30) || experts < 1 || experts > MSR_EXPERTS_MAX || in_f < 8 || out_f < 8 || in_f % 8 ||
        out_f % 8 || in_f > (1 << 20) || out_f > (1 << 20) || in_f * out_f >= (1 << 30)) {
        set_error("%s: need fewer than 2^30 rows, 1 to %d experts, in and out features multiples of 8 up to 2^20 and their "
                  "product below 2^30 (got %lld rows, %d experts, %lld x %lld)", name, MSR_EXPERTS_MAX, (long long)rows,
                  (int)experts, (long long)out_f, (long long)in_f);
        return MSR_ERR_ARG;
    }
    return MSR_OK;
}

constexpr int64_t X_LD = 1 << 21;   // row strides: a tile's rows span less than 2^31 bytes

// One operand's memory, for the overlap checks.
struct Span {
    const void *p;
    size_t n;
};
static size_t row_bytes(int64_t rows, int64_t ld, int64_t width) {
    return rows > 0 ? 2 * ((size_t)(rows - 1) * (size_t)ld + (size_t)width) : 0;
}
static int experts_spans(const char *name, Span out, const Span *in, int n) {
    for (int i = 0; i < n; ++i) {
        const uintptr_t u = (uintptr_t)out.p, v = (uintptr_t)in[i].p;
        if (out.n && in[i].n && u < v + in[i].n && v < u + out.n) {
            set_error("%s: the output overlaps operand %d", name, i);
            return MSR_ERR_OVERLAP;
        }
    }
    return MSR_OK;
}

// forward and dgrad: `width` features of the input rows `p`, `outw` of the result
static int experts_rows(const char *name, int kind, const uint16_t *p, int64_t ldp, const uint16_t *w, uint16_t *out,
                        const int32_t *offsets, int64_t rows, int32_t experts, int64_t width, int64_t outw, hipStream_t s) {
    if (!offsets || (rows > 0 && (!p || !w || !out)) || ldp < width || ldp > X_LD) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
    if (!aligned(p, 16) || !aligned(w, 16) || !aligned(out, 16) || !aligned(offsets, 4) || ldp % 8) {
        set_error("%s: operands must be 16-byte aligned with row strides a multiple of 8", name);
        return MSR_ERR_ALIGN;
    }
    const Span in[3] = {{p, row_bytes(rows, ldp, width)}, {w, 2 * (size_t)experts * (size_t)(width * outw)},
                        {offsets, 4 * ((size_t)experts + 1)}};
    const int rc = experts_spans(name, {out, row_bytes(rows, outw, outw)}, in, 3);
    if (rc || rows == 0) return rc;
    ExpertArgs a{};
    a.P = p; a.ldp = ldp; a.Q = w; a.D = out; a.offsets = offsets;
    a.rows = (int)rows; a.experts = experts; a.N = (int)outw; a.K = (int)width;
    a.ldq = kind == EX_FWD ? width : outw;
    return kind == EX_FWD ? experts_launch<EX_FWD, -1>(a, name, s) : experts_launch<EX_DGRAD, -1>(a, name, s);
}

static int experts_weights(const char *name, uint16_t *d, const uint16_t *x, int64_t ldx, const uint16_t *dy, int64_t lddy,
                           const int32_t *offsets, int64_t rows, int32_t experts, int64_t in_f, int64_t out_f, int mode,
                           uint32_t seed, int32_t zero_init, const uint16_t *inject, hipStream_t s) {
    if (!d || !offsets || (rows > 0 && (!x || !dy)) || ldx < in_f || lddy < out_f || ldx > X_LD || lddy > X_LD) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
    if (!aligned(d, 16) || !aligned(x, 16) || !aligned(dy, 16) || !aligned(offsets, 4) || ldx % 8 || lddy % 8) {
        set_error("%s: operands must be 16-byte aligned with row strides a multiple of 8", name);
        return MSR_ERR_ALIGN;
    }
    const Span in[3] = {{x, row_bytes(rows, ldx, in_f)}, {dy, row_bytes(rows, lddy, out_f)}, {offsets, 4 * ((size_t)experts + 1)}};
    const int rc = experts_spans(name, {d, 2 * (size_t)experts * (size_t)(in_f * out_f)}, in, 3);
    if (rc) return rc;
    ExpertArgs a{};
    a.P = dy; a.ldp = lddy; a.Q = x; a.ldq = ldx; a.D = d; a.offsets = offsets;
    a.rows = (int)rows; a.experts = experts; a.M = (int)out_f; a.N = (int)in_f; a.zero_init = zero_init != 0;
    a.ns.key = seed_key(seed, 0);
    a.ns.inject = inject;
    if (mode < 0) return experts_launch<EX_WGRAD, -1>(a, name, s);
    MSR_DISPATCH_NOISE(mode, MODE, return (experts_launch<EX_WGRAD, MODE>(a, name, s)));
    return MSR_OK;
}

}  // namespace msr

using namespace msr;

extern "C" {

int msr_experts_tile(int32_t product, int64_t rows, int32_t experts, int64_t in_features, int64_t out_features, int32_t *tile,
                     int32_t *split) {
    const int rc = experts_check("msr_experts_tile", rows, experts, in_features, out_features);
    if (rc) return rc;
    if (product < 0 || product > 3 || !tile || !split) { set_error("msr_experts_tile: bad arguments"); return MSR_ERR_ARG; }
    ExpertArgs a{};
    a.rows = (int)rows; a.experts = experts;
    a.M = (int)out_features;
    a.N = (int)(product == EX_FWD ? out_features : in_features);
    a.K = (int)(product == EX_FWD ? in_features : out_features);
    const ExpertPlan p = experts_plan(std::min(product, (int32_t)EX_WGRAD), product == 3, a);
    *tile = p.tile;
    *split = p.split;
    return MSR_OK;
}

int msr_experts_forward(const uint16_t *x, int64_t ldx, const uint16_t *w, uint16_t *y, const int32_t *offsets,
                        int64_t rows, int32_t experts, int64_t in_features, int64_t out_features, msr_stream_t stream) {
    const int rc = experts_check("msr_experts_forward", rows, experts, in_features, out_features);
    return rc ? rc : experts_rows("msr_experts_forward", EX_FWD, x, ldx, w, y, offsets, rows, experts, in_features, out_features,
                                  (hipStream_t)stream);
}

int msr_experts_dgrad(const uint16_t *dy, int64_t lddy, const uint16_t *w, uint16_t *dx, const int32_t *offsets,
                      int64_t rows, int32_t experts, int64_t in_features, int64_t out_features, msr_stream_t stream) {
    const int rc = experts_check("msr_experts_dgrad", rows, experts, in_features, out_features);
    return rc ? rc : experts_rows("msr_experts_dgrad", EX_DGRAD, dy, lddy, w, dx, offsets, rows, experts, out_features, in_features,
                                  (hipStream_t)stream);
}

int msr_experts_wgrad(uint16_t *dw, const uint16_t *x, int64_t ldx, const uint16_t *dy, int64_t lddy,
                      const int32_t *offsets, int64_t rows, int32_t experts, int64_t in_features, int64_t out_features,
                      msr_stream_t stream) {
    const int rc = experts_check("msr_experts_wgrad", rows, experts, in_features, out_features);
    return rc ? rc : experts_weights("msr_experts_wgrad", dw, x, ldx, dy, lddy, offsets, rows, experts, in_features, out_features,
                                     -1, 0, 1, nullptr, (hipStream_t)stream);
}

int msr_experts_wgrad_sr_accum(uint16_t *acc, const uint16_t *x, int64_t ldx, const uint16_t *dy, int64_t lddy,
                               const int32_t *offsets, int64_t rows, int32_t experts, int64_t in_features,
                               int64_t out_features, uint32_t seed, int32_t zero_init, int32_t noise_mode,
                               const uint16_t *inject, msr_stream_t stream) {
    if (noise_mode < 0 || noise_mode > 2 || (noise_mode == NOISE_INJECT && !inject)) {
        set_error("msr_experts_wgrad_sr_accum: bad noise_mode %d", (int)noise_mode);
        return MSR_ERR_ARG;
    }
    const int rc = experts_check("msr_experts_wgrad_sr_accum", rows, experts, in_features, out_features);
    return rc ? rc : experts_weights("msr_experts_wgrad_sr_accum", acc, x, ldx, dy, lddy, offsets, rows, experts, in_features,
                                     out_features, noise_mode, seed, zero_init, inject, (hipStream_t)stream);
}

}  // extern "C"
