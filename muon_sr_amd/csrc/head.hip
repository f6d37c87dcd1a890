// A language model's head with its loss: for rows x [rows][d], words W [vocab][d] and the word t[n] of each row
//     S[n][v] = <x[n], W[v]>,   l[n] = log sum_v exp S[n][v],   loss[n] = l[n] - S[n][t[n]]
//     G[n][v] = g[n] (exp(S[n][v] - l[n]) - [v = t[n]]),   dx = G W,   dW = G^T x
// with g[n] the gradient of loss[n].  S is never in memory: the forward pass keeps the maximum and the sum of each row of each
// tile, the backward pass forms S again, piece by piece of the vocabulary, and stores the piece's G as the bf16 operand of
// the two products that follow.  8 rows vocab d flop with gradients where 6 are the least; the logits kept in fp32 would be 4.2 GB
// for 8192 rows of 128256 words.
//
// What is stored is G / c, rounded to bf16: c is the significand of the first row's g (every row's, but for the reduction "none"), by which
// the products' sums are multiplied in fp32.  The target's element of an unlikely word is -g, a factor of its whole row: rounded with g, every
// such row would be off by the same share, up to 2^-8.  In dx, which has one such element to a row, what its rounding leaves is added
// exactly (rest W[t], by dx_kernel).  In dW it stays.  Gradients against 64 bits, dx and dW, where the rounding of the results is 0.0017: 8192 rows,
// 128256 words of 4096 0.0017 and 0.0019 (0.0019 and 0.0019 without the rest); 8192 rows, 32000 words of 2048 of the reduction "none",
// where c takes out the first row's significand alone, 0.0017 and 0.0022 (0.0022 both).  G as the sum of two bf16 numbers gives 0.0017
// throughout and takes 1.7 times as long (backward passes of these 21.2 and 35.8, 2.78 and 4.68 ms), so only few rows have it (LO_ROWS).
//
// Rows that are ignored take part in nothing: list_kernel numbers the others, pack_kernel lays them out one after the
// other (kept for the backward pass in x's place), and every kernel after it works on *count rows.  What an ignored row holds,
// NaN too, reaches no sum, and a padded batch costs what its tokens cost.
#include "rows.hpp"
#include "slabs.hpp"
#include "../../include/muon_sr_amd.h"

namespace msr {

constexpr int HEAD_NONE = 0, HEAD_SUM = 1, HEAD_MEAN = 2;
constexpr int HEAD_BAD = -1;                 // a row whose target is no word
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct HeadArgs {
    const uint16_t *x;           // [rows][d], packed: the rows that are not ignored
    const uint16_t *w;           // [vocab][d]
    const int32_t *kept;         // count, then rows numbers of rows, then their words
    float2 *sums;                // [rows], in the packed order: M and s of the row
    float2 *part;                // [tiles of words][rows]: of a tile
    float *picked;               // [rows]: S[n][t[n]]
    const float *dloss;          // [rows] in the given order, or one
    uint16_t *g;                 // [g_rows][ldg]: a piece of G / c, of few rows two numbers (low_of)
    float *rest;                 // [rows]: what rounding leaves of the target's element of G / c
    float *slots;                // fp32 sums [splits][g_rows][d] of dx, [splits][words of the piece][d] of dW
    uint16_t *out;               // dW or the accumulator
    int64_t ldg;
    int32_t rows, vocab, d, reduction;
    int32_t few, g_rows;         // rows that count, at most, for G / c to be the sum of two bf16 numbers; room for either
    int32_t v0, vn;              // the piece: words v0 to v0 + vn - 1
    int32_t tiles_n, splits, first, zero_init;   // first: the slots hold nothing yet
    Noise ns;
};

// (through the constant address space: a scalar load, as every work-group waits for it first)
typedef const __attribute__((address_space(4))) int32_t *const_i32_t;
__device__ __forceinline__ int kept_rows(const HeadArgs &a) { return min(max(*(const_i32_t)(uintptr_t)a.kept, 0), a.rows); }
__device__ __forceinline__ int word_of(const HeadArgs &a, int r) { return a.kept[1 + a.rows + r]; }
// The row of G where the second numbers of its rows begin; 0 where it has none
__device__ __forceinline__ int low_of(const HeadArgs &a, int count) { return count <= a.few ? count : 0; }
// g of packed row r
__device__ __forceinline__ float dloss_of(const HeadArgs &a, int r, int count) {
    const float g = a.dloss[a.reduction == HEAD_NONE ? a.kept[1 + r] : 0];
    return a.reduction == HEAD_MEAN ? g / (float)count : g;
}
// c, in [1, 2); 1 where the first row's g has no significand
__device__ __forceinline__ float unit_of(const HeadArgs &a, int count) {
    if (count == 0) return 1.0f;
    const float m = 2.0f * fabsf(__builtin_amdgcn_frexp_mantf(dloss_of(a, 0, count)));
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(m >= 1.0f && m < 2.0f ? m : 1.0f)));
}
// g / c of packed row r; NaN where its target is no word
__device__ __forceinline__ float slope_of(const HeadArgs &a, int r, int count, float unit) {
    return word_of(a, r) == HEAD_BAD ? __builtin_nanf("") : dloss_of(a, r, count) / unit;
}

// Tile v of tiles_m x tiles_n in each of `splits` shares of K.  Consecutive work-groups go to the 8 XCDs in turn: each XCD takes a
// contiguous eighth of the shares' tiles, WALK rows of tiles at a time, column by column, so that its L2 holds what they
// share (8192 rows, 128256 words of 4096, walks of 4, 8, 16, 32 rows: logits 6.70, 6.73, 7.08, 7.95 ms, dx 6.88 with 2 and 4, 6.87, 6.93,
// 7.20).
constexpr int WALK = 4;
__device__ __forceinline__ bool find_tile(int v, int tiles_m, int tiles_n, int splits, int &mt, int &nt, int &split) {
    const int tiles = tiles_m * tiles_n, total = tiles * splits, per = total / NXCD;
    if (v >= total) return false;
    if (v < per * NXCD) v = (v % NXCD) * per + v / NXCD;
    split = v / tiles;
    v -= split * tiles;
    const int pg = WALK * tiles_n, g = v / pg, rows = min(WALK, tiles_m - WALK * g), r = v - g * pg;
    mt = WALK * g + r % rows;
    nt = r / rows;
    return true;
}

// A set of logits is held as M, a number near the largest times log2(e), and s = sum exp2(x log2(e) - M): one multiply-add per
// exponential, and M is exact, whatever it was rounded from.  l = M ln 2 + log s is never formed: an l of 40 is rounded by 2^-19, and with it
// the gradient of a row whose word is nearly sure, and its loss.
__device__ __forceinline__ float exp_from(float x, float M) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, LOG2E, -M)); }

// (M, s) of the union of two sets; an empty set is (-inf, 0)
__device__ __forceinline__ float2 joined(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x), at = m == -INFINITY ? 0.0f : m;
    return make_float2(m, a.y * __builtin_amdgcn_exp2f(a.x - at) + b.y * __builtin_amdgcn_exp2f(b.x - at));
}

// ---------------------------------------------------------------------------
// rows that count
// ---------------------------------------------------------------------------

constexpr int LIST_THREADS = 1024, LIST_EACH = 8;

struct ListArgs {
    const void *target;
    int64_t ignore;
    int32_t *kept, *pos;         // pos [rows]: a row's packed number, -1 for an ignored one
    float *loss;                 // [rows], or null: 0 for ignored rows
    int32_t rows, vocab, i64;
    const uint16_t *x;           // where the same launch packs the rows
    int64_t ldx;
    uint16_t *packed;
    int32_t d;
};

// packed[r] = x[row of r] by one wave
__device__ __forceinline__ void pack_row(const uint16_t *from, uint16_t *to, int d) {
    for (int c = 8 * (int)(threadIdx.x & 63); c < d; c += 512) *reinterpret_cast<Bytes16 *>(to + c) = *reinterpret_cast<const Bytes16 *>(from + c);
}

// One work-group numbers the rows that are not ignored, in order: LIST_EACH rows per thread at a time, LIST_THREADS apart, so that a
// wave's accesses are 64 elements on end (4096 rows 9.4 us with eight neighbouring rows per thread, 4.7 so).
__global__ __launch_bounds__(LIST_THREADS) void list_kernel(ListArgs a) {
    constexpr int WAVES = LIST_THREADS / 64;
    static_assert(WAVES * LIST_EACH == 128, "two counts per lane of a wave");
    __shared__ int at[WAVES * LIST_EACH], total;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int base = 0;
    for (int64_t n0 = 0; n0 < a.rows; n0 += LIST_THREADS * LIST_EACH) {
        int64_t t[LIST_EACH];
        uint64_t kept[LIST_EACH];
#pragma unroll
        for (int i = 0; i < LIST_EACH; ++i) {
            const int64_t n = n0 + i * LIST_THREADS + tid;
            t[i] = a.ignore;
            if (n < a.rows) t[i] = a.i64 ? static_cast<const int64_t *>(a.target)[n] : static_cast<const int32_t *>(a.target)[n];
        }
#pragma unroll
        for (int i = 0; i < LIST_EACH; ++i) {
            kept[i] = __ballot(t[i] != a.ignore);
            if (lane == 0) at[i * WAVES + wave] = __popcll(kept[i]);
        }
        __syncthreads();
        if (wave == 0) {
            const int c0 = at[2 * lane], c1 = at[2 * lane + 1], to = wave_scan(c0 + c1);
            at[2 * lane] = to - c0 - c1;
            at[2 * lane + 1] = to - c1;
            if (lane == 63) total = to;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LIST_EACH; ++i) {
            const int64_t n = n0 + i * LIST_THREADS + tid;
            if (n >= a.rows) continue;
            const bool on = t[i] != a.ignore;
            const int place = base + at[i * WAVES + wave] + __popcll(kept[i] & ((1ull << lane) - 1));
            a.pos[n] = on ? place : -1;
            if (on) {
                a.kept[1 + place] = (int32_t)n;
                a.kept[1 + a.rows + place] = t[i] >= 0 && t[i] < a.vocab ? (int32_t)t[i] : HEAD_BAD;
            } else if (a.loss) {
                a.loss[n] = 0.0f;
            }
        }
        base += total;
        __syncthreads();
    }
    if (tid == 0) a.kept[0] = base;
    if (!a.packed) return;
    __syncthreads();                                  // (kept was written by this work-group)
    for (int r = wave; r < base; r += WAVES) pack_row(a.x + (int64_t)a.kept[1 + r] * a.ldx, a.packed + (int64_t)r * a.d, a.d);
}

__global__ __launch_bounds__(256) void pack_kernel(const uint16_t *x, int64_t ldx, uint16_t *packed, const int32_t *kept, int rows, int d) {
    const int count = min(max(kept[0], 0), rows);
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < count; r += (int64_t)gridDim.x * 4)
        pack_row(x + (int64_t)kept[1 + r] * ldx, packed + r * d, d);
}

// ---------------------------------------------------------------------------
// logits: their row maxima and sums, or a piece of G
// ---------------------------------------------------------------------------

// A work-group takes tiles blockIdx.x, blockIdx.x + gridDim.x, ..: the first slab of its next tile is on its way while the
// epilogue works in LDS of its own.  T = 256 has one work-group to a CU, whose epilogue nothing else covers (us, forward and a piece of G,
// with a tile per work-group and so: 4096 rows, 16384 words of 384 60.3 68.2, 58.6 64.9; 7370 rows, 32000 words of 2048 854 940, 844 925).
// What is left of the epilogue is its own arithmetic: 128 exponentials per lane and tile, some 3 of 15 us at width 384.
template <bool GRAD, int T, int BK>
__global__ __launch_bounds__(64 * Shape<T>::NW, 2) void logits_kernel(HeadArgs a) {
    using SH = Shape<T>;
    constexpr int NW = SH::NW, FM = SH::FM, FN = SH::FN, TN = SH::TN;
    using PR = Product<T, BK, 2, false, false>;
    constexpr int PB = PR::SP::BYTES;
    constexpr int WROW = TN * 2;                                  // bytes of a staged row of G
    __shared__ __attribute__((aligned(1024))) char p_0[PB], p_1[PB], q_0[PB], q_1[PB];
    __shared__ __attribute__((aligned(16))) char own[GRAD ? NW * 32 * WROW : SH::WN * T * 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / SH::WN, wn = wave % SH::WN;
    const int count = kept_rows(a), tiles_m = (count + T - 1) / T, slabs = (a.d + BK - 1) / BK, low = low_of(a, count);
    const float unit = GRAD ? unit_of(a, count) : 1.0f;
    PR pr;
    auto lds_p = [&](auto ST) __attribute__((always_inline)) -> char * { return decltype(ST)::value == 0 ? p_0 : p_1; };
    auto lds_q = [&](auto ST) __attribute__((always_inline)) -> char * { return decltype(ST)::value == 0 ? q_0 : q_1; };
    auto side_p = [&](int mt) __attribute__((always_inline)) {
        return typename PR::Side{a.x + (int64_t)mt * T * a.d, a.d, min(T, count - mt * T), 0, a.d};
    };
    auto side_q = [&](int nt) __attribute__((always_inline)) {    // nt: from v0 on
        return typename PR::Side{a.w + (int64_t)(a.v0 + nt * T) * a.d, a.d, min(T, a.vn - nt * T), 0, a.d};
    };
    int mt, nt, split;
    int v = blockIdx.x;
    if (!find_tile(v, tiles_m, a.tiles_n, 1, mt, nt, split)) return;
    pr.init(wave, lane, a.d, a.d);
    pr.ahead(lds_p, lds_q, side_p(mt), side_q(nt), 0, slabs);
    for (;;) {
        const int m0 = mt * T, n0 = nt * T;
        // what the epilogue needs of the lane's rows, loaded ahead of the products
        int word[FM];
        float M[FM], slope[FM], share[FM];                    // share: slope / s
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int row = m0 + wm * SH::TM + 32 * i + (lane & 31);
            word[i] = HEAD_BAD;
            M[i] = slope[i] = share[i] = 0.0f;
            if (row < count) {
                word[i] = word_of(a, row);
                if constexpr (GRAD) {
                    const float2 sums = a.sums[row];
                    M[i] = sums.x;
                    slope[i] = slope_of(a, row, count, unit);
                    share[i] = slope[i] / sums.y;
                }
            }
        }
        pr.template run<true>(lds_p, lds_q, side_p(mt), side_q(nt), 0, slabs);
        wait_vm<0>();                                             // no load writes the stages any more
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        v += gridDim.x;
        const bool more = find_tile(v, tiles_m, a.tiles_n, 1, mt, nt, split);
        if (more) pr.ahead(lds_p, lds_q, side_p(mt), side_q(nt), 0, slabs);

        // lane l: row l % 32 of each 32-row block i, columns 32 j + 8 r + 4 (l / 32) + q
        int etid = tid;
        asm volatile("" : "+v"(etid));                            // (addresses formed here, not kept through the loop)
        const int elane = etid & 63, r32 = elane & 31, khalf = elane >> 5;
        const int nw = n0 + wn * TN + 4 * khalf, m1 = m0 + wm * SH::TM + r32;
        if (n0 + T > a.vn) {                                      // words that are not there
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        if (nw + 32 * j + 8 * (x >> 2) + (x & 3) >= a.vn) pr.acc[i][j][x] = -INFINITY;
        }
        if constexpr (!GRAD) {
            float2 *const stat = reinterpret_cast<float2 *>(own);   // [WN][T]
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                float m = -INFINITY;
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int x = 0; x < 16; ++x) m = fmaxf(m, pr.acc[i][j][x]);
                m = fmaxf(m, __shfl_xor(m, 32));
                m = m == -INFINITY ? m : m * LOG2E;
                const float at = m == -INFINITY ? 0.0f : m;
                float s = 0.0f;
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int x = 0; x < 16; ++x) s += exp_from(pr.acc[i][j][x], at);
                s += __shfl_xor(s, 32);
                if (khalf == 0) stat[wn * T + wm * SH::TM + 32 * i + r32] = make_float2(m, s);
                const int row = m1 + 32 * i;
                const int rel = word[i] - a.v0 - nw;              // this lane's columns: those with bit 2 of rel clear
                if (__any(rel >= 0 && rel < TN && !(rel & 4))) {
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            if (rel == 32 * j + 8 * (x >> 2) + (x & 3)) a.picked[row] = pr.acc[i][j][x];
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // (the next tile's loads stay on their way)
            for (int m = tid; m < T && m0 + m < count; m += 64 * NW) {
                float2 all = stat[m];
#pragma unroll
                for (int k = 1; k < SH::WN; ++k) all = joined(all, stat[k * T + m]);
                a.part[(int64_t)(n0 / T) * a.rows + m0 + m] = all;
            }
        } else {
            // Each wave stages its sub-tile, one 32-row block at a time (LDS accesses of one wave execute in order): 16-byte
            // chunk c of row r at c ^ (r & (chunks - 1)), so that the rows of a write fall in different banks
            constexpr int WC = TN / 8, RPP = 64 / WC, NP = 32 / RPP;   // chunks per row, rows per access, accesses per block
            char *const wst = own + wave * (32 * WROW);
            const int crow = elane / WC, cchk = elane % WC, nc = n0 + wn * TN + 8 * cchk;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const float g = slope[i];
                const int rel = word[i] - a.v0 - nw;
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int x = 0; x < 16; ++x) pr.acc[i][j][x] = share[i] * exp_from(pr.acc[i][j][x], M[i]);
                const bool mine = rel >= 0 && rel < TN && !(rel & 4);
                if (__any(mine)) {
                    float rest = 0.0f;
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            if (rel == 32 * j + 8 * (x >> 2) + (x & 3)) rest = pr.acc[i][j][x] -= g;
                    rest -= bf16_to_f32((uint16_t)rne_bf16(rest));
                    if (low) rest -= bf16_to_f32((uint16_t)rne_bf16(rest));
                    if (mine) a.rest[m1 + 32 * i] = rest;
                }
                auto put = [&](int first) __attribute__((always_inline)) {
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            *reinterpret_cast<uint2 *>(wst + r32 * WROW + (((4 * j + r) ^ (r32 & (WC - 1))) * 16 + khalf * 8)) =
                                make_uint2(rne_bf16x2(pr.acc[i][j][4 * r], pr.acc[i][j][4 * r + 1]),
                                           rne_bf16x2(pr.acc[i][j][4 * r + 2], pr.acc[i][j][4 * r + 3]));
#pragma unroll
                    for (int y = 0; y < NP; ++y) {
                        const int rr = crow + RPP * y, m = m0 + wm * SH::TM + 32 * i + rr;
                        const u32x4_t c = *reinterpret_cast<const u32x4_t *>(wst + rr * WROW + ((cchk ^ (rr & (WC - 1))) * 16));
                        if (m < count && nc < a.vn) *reinterpret_cast<u32x4_t *>(a.g + (int64_t)(first + m) * a.ldg + nc) = c;
                    }
                };
                put(0);
                if (!low) continue;
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int x = 0; x < 16; ++x) pr.acc[i][j][x] -= bf16_to_f32((uint16_t)rne_bf16(pr.acc[i][j][x]));
                put(low);
            }
        }
        if (!more) return;
        pr.clear();
    }
}

// The tiles' sets are joined with s in 64 bits: beside a tile that holds a row's nearly sure word, s near 1, each of the others may be
// less than half an ulp, and hundreds of them more than what is left of the row's loss.
struct Joined {
    float m;
    double s;
};
__device__ __forceinline__ Joined joined(Joined a, float m2, double s2) {
    const float m = fmaxf(a.m, m2), at = m == -INFINITY ? 0.0f : m;
    return {m, a.s * (double)__builtin_amdgcn_exp2f(a.m - at) + s2 * (double)__builtin_amdgcn_exp2f(m2 - at)};
}
// The sums and losses of 16 rows from their tiles' parts, 16 threads each
__device__ __forceinline__ void join_rows(const HeadArgs &a, float *loss, int n0, int count, Joined (&part)[16][17]) {
    const int r = threadIdx.x & 15, g = threadIdx.x >> 4, n = n0 + r;
    Joined all{-INFINITY, 0.0};
    if (n < count)
        for (int t = g; t < a.tiles_n; t += 16) {
            const float2 tile = a.part[(int64_t)t * a.rows + n];
            all = joined(all, tile.x, tile.y);
        }
    part[g][r] = all;
    __syncthreads();
    if (g == 0 && n < count) {
        for (int k = 1; k < 16; ++k) all = joined(all, part[k][r].m, part[k][r].s);
        const float2 v = make_float2(all.m, (float)all.s);
        a.sums[n] = v;
        const float l = logf(v.y) + LN2 * __builtin_fmaf(a.picked[n], -LOG2E, v.x);
        loss[a.reduction == HEAD_NONE ? a.kept[1 + n] : n] = word_of(a, n) == HEAD_BAD ? __builtin_nanf("") : l;
    }
    __syncthreads();
}
// The sum or the mean (0 of no rows) of the rows' losses, in 64 bits, by one work-group
__device__ __forceinline__ void total_loss(const float *loss, int count, bool mean, float *out) {
    __shared__ double sums[16];
    double s = 0.0;
    for (int n = threadIdx.x; n < count; n += blockDim.x) s += loss[n];
    for (int w = 32; w; w >>= 1) s += __shfl_xor(s, w);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < (int)blockDim.x / 64; ++w) s += sums[w];
    out[0] = (float)(mean ? s / max(count, 1) : s);
}
// total: the one work-group of a small call adds the losses up too
__global__ __launch_bounds__(256) void join_kernel(HeadArgs a, float *loss, float *total) {
    __shared__ Joined part[16][17];
    const int count = kept_rows(a);
    for (int n0 = (int)blockIdx.x * 16; n0 < count; n0 += (int)gridDim.x * 16) join_rows(a, loss, n0, count, part);
    if (total) total_loss(loss, count, a.reduction == HEAD_MEAN, total);
}
__global__ __launch_bounds__(1024) void total_kernel(const float *loss, const int32_t *kept, int rows, int mean, float *out) {
    total_loss(loss, min(max(kept[0], 0), rows), mean, out);
}

// ---------------------------------------------------------------------------
// the products of a piece of G
// ---------------------------------------------------------------------------

enum : int { HD_DX = 0, HD_DW = 1 };
enum : int { OUT_SLOTS = -2, OUT_STORE = -1 };   // or a noise mode: accumulated

// acc <- SR(acc + bf16(w)) of 8 elements at o0 (a multiple of 8)
template <int MODE>
__device__ __forceinline__ void accumulate8(const HeadArgs &a, int64_t o0, const uint32_t gw[4]) {
    uint32_t cw[4] = {0u, 0u, 0u, 0u}, rn[8], o[4];
    if (!a.zero_init) {
        const u32x4_t c = ld_nt4(a.out + o0);
        cw[0] = c.x; cw[1] = c.y; cw[2] = c.z; cw[3] = c.w;
    }
    noise8<MODE>(a.ns, o0, 8, rn);
#pragma unroll
    for (int q = 0; q < 4; ++q)
        o[q] = pack2(sr_bf16(bf16_lo(cw[q]) + bf16_lo(gw[q]), rn[2 * q]), sr_bf16(bf16_hi(cw[q]) + bf16_hi(gw[q]), rn[2 * q + 1]));
    st_nt4(a.out + o0, u32x4_t{o[0], o[1], o[2], o[3]});
}

// HD_DX: rows of G x words of W, over the piece's words; HD_DW: words of G x features of x, over the rows.
// OUT: fp32 sums added to a split's slot, dW stored, or accumulated with a noise mode.
template <int KIND, int OUT, int T, int BK, int S_, int WPS>
__global__ __launch_bounds__(64 * Shape<T>::NW, WPS) void piece_kernel(HeadArgs a) {
    using SH = Shape<T>;
    constexpr int NW = SH::NW, FM = SH::FM, FN = SH::FN, TN = SH::TN;
    using PR = Product<T, BK, S_, KIND == HD_DW, true>;
    constexpr int PB = PR::SP::BYTES;
    __shared__ __attribute__((aligned(1024))) char p_0[PB], p_1[PB], q_0[PB], q_1[PB];
    __shared__ __attribute__((aligned(1024))) char p_2[S_ > 2 ? PB : 16], q_2[S_ > 2 ? PB : 16];
    __shared__ __attribute__((aligned(1024))) char p_3[S_ > 3 ? PB : 16], q_3[S_ > 3 ? PB : 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / SH::WN, wn = wave % SH::WN;
    const int count = kept_rows(a);
    const float unit = OUT == OUT_SLOTS ? 1.0f : unit_of(a, count);
    const int low = low_of(a, count), M = KIND == HD_DX ? low + count : a.vn, K = KIND == HD_DX ? a.vn : count;
    int mt, nt, split;
    if (!find_tile(blockIdx.x, (M + T - 1) / T, a.tiles_n, a.splits, mt, nt, split)) return;
    const int m0 = mt * T, n0 = nt * T;
    // this split's share of K: `slabs` of them from kb on.  The words of a piece are rounded up to 8 in G, whose columns
    // there are 0, not in W.
    const int slabs = ((K + BK - 1) / BK + a.splits - 1) / a.splits, kb = split * slabs * BK, vn8 = (a.vn + 7) & ~7;
    const int kend = min(K, kb + slabs * BK);
    PR pr;
    pr.init(wave, lane, a.ldg, a.d);
    auto lds_p = [&](auto ST) __attribute__((always_inline)) -> char * {
        constexpr int st = decltype(ST)::value;
        return st == 0 ? p_0 : st == 1 ? p_1 : st == 2 ? p_2 : p_3;
    };
    auto lds_q = [&](auto ST) __attribute__((always_inline)) -> char * {
        constexpr int st = decltype(ST)::value;
        return st == 0 ? q_0 : st == 1 ? q_1 : st == 2 ? q_2 : q_3;
    };
    if (kb < K) {
        if constexpr (KIND == HD_DX)
            pr.run(lds_p, lds_q, {a.g + (int64_t)m0 * a.ldg, a.ldg, min(T, M - m0), 0, min(vn8, kb + slabs * BK)},
                   {a.w + (int64_t)a.v0 * a.d + n0, a.d, 0, a.d - n0, kend}, kb, slabs);
        else
            for (int first = 0;; first = low) {
                pr.run(lds_p, lds_q, {a.g + (int64_t)first * a.ldg + m0, a.ldg, 0, vn8 - m0, kend}, {a.x + n0, a.d, 0, a.d - n0, kend}, kb, slabs);
                if (first == low) break;
                wait_vm<0>();
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
    }
    wait_vm<0>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    int etid = tid;
    asm volatile("" : "+v"(etid));
    const int elane = etid & 63, r32 = elane & 31, khalf = elane >> 5;
    if constexpr (OUT == OUT_SLOTS) {
        const int64_t rows = KIND == HD_DX ? a.g_rows : a.vn;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int m = m0 + wm * SH::TM + 32 * i + r32;
            float *const to = a.slots + ((int64_t)split * rows + m) * a.d;
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int n = n0 + wn * TN + 32 * j + 8 * r + 4 * khalf;
                    if (m >= M || n >= a.d) continue;
                    f32x4_t v = {pr.acc[i][j][4 * r], pr.acc[i][j][4 * r + 1], pr.acc[i][j][4 * r + 2], pr.acc[i][j][4 * r + 3]};
                    f32x4_t *const at = reinterpret_cast<f32x4_t *>(to + n);
                    if (!a.first) {
                        const f32x4_t o = *at;
                        v = f32x4_t{o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w};
                    }
                    *at = v;
                }
        }
    } else {
        constexpr int EP = TN + 8, WC = TN / 8, RPP = 64 / WC, NP = 32 / RPP, PER = PB / (32 * EP * 2);
        static_assert(PER > 0 && NW <= 4 * PER, "the staging fits the first two stages");
        const int sv = wave / PER;
        char *const wst = (sv == 0 ? p_0 : sv == 1 ? q_0 : sv == 2 ? p_1 : q_1) + (wave % PER) * (32 * EP * 2);
        const int crow = elane / WC, cchk = elane % WC, n = n0 + wn * TN + 8 * cchk;
        auto block = [&](auto I) __attribute__((always_inline)) {      // (acc indexed by constants)
            constexpr int i = decltype(I)::value;
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    *reinterpret_cast<uint2 *>(wst + r32 * (EP * 2) + (j * 32 + 8 * r + 4 * khalf) * 2) =
                        make_uint2(rne_bf16x2(unit * pr.acc[i][j][4 * r], unit * pr.acc[i][j][4 * r + 1]),
                                   rne_bf16x2(unit * pr.acc[i][j][4 * r + 2], unit * pr.acc[i][j][4 * r + 3]));
#pragma unroll
            for (int y = 0; y < NP; ++y) {
                const int m = m0 + wm * SH::TM + 32 * i + crow + RPP * y;
                const u32x4_t v = *reinterpret_cast<const u32x4_t *>(wst + (crow + RPP * y) * (EP * 2) + 16 * cchk);
                if (m >= M || n >= a.d) continue;
                const int64_t o0 = (int64_t)(a.v0 + m) * a.d + n;
                if constexpr (OUT == OUT_STORE) {
                    st_nt4(a.out + o0, v);
                } else {
                    const uint32_t gw[4] = {v.x, v.y, v.z, v.w};
                    accumulate8<OUT>(a, o0, gw);
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
}

// The sum of a row's slots and of what the target's element of G / c left, times W[target], times c, rounded: dx of every row (0 for an
// ignored one), 8 elements per thread
__global__ __launch_bounds__(256) void dx_kernel(HeadArgs a, uint16_t *dx) {
    const int rows = a.rows, d = a.d;
    const int32_t *const pos = a.kept + 1 + 2 * (int64_t)rows;
    const int64_t chunks = (int64_t)rows * (d / 8);
    const int count = kept_rows(a), low = low_of(a, count);
    const float unit = unit_of(a, count);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
        const int64_t n = i / (d / 8);
        const int c = (int)(i % (d / 8)) * 8, p = pos[n];
        float f[8] = {};
        if (p >= 0) {
            const int word = word_of(a, p);
            if (word >= 0 && word < a.vocab) {         // (HEAD_BAD is not)
                const float rest = a.rest[p];
                float h[8];
                unpack8(reinterpret_cast<const Bytes16 *>(a.w + (int64_t)word * d + c)->w, h);
#pragma unroll
                for (int x = 0; x < 8; ++x) f[x] = rest * h[x];
            }
            for (int s = 0; s < a.splits; ++s) {
                float h[8];
                load_f32x8<true>(a.slots, ((int64_t)s * a.g_rows + p) * d + c, 8, h);
#pragma unroll
                for (int x = 0; x < 8; ++x) f[x] += h[x];
                if (!low) continue;
                load_f32x8<true>(a.slots, ((int64_t)s * a.g_rows + low + p) * d + c, 8, h);
#pragma unroll
                for (int x = 0; x < 8; ++x) f[x] += h[x];
            }
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) f[x] *= unit;
        st_nt4(dx + n * d + c, u32x4_t{rne_bf16x2(f[0], f[1]), rne_bf16x2(f[2], f[3]), rne_bf16x2(f[4], f[5]), rne_bf16x2(f[6], f[7])});
    }
}

// The same for a piece of dW
template <int OUT>
__global__ __launch_bounds__(256) void dw_kernel(HeadArgs a) {
    const int64_t n = (int64_t)a.vn * a.d;
    const float unit = unit_of(a, kept_rows(a));
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 2048) {
        float f[8] = {};
        for (int s = 0; s < a.splits; ++s) {
            float h[8];
            load_f32x8<true>(a.slots, (int64_t)s * n + i, 8, h);
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] += h[x];
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) f[x] *= unit;
        const uint32_t gw[4] = {rne_bf16x2(f[0], f[1]), rne_bf16x2(f[2], f[3]), rne_bf16x2(f[4], f[5]), rne_bf16x2(f[6], f[7])};
        const int64_t o0 = (int64_t)a.v0 * a.d + i;
        if constexpr (OUT == OUT_STORE) st_nt4(a.out + o0, u32x4_t{gw[0], gw[1], gw[2], gw[3]});
        else accumulate8<OUT>(a, o0, gw);
    }
}

// ---------------------------------------------------------------------------
// plans
// ---------------------------------------------------------------------------

// The estimated time (us) of M x N results over K in tiles of T, `splits` shares of K: p per slab of 64 k of a tile with every CU
// busy, u for a tile that has its CU to itself, o for its start and end; the last round of tiles counts half if it is not full.
// Fitted to these times of whole backward passes with one product's tile (and shares of K) changed, us, best and others:
//   rows, words, width       logits 64  128  256     dx                                dW
//   4096, 16384, 384                265  237  230    (128, 4) 231 (256, 8) 240         (128, 1) 209 (256, 1) 227 (128, 2) 219
//   1024, 32000, 1024               271  241  230    (256, 12) 224 (128, 8) 227        (256, 1) 226 (128, 1) 229 (64, 1) 270
//   300, 50257, 768                 141  132  137    (128, 12) 129 (64, 12) 134        (128, 1) 132 (256, 1) 137
//   2000, 8000, 4096                478  422  401    (256, 2) 401 (128, 1) 420         (256, 1) 401 (128, 1) 418
//   16384, 512, 512                  77   76   76    (64, 1) 75 (128, 1) 76            (128, 16) 75 (64, 8) 76 (128, 1) 192
//   8191, 32000, 2048              3548 3035 2810    (256, 1) 2811 (256, 2) 2845       (256, 1) 2814 (256, 2) 3048
// and of forward passes (64, 128, 256): 700, 3000, 2048 34 40 58; 64, 128256, 4096 246 214 246; 300, 50257, 768 73 58 58.
static float tiles_cost(int64_t M, int64_t N, int64_t K, int T, int splits) {
    const int i = T == 256 ? 2 : T == 128 ? 1 : 0;
    constexpr float P[3] = {0.32f, 0.62f, 1.9f}, U[3] = {0.5f, 1.0f, 1.3f}, O[3] = {2.0f, 4.0f, 8.0f};
    const float all = (float)((M + T - 1) / T) * (float)((N + T - 1) / T) * (float)splits / 256.0f, n = 0.5f * (all + ceilf(all));
    return ceilf((float)K / 64.0f / (float)splits) * std::max(n * P[i], U[i]) + std::max(n, 1.0f) * O[i];
}
struct Tiling {
    int tile, splits;
};
// slots: 0: K is not split; 1: results go through a slot anyway (dx); 2: they do where K is split, in one more launch (dW)
static Tiling tiling(int64_t M, int64_t N, int64_t K, int slots, int most = 256) {
    Tiling best{128, 1};
    float least = 1e30f;
    for (const int T : {64, 128, 256})
        if (T <= most)
        for (int s = 1; s <= (slots ? 16 : 1); ++s) {
            if (s > 1 && K < 256 * s) break;
            // a slot is written and read: 8 bytes per result at 4 TB/s
            const float each = (float)(M * N) * 8.0f / 4e6f;
            const float c = tiles_cost(M, N, K, T, s) + (s == 1 ? 0.0f : slots == 1 ? (float)(s - 1) * each : (float)s * each + 5.0f);
            if (c < least) {
                least = c;
                best = {T, s};
            }
        }
    return best;
}

// Of G, about.  Gradients of 8192 rows, 128256 words of 4096: 20.62 ms in pieces of 128 MiB, 20.58 of 256, 20.32 of 512, 20.28 of
// 1024; of 8191 rows, 32000 words of 2048: 2.79, 2.81, 2.77, 2.77 ms.
constexpr int64_t PIECE_BYTES = int64_t(512) << 20;
constexpr int64_t PIECE_WORDS = 1 << 18;              // at most: a slab's rows of G span less than 2^31 bytes
// A call of at most so many rows packs them where it lists them, and adds up its losses, of at most so many parts, where it
// joins them: a launch less each (7 rows, 512 words of 256: 78 us a pass with the launches, 71 so).
constexpr int64_t FEW_ROWS = 32, FEW_PARTS = 1 << 12;
// Of so few rows the roundings of G's largest elements do not average out over a gradient's sums, and the products' tiles have rows to
// spare: there G / c is the sum of two bf16 numbers.  The rows that count decide, so the kernels do: a padded batch of thousands of
// rows has its second numbers behind the first ones in the same space.  Each row has its own g for the reduction "none", which c
// does not take out, so there more rows count as few.  Largest of 12 errors of dW against 64 bits, where the rounding of the results is 0.0017:
// with one number 33 rows, 512 words of 256 0.0022 (0.0027 "none"), 128 rows, 896 words of 144 0.0021 (0.0025); with two 0.0017.
// us of backward passes: 7 rows, 512 words of 256 15.3 with one and 16.9 with two, 128256 of 4096 584 and 636, 64 rows of the latter
// 664 and 790.
constexpr int64_t LO_ROWS = 32, LO_ROWS_NONE = 128;

struct HeadPlan {
    Tiling fwd, logits, dx, dw;
    int64_t piece, ldg, few, g_rows;                   // words of a piece
    size_t fwd_bytes, bwd_bytes, g_at, rest_at, dx_at, dw_at;
};
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

static HeadPlan head_plan(int64_t rows, int64_t vocab, int64_t d, int32_t reduction) {
    HeadPlan p{};
    p.fwd = tiling(rows, vocab, d, 0);
    const int64_t tn = (vocab + p.fwd.tile - 1) / p.fwd.tile;
    p.fwd_bytes = up256((size_t)tn * (size_t)rows * 8) + 2 * up256((size_t)rows * 4);
    // whole tiles of 256 words, in pieces of one size
    const int64_t most = std::min<int64_t>(std::max<int64_t>(PIECE_BYTES / 2 / std::max<int64_t>(rows, 1) / 256 * 256, 256), PIECE_WORDS);
    const int64_t pieces = (vocab + most - 1) / most;
    p.piece = std::min<int64_t>(((vocab + pieces - 1) / pieces + 255) / 256 * 256, (vocab + 7) / 8 * 8);
    p.ldg = p.piece;
    p.few = std::min<int64_t>(rows, reduction == HEAD_NONE ? LO_ROWS_NONE : LO_ROWS);
    p.g_rows = std::max(rows, 2 * p.few);
    const int64_t products = p.few == rows ? 2 * rows : rows;   // rows of G, if all count
    const int most_tile = p.few == rows ? 128 : 256;
    p.logits = tiling(rows, p.piece, d, 0, most_tile);
    p.dx = tiling(products, d, p.piece, 1, most_tile);
    p.dw = tiling(p.piece, d, rows, 2, most_tile);
    p.g_at = 0;
    p.rest_at = up256((size_t)p.g_rows * (size_t)p.ldg * 2);
    p.dx_at = p.rest_at + up256((size_t)rows * 4);
    p.dw_at = p.dx_at + up256((size_t)p.dx.splits * (size_t)p.g_rows * (size_t)d * 4);
    p.bwd_bytes = p.dw_at + (p.dw.splits > 1 ? up256((size_t)p.dw.splits * (size_t)p.piece * (size_t)d * 4) : 0);
    return p;
}

static int64_t tiles_of(int64_t M, int64_t N, const Tiling &t) { return (M + t.tile - 1) / t.tile * ((N + t.tile - 1) / t.tile) * t.splits; }
static int head_grids(const char *name, const HeadPlan &p, int64_t rows, int64_t vocab, int64_t d) {
    const int64_t most = std::max({tiles_of(rows, vocab, p.fwd), tiles_of(rows, p.piece, p.logits), tiles_of(p.g_rows, d, p.dx), tiles_of(p.piece, d, p.dw)});
    if (most < (1 << 22)) return MSR_OK;       // 512 threads each: fewer than 2^31 in a launch
    set_error("%s: too many tiles for a launch (%lld)", name, (long long)most);
    return MSR_ERR_ARG;
}

constexpr int64_t HEAD_WGS = 256;                     // work-groups of 256-wide tiles: one per CU
template <bool GRAD>
static int logits_launch(const HeadArgs &a, int T, int64_t tiles, hipStream_t s) {
    const unsigned grid = (unsigned)(T == 256 ? std::min<int64_t>(tiles, HEAD_WGS) : tiles);
    if (T == 256) hipLaunchKernelGGL((logits_kernel<GRAD, 256, 64>), dim3(grid), dim3(512), 0, s, a);
    else if (T == 128) hipLaunchKernelGGL((logits_kernel<GRAD, 128, 64>), dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((logits_kernel<GRAD, 64, 64>), dim3(grid), dim3(256), 0, s, a);
    return check_launch("logits_kernel");
}

template <int KIND, int OUT>
static int piece_launch(HeadArgs a, const Tiling &t, hipStream_t s) {
    const int64_t M = KIND == HD_DX ? a.g_rows : a.vn;
    a.tiles_n = (a.d + t.tile - 1) / t.tile;
    a.splits = t.splits;
    const unsigned grid = (unsigned)((M + t.tile - 1) / t.tile * a.tiles_n * t.splits);
    if (t.tile == 256) hipLaunchKernelGGL((piece_kernel<KIND, OUT, 256, 32, 4, 2>), dim3(grid), dim3(512), 0, s, a);
    else if (t.tile == 128) hipLaunchKernelGGL((piece_kernel<KIND, OUT, 128, 32, 3, 3>), dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((piece_kernel<KIND, OUT, 64, 64, 2, 2>), dim3(grid), dim3(256), 0, s, a);
    return check_launch("piece_kernel");
}

template <int OUT>
static int dw_launch(HeadArgs a, const HeadPlan &p, float *slots, hipStream_t s) {
    if (p.dw.splits == 1) return piece_launch<HD_DW, OUT>(a, p.dw, s);
    a.slots = slots;
    a.first = 1;
    const int rc = piece_launch<HD_DW, OUT_SLOTS>(a, p.dw, s);
    if (rc) return rc;
    a.splits = p.dw.splits;
    hipLaunchKernelGGL((dw_kernel<OUT>), dim3(grid_for((int64_t)a.vn * a.d / 8, 256, 256 * 8)), dim3(256), 0, s, a);
    return check_launch("dw_kernel");
}

static int head_check(const char *name, int64_t rows, int64_t vocab, int64_t d) {
    if (rows < 0 || rows >= (1 << 24) || vocab < 1 || vocab >= (1 << 24) || d < 8 || d % 8 || d > (1 << 16) || rows * vocab >= (int64_t(1) << 40)) {
        set_error("%s: need fewer than 2^24 rows and words, their product below 2^40, and a width that is a multiple of 8 up to 2^16 "
                  "(got %lld rows, %lld words, width %lld)", name, (long long)rows, (long long)vocab, (long long)d);
        return MSR_ERR_ARG;
    }
    return MSR_OK;
}

}  // namespace msr

using namespace msr;

extern "C" {

int msr_head_workspace_bytes(int64_t rows, int64_t vocab, int64_t d, size_t *forward, size_t *backward) {
    const int rc = head_check("msr_head_workspace_bytes", rows, vocab, d);
    if (rc) return rc;
    if (!forward || !backward) { set_error("msr_head_workspace_bytes: a pointer is NULL"); return MSR_ERR_ARG; }
    const HeadPlan p = head_plan(rows, vocab, d, HEAD_MEAN);
    *forward = p.fwd_bytes;
    *backward = std::max(p.bwd_bytes, head_plan(rows, vocab, d, HEAD_NONE).bwd_bytes);
    return MSR_OK;
}

int msr_head_plan(int64_t rows, int64_t vocab, int64_t d, int32_t *plan) {
    const int rc = head_check("msr_head_plan", rows, vocab, d);
    if (rc) return rc;
    if (!plan) { set_error("msr_head_plan: a pointer is NULL"); return MSR_ERR_ARG; }
    const HeadPlan p = head_plan(rows, vocab, d, HEAD_MEAN);
    const int32_t out[7] = {p.fwd.tile, p.logits.tile, p.dx.tile, p.dx.splits, p.dw.tile, p.dw.splits, (int32_t)p.piece};
    for (int i = 0; i < 7; ++i) plan[i] = out[i];
    return MSR_OK;
}

int msr_head_forward(const uint16_t *x, int64_t ldx, const uint16_t *w, const void *target, int32_t target_i64, int64_t ignore_index,
                     int64_t rows, int64_t vocab, int64_t d, int32_t reduction, uint16_t *packed, int32_t *kept, float *sums,
                     float *loss, void *workspace, size_t workspace_bytes, msr_stream_t stream) {
    const char *const name = "msr_head_forward";
    int rc = head_check(name, rows, vocab, d);
    if (rc) return rc;
    if (reduction < HEAD_NONE || reduction > HEAD_MEAN || !w || !kept || (rows > 0 && (!x || !target || !packed || !sums)) ||
        ((rows > 0 || reduction != HEAD_NONE) && !loss) || ldx < d) {
        set_error("%s: bad arguments", name);
        return MSR_ERR_ARG;
    }
    if (!aligned(x, 2) || !aligned(w, 16) || !aligned(packed, 16) || !aligned(target, target_i64 ? 8 : 4) || !aligned(kept, 4) ||
        !aligned(sums, 8) || !aligned(loss, 4) || !aligned(workspace, 16)) {
        set_error("%s: w, packed and the workspace must be 16-byte aligned, sums 8-byte aligned, the others to their types", name);
        return MSR_ERR_ALIGN;
    }
    const HeadPlan p = head_plan(rows, vocab, d, reduction);
    if ((rc = head_grids(name, p, rows, vocab, d))) return rc;
    if (rows > 0 && (!workspace || workspace_bytes < p.fwd_bytes)) {
        set_error("%s: workspace of %zu bytes is smaller than the %zu required", name, workspace_bytes, p.fwd_bytes);
        return MSR_ERR_WORKSPACE;
    }
    const size_t n = (size_t)rows;
    const Range r[8] = {{packed, 2 * n * (size_t)d}, {kept, 4 * (3 * n + 1)}, {sums, 8 * n}, {loss, reduction == HEAD_NONE ? 4 * n : 4},
                        {workspace, rows ? p.fwd_bytes : 0}, {x, rows ? 2 * ((n - 1) * (size_t)ldx + (size_t)d) : 0},
                        {w, 2 * (size_t)vocab * (size_t)d}, {target, n * (target_i64 ? 8 : 4)}};
    rc = ranges_apart(name, r, 8, 5);
    if (rc) return rc;
    const int T = p.fwd.tile;
    const int64_t tn = (vocab + T - 1) / T, tiles = (rows + T - 1) / T * tn;
    hipStream_t s = (hipStream_t)stream;
    HeadArgs a{};
    a.x = packed; a.w = w; a.kept = kept; a.sums = reinterpret_cast<float2 *>(sums);
    a.part = static_cast<float2 *>(workspace);
    char *const after = static_cast<char *>(workspace) + up256((size_t)tn * n * 8);
    a.picked = reinterpret_cast<float *>(after);
    float *const losses = reduction == HEAD_NONE ? loss : reinterpret_cast<float *>(after + up256(n * 4));
    a.rows = (int)rows; a.vocab = (int)vocab; a.d = (int)d; a.reduction = reduction;
    a.v0 = 0; a.vn = (int)vocab; a.tiles_n = (int)tn;
    ListArgs l{target, ignore_index, kept, kept + 1 + 2 * rows, reduction == HEAD_NONE ? loss : nullptr, (int)rows, (int)vocab, target_i64 != 0};
    const bool few = rows <= FEW_ROWS, alone = few && reduction != HEAD_NONE && rows * tn <= FEW_PARTS;
    if (few) {
        l.x = x; l.ldx = ldx; l.packed = packed; l.d = (int)d;
    }
    hipLaunchKernelGGL(list_kernel, dim3(1), dim3(LIST_THREADS), 0, s, l);
    if ((rc = check_launch("list_kernel"))) return rc;
    if (rows > 0) {
        if (!few) {
            hipLaunchKernelGGL(pack_kernel, dim3(grid_for(rows, 4, 256 * 8)), dim3(256), 0, s, x, ldx, packed, kept, (int)rows, (int)d);
            if ((rc = check_launch("pack_kernel"))) return rc;
        }
        if ((rc = logits_launch<false>(a, T, tiles, s))) return rc;
        hipLaunchKernelGGL(join_kernel, dim3(alone ? 1 : (unsigned)((rows + 15) / 16)), dim3(256), 0, s, a, losses, alone ? loss : nullptr);
        if ((rc = check_launch("join_kernel"))) return rc;
    }
    if (reduction != HEAD_NONE && !(alone && rows > 0)) {
        hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, s, losses, kept, (int)rows, reduction == HEAD_MEAN, loss);
        rc = check_launch("total_kernel");
    }
    return rc;
}

int msr_head_backward(const uint16_t *packed, const uint16_t *w, const int32_t *kept, const float *sums, const float *dloss,
                      int64_t rows, int64_t vocab, int64_t d, int32_t reduction, uint16_t *dx, uint16_t *dw, int32_t noise_mode,
                      uint32_t seed, int32_t zero_init, const uint16_t *inject, void *workspace, size_t workspace_bytes,
                      msr_stream_t stream) {
    const char *const name = "msr_head_backward";
    int rc = head_check(name, rows, vocab, d);
    if (rc) return rc;
    if (reduction < HEAD_NONE || reduction > HEAD_MEAN || !w || !kept || (rows > 0 && (!packed || !sums || !dloss)) || noise_mode < -1 ||
        noise_mode > 2 || (noise_mode == NOISE_INJECT && !inject)) {
        set_error("%s: bad arguments", name);
        return MSR_ERR_ARG;
    }
    if (!aligned(w, 16) || !aligned(packed, 16) || !aligned(dx, 16) || !aligned(dw, 16) || !aligned(kept, 4) || !aligned(sums, 8) ||
        !aligned(dloss, 4) || !aligned(inject, 2) || !aligned(workspace, 16)) {
        set_error("%s: operands and the workspace must be 16-byte aligned, sums 8-byte aligned, kept and dloss to their types", name);
        return MSR_ERR_ALIGN;
    }
    const HeadPlan p = head_plan(rows, vocab, d, reduction);
    if ((rc = head_grids(name, p, rows, vocab, d))) return rc;
    if (rows > 0 && (!workspace || workspace_bytes < p.bwd_bytes)) {
        set_error("%s: workspace of %zu bytes is smaller than the %zu required", name, workspace_bytes, p.bwd_bytes);
        return MSR_ERR_WORKSPACE;
    }
    const size_t n = (size_t)rows, wb = 2 * (size_t)vocab * (size_t)d;
    const Range r[9] = {{dx, 2 * n * (size_t)d}, {dw, wb}, {workspace, rows ? p.bwd_bytes : 0}, {packed, 2 * n * (size_t)d}, {w, wb},
                        {kept, 4 * (3 * n + 1)}, {sums, 8 * n}, {dloss, reduction == HEAD_NONE ? 4 * n : 4},
                        {inject, noise_mode == NOISE_INJECT ? wb : 0}};
    rc = ranges_apart(name, r, 9, 3);
    if (rc) return rc;
    hipStream_t s = (hipStream_t)stream;
    HeadArgs a{};
    char *const ws = static_cast<char *>(workspace);
    a.x = packed; a.w = w; a.kept = kept; a.sums = reinterpret_cast<float2 *>(const_cast<float *>(sums)); a.dloss = dloss;
    a.g = reinterpret_cast<uint16_t *>(ws); a.ldg = p.ldg; a.few = (int)p.few; a.g_rows = (int)p.g_rows; a.out = dw;
    a.rows = (int)rows; a.vocab = (int)vocab; a.d = (int)d; a.reduction = reduction; a.zero_init = zero_init != 0;
    a.ns.key = seed_key(seed, 0);
    a.ns.inject = inject;
    a.rest = reinterpret_cast<float *>(ws + p.rest_at);
    float *const dxs = reinterpret_cast<float *>(ws + p.dx_at), *const dws = reinterpret_cast<float *>(ws + p.dw_at);
    const int T = p.logits.tile;
    for (int64_t v0 = 0; v0 < vocab && (dx || dw); v0 += p.piece) {
        a.v0 = (int)v0;
        a.vn = (int)std::min(p.piece, vocab - v0);
        if (rows > 0) {
            a.tiles_n = (a.vn + T - 1) / T;
            const int64_t tiles = (rows + T - 1) / T * a.tiles_n;
            if ((rc = logits_launch<true>(a, T, tiles, s))) return rc;
            if (dx) {
                a.slots = dxs;
                a.first = v0 == 0;
                if ((rc = piece_launch<HD_DX, OUT_SLOTS>(a, p.dx, s))) return rc;
            }
        }
        if (!dw) continue;
        if (noise_mode < 0) rc = dw_launch<OUT_STORE>(a, p, dws, s);
        else MSR_DISPATCH_NOISE(noise_mode, MODE, rc = (dw_launch<MODE>(a, p, dws, s)));
        if (rc) return rc;
    }
    if (dx && rows > 0) {
        a.slots = dxs;
        a.splits = p.dx.splits;
        hipLaunchKernelGGL(dx_kernel, dim3(grid_for(rows * (d / 8), 256, 256 * 8)), dim3(256), 0, s, a, dx);
        rc = check_launch("dx_kernel");
    }
    return rc;
}

}  // extern "C"
