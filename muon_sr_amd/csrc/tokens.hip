// Tokens sorted by expert and back, for mixture-of-experts layers.
//
// Order: a stable counting sort of the n = tokens * k slots by expert.  Slot s of expert e
// gets row  offsets[e] + #{s' < s : expert(s') = e}.  The slots are cut into one chunk per
// work-group.  place_kernel needs the slots per expert in the chunks before its own, and in all for the
// offsets: up to ORD_SELF slots every work-group counts them all itself; beyond that count_kernel counts
// each chunk, and the work-groups add its counts (a few thousand numbers from L2).  It then ranks its
// slots wave by wave, 64 at a time by ballots, one per bit of the expert number: only the counts are
// atomic, no order depends on them.  Dropped slots count as one more expert, which gives the rows without
// a slot.  One or two launches of some 4 (14 slots) to 18 us (262144 of them), far above what their bytes take; how much
// of that is latency and how much the LDS atomics, two per slot up to ORD_SELF, was not told apart.
//
// The four passes between tokens and rows (see the header) move d elements per slot and do
// next to nothing with them, so HBM bounds them.  All are written from the token's side: a piece of a
// token's k rows is read or written by the same wave, so x and dy are read once, not k times, y
// and dx are sums in registers, and nothing is added atomically.
#include <type_traits>

#include "common.hpp"
#include "vecio.hpp"
#include "../../include/muon_sr_amd.h"

namespace msr {

// ---------------------------------------------------------------------------
// order
// ---------------------------------------------------------------------------

constexpr int ORD_THREADS = 1024, ORD_WAVES = ORD_THREADS / 64;
// Slots of a work-group, while there are at most ORD_MAXWG of them: half as many up to 65536 (16384 slots over 64
// experts 9.1 us with 1024, 9.9 with 2048; 262144 over 128 17.0 and 15.1).
constexpr int order_chunk(int64_t n) { return n <= 65536 ? 1024 : 2048; }
constexpr int ORD_MAXWG = 256;
constexpr int ORD_SELF = 32768;          // slots that every work-group counts by itself
constexpr int ORD_AHEAD = 8;             // chunks' counts that a thread loads at once

struct OrderArgs {
    const void *ids;
    int32_t *offsets, *position, *source;
    int32_t *counts;                     // [work-groups][experts + 1]
    int64_t n;                           // slots
    int32_t experts, i64, chunk;
};

__device__ __forceinline__ int expert_of(const OrderArgs &a, int64_t s) {
    if (a.i64) {
        const int64_t e = static_cast<const int64_t *>(a.ids)[s];
        return e >= 0 && e < a.experts ? (int)e : a.experts;
    }
    const int32_t e = static_cast<const int32_t *>(a.ids)[s];
    return e >= 0 && e < a.experts ? e : a.experts;
}

__global__ __launch_bounds__(ORD_THREADS) void count_kernel(OrderArgs a) {
    __shared__ int hist[MSR_EXPERTS_MAX + 1];
    for (int e = threadIdx.x; e <= a.experts; e += ORD_THREADS) hist[e] = 0;
    __syncthreads();
    const int64_t s0 = (int64_t)blockIdx.x * a.chunk, s1 = min(s0 + a.chunk, a.n);
    for (int64_t s = s0 + threadIdx.x; s < s1; s += ORD_THREADS) atomicAdd(&hist[expert_of(a, s)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= a.experts; e += ORD_THREADS) a.counts[(int64_t)blockIdx.x * (a.experts + 1) + e] = hist[e];
}

__global__ __launch_bounds__(ORD_THREADS) void place_kernel(OrderArgs a) {
    extern __shared__ int wave_at[];                 // [ORD_WAVES][experts + 1]: counts, then the next row
    __shared__ int wave_sum[ORD_WAVES], all[MSR_EXPERTS_MAX + 1], before[MSR_EXPERTS_MAX + 1];
    const int E1 = a.experts + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < ORD_WAVES * E1; i += ORD_THREADS) wave_at[i] = 0;
    for (int e = tid; e < E1; e += ORD_THREADS) all[e] = before[e] = 0;
    __syncthreads();
    // each wave takes a run of the chunk's slots
    const int run = a.chunk / ORD_WAVES;
    const int64_t s0 = (int64_t)blockIdx.x * a.chunk + (int64_t)wave * run, s1 = min(s0 + run, a.n);
    int *const mine = wave_at + wave * E1;
    // Each expert's slots in all chunks and in those before this one.
    if (!a.counts) {
        // four loads in flight; a slot counts in `all`, and in `before` or its wave's count of this chunk
        const int c0 = (int)blockIdx.x * a.chunk, n = (int)a.n;
        for (int t = tid; t < n; t += 4 * ORD_THREADS) {
            int e[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) e[u] = t + u * ORD_THREADS < n ? expert_of(a, t + u * ORD_THREADS) : -1;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (e[u] < 0) continue;
                atomicAdd(&all[e[u]], 1);
                const int at = t + u * ORD_THREADS - c0;
                if (at < 0) atomicAdd(&before[e[u]], 1);
                else if (at < a.chunk) atomicAdd(&wave_at[at / run * E1 + e[u]], 1);
            }
        }
    } else {
        for (int64_t s = s0 + lane; s < s1; s += 64) atomicAdd(&mine[expert_of(a, s)], 1);
        // a thread per expert and part of the chunks (the dropped slots: one wave), eight loads in flight
        const int cols = (a.experts + 63) & ~63, parts = ORD_THREADS / cols, chunks = gridDim.x;
        auto add = [&](int e, int from, int step) __attribute__((always_inline)) {
            int n = 0, m = 0;
            for (int b = from; b < chunks; b += ORD_AHEAD * step) {
                int c[ORD_AHEAD];
#pragma unroll
                for (int u = 0; u < ORD_AHEAD; ++u) c[u] = b + u * step < chunks ? a.counts[(int64_t)(b + u * step) * E1 + e] : 0;
#pragma unroll
                for (int u = 0; u < ORD_AHEAD; ++u) {
                    n += c[u];
                    m += b + u * step < (int)blockIdx.x ? c[u] : 0;
                }
            }
            atomicAdd(&all[e], n);
            atomicAdd(&before[e], m);
        };
        if (tid < parts * cols && tid % cols < a.experts) add(tid % cols, tid / cols, parts);
        if (wave == ORD_WAVES - 1) add(a.experts, lane, 64);
    }
    __syncthreads();
    // Thread e: the sum over the experts before e gives its first row.  experts + 1 <= 1025 numbers: two
    // rounds at most.
    int carry = 0;
    for (int e0 = 0; e0 < E1; e0 += ORD_THREADS) {
        const int e = e0 + tid, n = e < E1 ? all[e] : 0;
        const int incl = wave_scan(n);
        if (lane == 63) wave_sum[wave] = incl;
        __syncthreads();
        int first = carry + incl - n, total = 0;
        for (int w = 0; w < ORD_WAVES; ++w) {
            first += w < wave ? wave_sum[w] : 0;
            total += wave_sum[w];
        }
        carry += total;
        if (e < E1) {
            if (blockIdx.x == 0) a.offsets[e] = first;   // expert `experts` is the dropped slots': their first row
            int at = first + before[e], c[ORD_WAVES];
#pragma unroll
            for (int w = 0; w < ORD_WAVES; ++w) c[w] = wave_at[w * E1 + e];
#pragma unroll
            for (int w = 0; w < ORD_WAVES; ++w) {
                wave_at[w * E1 + e] = at;
                at += c[w];
            }
        }
        __syncthreads();
    }
    // Ranks: the lanes with this lane's expert, from one ballot per bit of its number.
    const int bits = 32 - __clz(a.experts);
    for (int64_t s = s0; s < s1; s += 64) {
        const bool on = s + lane < s1;
        const int e = on ? expert_of(a, s + lane) : 0;
        uint64_t same = __ballot(on);
        for (int b = 0; b < bits; ++b) {
            const uint64_t m = __ballot((e >> b) & 1);
            same &= (e >> b) & 1 ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (on) {
            const int row = mine[e] + rank;
            const bool kept = e < a.experts;
            a.position[s + lane] = kept ? row : -1;
            a.source[row] = kept ? (int)(s + lane) : -1;
        }
        // a wave's LDS accesses execute in order: every lane has read mine[e] before the last lane
        // of an expert moves it on, and reads what that lane wrote in the next round
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (on && (same >> lane) == 1) mine[e] += rank + 1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

struct OrderPlan {
    int wgs, chunk;
};
static OrderPlan order_plan(int64_t n) {
    const int64_t wgs = std::min<int64_t>(std::max<int64_t>((n + order_chunk(n) - 1) / order_chunk(n), 1), ORD_MAXWG);
    const int64_t chunk = ((n + wgs - 1) / wgs + ORD_THREADS - 1) / ORD_THREADS * ORD_THREADS;   // whole waves' runs
    return {(int)std::max<int64_t>((n + chunk - 1) / std::max<int64_t>(chunk, 1), 1), (int)std::max<int64_t>(chunk, ORD_THREADS)};
}

// ---------------------------------------------------------------------------
// passes between tokens and rows
// ---------------------------------------------------------------------------

constexpr int MOVE_THREADS = 256, MOVE_WAVES = MOVE_THREADS / 64;
// Work-groups at most: four times what the card holds (combine's gradient of 32768 x 4 of width 256 26 us so, 29 with
// 8 per CU).
constexpr int MOVE_GRID = 256 * 32;

// 16 bytes of a row per lane (VEC), or one element, as they lie in memory: converted where they are used, so that the
// loads of several rows are in flight together.  Stores are non-temporal: the four passes over 32768 tokens x 8
// of width 2048 take 1100 us so (5.4 TB/s), 1166 with plain stores, and over 8192 x 2 73 and 77 us; loads are not,
// as the rows were mostly written just before.
template <typename T, bool VEC>
struct Pack {
    static constexpr int N = VEC ? 16 / (int)sizeof(T) : 1;
    using V = std::conditional_t<!VEC, T, std::conditional_t<sizeof(T) == 2, u32x4_t, f32x4_t>>;
    V v;
    __device__ __forceinline__ void load(const T *p) { v = *reinterpret_cast<const V *>(p); }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (VEC) __builtin_nontemporal_store(v, reinterpret_cast<V *>(p));
        else *p = v;
    }
    __device__ __forceinline__ void zero() { v = V{}; }
    __device__ __forceinline__ void get(float (&f)[N]) const {
        if constexpr (!VEC) {
            if constexpr (sizeof(T) == 2) f[0] = bf16_to_f32(v);
            else f[0] = v;
        } else if constexpr (sizeof(T) == 2) {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            unpack8(w, f);
        } else {
            f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
        }
    }
    __device__ __forceinline__ void set(const float (&f)[N]) {
        if constexpr (!VEC) {
            if constexpr (sizeof(T) == 2) v = (T)rne_bf16(f[0]);
            else v = f[0];
        } else if constexpr (sizeof(T) == 2) {
            v = u32x4_t{rne_bf16x2(f[0], f[1]), rne_bf16x2(f[2], f[3]), rne_bf16x2(f[4], f[5]), rne_bf16x2(f[6], f[7])};
        } else {
            v = f32x4_t{f[0], f[1], f[2], f[3]};
        }
    }
};

struct MoveArgs {
    const void *tok;             // x or dy: [tokens] rows of ldtok elements
    int64_t ldtok;
    const void *rows;            // [n][d], read
    const void *w;               // [n] slot weights
    void *out;                   // rows or dx, y, drows
    void *dw;                    // [n]
    const int32_t *position, *offsets;
    int64_t tokens, n, d;
    int32_t k, experts, w32;
    int32_t pieces, share;       // of a row; 2^share waves of a work-group take them in turn (set by the launch)
};

// A token's slots, 64 at a time: lane j holds the row (-1: none) and the weight of slot first + j, so that one
// load of each fetches them all ahead of the rows.
struct Slots {
    int row;
    float w;
    __device__ __forceinline__ void load(const MoveArgs &a, int64_t first, int count) {
        const int lane = threadIdx.x & 63;
        row = -1;
        w = 0.0f;
        if (lane < count) {
            row = a.position[first + lane];
            if (row >= a.n) row = -1;
            if (a.w) w = a.w32 ? static_cast<const float *>(a.w)[first + lane] : bf16_to_f32(static_cast<const uint16_t *>(a.w)[first + lane]);
        }
    }
    __device__ __forceinline__ int row_of(int j) const { return __builtin_amdgcn_readlane(row, j); }
    __device__ __forceinline__ float weight_of(int j) const {
        return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(w), j));
    }
};
// A wave's piece of a row: U packs per lane, 64 packs apart, from column c on.  Whole rows (or 4 KiB of
// them) at a time: a wave that went through a token's rows 1 KiB at a time would return to each row's memory page
// several times (combine of 32768 x 8 rows of 4 KiB 231 us so, 221 a whole row at a time).
template <typename T, bool VEC, int U>
struct Piece {
    static constexpr int N = Pack<T, VEC>::N, WIDTH = 64 * N * U;
    Pack<T, VEC> p[U];
    static __device__ __forceinline__ int64_t col(int64_t c, int u) { return c + ((int64_t)u * 64 + (threadIdx.x & 63)) * N; }
    __device__ __forceinline__ void load(const T *row, int64_t c, int64_t d) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (col(c, u) < d) p[u].load(row + col(c, u));
            else p[u].zero();
        }
    }
    __device__ __forceinline__ void store(T *row, int64_t c, int64_t d) const {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (col(c, u) < d) p[u].store(row + col(c, u));
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int u = 0; u < U; ++u) p[u].zero();
    }
};
// Rows whose loads are in flight together (32768 x 8 of width 2048: combine 221 us, 227 with two; 300 x 8 of
// width 7168: 7.5 and 7.9).
constexpr int MOVE_AHEAD = 4;

// Rows without a slot, [offsets[experts], n), to zero: the waves of the launch in turn.
template <typename T, bool VEC>
__device__ __forceinline__ void zero_tail(const MoveArgs &a, int64_t wave, int64_t waves) {
    constexpr int N = Pack<T, VEC>::N;
    Pack<T, VEC> z;
    z.zero();
    for (int64_t r = max(0, a.offsets[a.experts]) + wave; r < a.n; r += waves)
        for (int64_t c = (int64_t)(threadIdx.x & 63) * N; c < a.d; c += 64 * N) z.store(static_cast<T *>(a.out) + r * a.d + c);
}

__device__ __forceinline__ int64_t this_wave() {
    return (int64_t)blockIdx.x * MOVE_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}

// rows[position[t][j]] = x[t]
template <typename T, bool VEC, int U>
__global__ __launch_bounds__(MOVE_THREADS) void dispatch_kernel(MoveArgs a) {
    using P = Piece<T, VEC, U>;
    const int64_t waves = (int64_t)gridDim.x * MOVE_WAVES;
    for (int64_t i = this_wave(); i >> a.share < a.tokens; i += waves) {
        const int64_t t = i >> a.share;
        for (int64_t c = (i & ((1 << a.share) - 1)) * P::WIDTH; c < a.d; c += (int64_t)P::WIDTH << a.share) {
            P v;
            v.load(static_cast<const T *>(a.tok) + t * a.ldtok, c, a.d);
            for (int j0 = 0; j0 < a.k; j0 += 64) {
                const int js = min(64, a.k - j0);
                Slots s;
                s.load(a, t * a.k + j0, js);
                for (int j = 0; j < js; ++j) {
                    const int p = s.row_of(j);
                    if (p >= 0) v.store(static_cast<T *>(a.out) + (int64_t)p * a.d, c, a.d);
                }
            }
        }
    }
    zero_tail<T, VEC>(a, this_wave(), waves);
}

// out[t] = sum_j w[t][j] rows[position[t][j]], or without weights (WEIGHTED false), j ascending
template <typename T, bool VEC, int U, bool WEIGHTED>
__global__ __launch_bounds__(MOVE_THREADS) void combine_kernel(MoveArgs a) {
    using P = Piece<T, VEC, U>;
    constexpr int A = MOVE_AHEAD;
    for (int64_t i = this_wave(); i >> a.share < a.tokens; i += (int64_t)gridDim.x * MOVE_WAVES) {
        const int64_t t = i >> a.share;
        Slots s;
        s.load(a, t * a.k, min(64, a.k));
        for (int64_t c = (i & ((1 << a.share) - 1)) * P::WIDTH; c < a.d; c += (int64_t)P::WIDTH << a.share) {
            float sum[U][P::N] = {};
            for (int j0 = 0; j0 < a.k; j0 += A) {
                if (a.k > 64 && (j0 & 63) == 0) s.load(a, t * a.k + j0, min(64, a.k - j0));
                P v[A];
#pragma unroll
                for (int y = 0; y < A; ++y) {
                    const int p = j0 + y < a.k ? s.row_of((j0 + y) & 63) : -1;
                    if (p >= 0) v[y].load(static_cast<const T *>(a.rows) + (int64_t)p * a.d, c, a.d);
                }
#pragma unroll
                for (int y = 0; y < A; ++y) {
                    if (j0 + y >= a.k || s.row_of((j0 + y) & 63) < 0) continue;
                    const float w = WEIGHTED ? s.weight_of((j0 + y) & 63) : 1.0f;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        float f[P::N];
                        v[y].p[u].get(f);
#pragma unroll
                        for (int x = 0; x < P::N; ++x) sum[u][x] = WEIGHTED ? __builtin_fmaf(w, f[x], sum[u][x]) : sum[u][x] + f[x];
                    }
                }
            }
            P out;
#pragma unroll
            for (int u = 0; u < U; ++u) out.p[u].set(sum[u]);
            out.store(static_cast<T *>(a.out) + t * a.d, c, a.d);
        }
    }
}

// The sums of x and of y over the wave, in registers: lanes 0 to 31 add up x, the others y.
struct Sums2 {
    float v;
    __device__ __forceinline__ Sums2(float x, float y) {
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
        v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
        const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(q[0]) + __uint_as_float(q[1]);
        v = turned<0x128>(turned<0x124>(turned<0x122>(turned<0x121>(v))));
    }
    template <int CTRL>   // row_ror: 1, 2, 4, 8 lanes within 16
    static __device__ __forceinline__ float turned(float x) {
        return x + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
    }
    __device__ __forceinline__ float of(int y) const { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), y * 32)); }
};

// drows[position[t][j]] = w[t][j] dy[t];  dw[t][j] = <dy[t], rows[position[t][j]]>: the parts of the waves that
// share a token are added in their order
template <typename T, bool VEC, int U, bool SHARED>
__global__ __launch_bounds__(MOVE_THREADS) void combine_grad_kernel(MoveArgs a) {
    using P = Piece<T, VEC, U>;
    constexpr int A = MOVE_AHEAD;
    static_assert(A % 2 == 0, "dw is summed in pairs");
    __shared__ float part[SHARED ? MOVE_WAVES : 1][64];
    const int share = SHARED ? a.share : 0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w0 = wave & ((1 << share) - 1);
    const int64_t c0 = (int64_t)w0 * P::WIDTH;
    const bool whole = a.pieces <= 1 << share;     // the wave's part of dy[t] stays in registers
    // every wave of the work-group makes the same rounds (barriers)
    for (int64_t i0 = (int64_t)blockIdx.x * MOVE_WAVES; i0 >> share < a.tokens; i0 += (int64_t)gridDim.x * MOVE_WAVES) {
        const int64_t t = (i0 + wave) >> share;
        const bool on = t < a.tokens;
        const T *dy = static_cast<const T *>(a.tok) + t * a.ldtok;
        P g;
        if (whole && on) g.load(dy, c0, a.d);
        for (int j1 = 0; j1 < a.k; j1 += 64) {
            const int js = on ? min(64, a.k - j1) : 0;
            Slots s;
            s.load(a, t * a.k + j1, js);
            float mine = 0.0f;                       // lane j: the dot product of slot j1 + j
            for (int j0 = 0; j0 < js; j0 += A) {
                float dot[A] = {};
                for (int64_t c = c0; c < a.d; c += (int64_t)P::WIDTH << share) {
                    if (!whole) g.load(dy, c, a.d);
                    if (a.dw) {
                        P r[A];
#pragma unroll
                        for (int y = 0; y < A; ++y) {
                            const int p = j0 + y < js ? s.row_of(j0 + y) : -1;
                            if (p >= 0) r[y].load(static_cast<const T *>(a.rows) + (int64_t)p * a.d, c, a.d);
                        }
#pragma unroll
                        for (int y = 0; y < A; ++y) {
                            if (j0 + y >= js || s.row_of(j0 + y) < 0) continue;
#pragma unroll
                            for (int u = 0; u < U; ++u) {
                                float f[P::N], h[P::N];
                                g.p[u].get(f);
                                r[y].p[u].get(h);
#pragma unroll
                                for (int x = 0; x < P::N; ++x) dot[y] = __builtin_fmaf(f[x], h[x], dot[y]);
                            }
                        }
                    }
                    if (a.out) {
#pragma unroll
                        for (int y = 0; y < A; ++y) {
                            const int p = j0 + y < js ? s.row_of(j0 + y) : -1;
                            if (p < 0) continue;
                            const float w = s.weight_of(j0 + y);
                            P o;
#pragma unroll
                            for (int u = 0; u < U; ++u) {
                                float f[P::N];
                                g.p[u].get(f);
#pragma unroll
                                for (int x = 0; x < P::N; ++x) f[x] *= w;
                                o.p[u].set(f);
                            }
                            o.store(static_cast<T *>(a.out) + (int64_t)p * a.d, c, a.d);
                        }
                    }
                }
                if (a.dw) {
#pragma unroll
                    for (int y = 0; y < A; y += 2) {
                        const Sums2 sums(dot[y], dot[y + 1]);
                        mine = lane == j0 + y ? sums.of(0) : lane == j0 + y + 1 ? sums.of(1) : mine;
                    }
                }
            }
            if (a.dw) {
                if constexpr (SHARED) {
                    part[wave][lane] = mine;
                    __syncthreads();
                    mine = part[wave - w0][lane];
                    for (int w = 1; w < 1 << share; ++w) mine = mine + part[wave - w0 + w][lane];
                    __syncthreads();
                }
                if (w0 == 0 && lane < js) {
                    const int64_t at = t * a.k + j1 + lane;
                    if (a.w32) static_cast<float *>(a.dw)[at] = mine;
                    else static_cast<uint16_t *>(a.dw)[at] = (uint16_t)rne_bf16(mine);
                }
            }
        }
    }
    if (a.out) zero_tail<T, VEC>(a, this_wave(), (int64_t)gridDim.x * MOVE_WAVES);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

static bool touch(const void *p, size_t np, const void *q, size_t nq) {
    const uintptr_t u = (uintptr_t)p, v = (uintptr_t)q;
    return p && q && np && nq && u < v + nq && v < u + np;
}

static int move_check(const char *name, const MoveArgs &a, int32_t elem, int32_t welem) {
    if (a.tokens < 0 || a.k < 1 || a.d < 0 || a.tokens > (int64_t(1) << 30) / a.k || a.d > (int64_t(1) << 30) ||
        (elem != MSR_BF16 && elem != MSR_F32) || (welem != MSR_BF16 && welem != MSR_F32)) {
        set_error("%s: bad sizes or types (tokens %lld, k %d, d %lld)", name, (long long)a.tokens, (int)a.k, (long long)a.d);
        return MSR_ERR_ARG;
    }
    return MSR_OK;
}

static bool move_vec(int64_t d, int64_t ld, size_t es, const void *p, const void *q, const void *r) {
    const int64_t n = 16 / (int64_t)es;
    return d % n == 0 && ld % n == 0 && aligned(p, 16) && aligned(q, 16) && aligned(r, 16);
}

// Sets the pieces of a pass's rows; returns their packs per lane: at most 4, and as even as the row allows (6 packs: 2
// pieces of 3).  Up to 4 waves share a token's pieces, so that few tokens of wide rows have waves too: 300 x 8 of width
// 7168 take 8, 8, 15 and 8 us (dispatch, combine, its gradient, dispatch's), with a wave per token 8, 19, 36 and 19; of
// 32768 x 2 of width 4096 119, 146, 264, 145 and 122, 154, 286, 154.  Rows moved by single elements gain only while
// tokens are few (width 1001: 2048 x 2 5.2, 5.5, 9.3, 5.1 us shared, 5.7, 6.5, 9.9, 6.1 not; 8192 x 2 10.6, 13.2, 26.8,
// 12.5 and 10.1, 11.2, 22.7, 11.3).
static int move_plan(MoveArgs &a, int32_t elem, bool vec) {
    const int64_t pack = 64 * (!vec ? 1 : elem == MSR_BF16 ? 8 : 4), packs = std::max<int64_t>((a.d + pack - 1) / pack, 1);
    const int64_t u = (packs + (packs + 3) / 4 - 1) / ((packs + 3) / 4);
    a.pieces = (int32_t)((packs + u - 1) / u);
    a.share = !vec && a.tokens > 4096 ? 0 : a.pieces > 2 ? 2 : a.pieces - 1;
    return (int)u;
}
// launch(type, VEC, U): the pass's kernel
template <typename T, typename V, typename F>
static void move_packs(int u, F launch) {
    if (u > 3) launch(T{}, V{}, std::integral_constant<int, 4>{});
    else if (u > 2) launch(T{}, V{}, std::integral_constant<int, 3>{});
    else if (u > 1) launch(T{}, V{}, std::integral_constant<int, 2>{});
    else launch(T{}, V{}, std::integral_constant<int, 1>{});
}
template <typename F>
static void move_launch(int32_t elem, bool vec, int u, F launch) {
    if (elem == MSR_BF16) {
        if (vec) move_packs<uint16_t, std::true_type>(u, launch);
        else move_packs<uint16_t, std::false_type>(u, launch);
    } else {
        if (vec) move_packs<float, std::true_type>(u, launch);
        else move_packs<float, std::false_type>(u, launch);
    }
}
static dim3 move_grid(const MoveArgs &a) {
    const int64_t wgs = ((a.tokens << a.share) + MOVE_WAVES - 1) / MOVE_WAVES;
    return dim3((unsigned)std::min<int64_t>(std::max<int64_t>(wgs, 1), MOVE_GRID));
}
#define MOVE_LAUNCH(KERNEL, ...)                                                                                       \
    move_launch(elem, vec, packs, [&](auto t, auto v, auto u) {                                                              \
        hipLaunchKernelGGL((KERNEL<decltype(t), decltype(v)::value, decltype(u)::value __VA_OPT__(, ) __VA_ARGS__>),         \
                           move_grid(a), dim3(MOVE_THREADS), 0, (hipStream_t)stream, a);                               \
    })

}  // namespace msr

using namespace msr;

extern "C" {

int msr_order_workspace_bytes(int64_t tokens, int32_t k, int32_t experts, size_t *bytes) {
    if (!bytes || tokens < 0 || k < 1 || experts < 1 || experts > MSR_EXPERTS_MAX || tokens >= (int64_t(1) << 30) / k) {
        set_error("msr_order_workspace_bytes: bad arguments (tokens %lld, k %d, %d experts)", (long long)tokens, (int)k, (int)experts);
        return MSR_ERR_ARG;
    }
    const OrderPlan p = order_plan(tokens * k);
    *bytes = tokens * k > ORD_SELF ? (size_t)p.wgs * (size_t)(experts + 1) * 4 : 0;
    return MSR_OK;
}

int msr_order_tokens(const void *ids, int32_t ids_i64, int64_t tokens, int32_t k, int32_t experts, int32_t *offsets,
                     int32_t *position, int32_t *source, void *workspace, size_t workspace_bytes, msr_stream_t stream) {
    size_t need = 0;
    if (msr_order_workspace_bytes(tokens, k, experts, &need)) {
        set_error("msr_order_tokens: need tokens * k < 2^30 and 1 to %d experts (got %lld x %d, %d experts)", MSR_EXPERTS_MAX,
                  (long long)tokens, (int)k, (int)experts);
        return MSR_ERR_ARG;
    }
    const int64_t n = tokens * k;
    if (!offsets || (n > 0 && (!ids || !position || !source))) { set_error("msr_order_tokens: a pointer is NULL"); return MSR_ERR_ARG; }
    if (!aligned(ids, ids_i64 ? 8 : 4) || !aligned(offsets, 4) || !aligned(position, 4) || !aligned(source, 4) || !aligned(workspace, 4)) {
        set_error("msr_order_tokens: operands must be aligned to their types");
        return MSR_ERR_ALIGN;
    }
    if (need && (!workspace || workspace_bytes < need)) {
        set_error("msr_order_tokens: workspace of %zu bytes is smaller than the %zu required", workspace_bytes, need);
        return MSR_ERR_WORKSPACE;
    }
    const void *ops[5] = {ids, offsets, position, source, workspace};
    const size_t len[5] = {(size_t)n * (ids_i64 ? 8 : 4), ((size_t)experts + 1) * 4, (size_t)n * 4, (size_t)n * 4, need};
    for (int i = 0; i < 5; ++i)
        for (int j = i + 1; j < 5; ++j)
            if (touch(ops[i], len[i], ops[j], len[j])) {
                set_error("msr_order_tokens: operands %d and %d overlap", i, j);
                return MSR_ERR_OVERLAP;
            }
    const OrderPlan p = order_plan(n);
    OrderArgs a{ids, offsets, position, source, need ? static_cast<int32_t *>(workspace) : nullptr, n, experts, ids_i64 != 0, p.chunk};
    hipStream_t s = (hipStream_t)stream;
    if (need) {
        hipLaunchKernelGGL(count_kernel, dim3(p.wgs), dim3(ORD_THREADS), 0, s, a);
        const int rc = check_launch("count_kernel");
        if (rc) return rc;
    }
    hipLaunchKernelGGL(place_kernel, dim3(p.wgs), dim3(ORD_THREADS), ORD_WAVES * (experts + 1) * 4, s, a);
    return check_launch("place_kernel");
}

int msr_dispatch(const void *x, int64_t ldx, void *rows, const int32_t *position, const int32_t *offsets,
                 int32_t experts, int64_t tokens, int32_t k, int64_t d, int32_t elem, msr_stream_t stream) {
    MoveArgs a{};
    a.tok = x; a.ldtok = ldx; a.out = rows; a.position = position; a.offsets = offsets;
    a.tokens = tokens; a.d = d; a.k = k; a.experts = experts;
    int rc = move_check("msr_dispatch", a, elem, MSR_F32);
    if (rc) return rc;
    a.n = tokens * k;
    if (a.n == 0 || d == 0) return MSR_OK;
    const size_t es = elem == MSR_BF16 ? 2 : 4;
    if (!x || !rows || !position || !offsets || ldx < d || experts < 0) { set_error("msr_dispatch: bad arguments"); return MSR_ERR_ARG; }
    if (!aligned(x, es) || !aligned(rows, es)) { set_error("msr_dispatch: operands must be aligned to their types"); return MSR_ERR_ALIGN; }
    const size_t rb = (size_t)a.n * (size_t)d * es;
    if (touch(rows, rb, x, ((size_t)(tokens - 1) * (size_t)ldx + (size_t)d) * es) || touch(rows, rb, position, (size_t)a.n * 4) ||
        touch(rows, rb, offsets, ((size_t)experts + 1) * 4)) {
        set_error("msr_dispatch: rows overlap an input");
        return MSR_ERR_OVERLAP;
    }
    const bool vec = move_vec(d, ldx, es, x, rows, nullptr);
    const int packs = move_plan(a, elem, vec);
    MOVE_LAUNCH(dispatch_kernel);
    return check_launch("dispatch_kernel");
}

int msr_dispatch_grad(const void *drows, void *dx, const int32_t *position, int64_t tokens, int32_t k, int64_t d,
                      int32_t elem, msr_stream_t stream) {
    MoveArgs a{};
    a.rows = drows; a.out = dx; a.position = position; a.tokens = tokens; a.d = d; a.k = k;
    int rc = move_check("msr_dispatch_grad", a, elem, MSR_F32);
    if (rc) return rc;
    a.n = tokens * k;
    if (a.n == 0 || d == 0) return MSR_OK;
    const size_t es = elem == MSR_BF16 ? 2 : 4;
    if (!drows || !dx || !position) { set_error("msr_dispatch_grad: a pointer is NULL"); return MSR_ERR_ARG; }
    if (!aligned(drows, es) || !aligned(dx, es)) { set_error("msr_dispatch_grad: operands must be aligned to their types"); return MSR_ERR_ALIGN; }
    const size_t rb = (size_t)a.n * (size_t)d * es, tb = (size_t)tokens * (size_t)d * es;
    if (touch(dx, tb, drows, rb) || touch(dx, tb, position, (size_t)a.n * 4)) { set_error("msr_dispatch_grad: dx overlaps an input"); return MSR_ERR_OVERLAP; }
    const bool vec = move_vec(d, d, es, drows, dx, nullptr);
    const int packs = move_plan(a, elem, vec);
    MOVE_LAUNCH(combine_kernel, false);
    return check_launch("combine_kernel");
}

int msr_combine(const void *rows, const void *w, void *y, const int32_t *position, int64_t tokens, int32_t k, int64_t d,
                int32_t elem, int32_t welem, msr_stream_t stream) {
    MoveArgs a{};
    a.rows = rows; a.w = w; a.out = y; a.position = position; a.tokens = tokens; a.d = d; a.k = k; a.w32 = welem == MSR_F32;
    int rc = move_check("msr_combine", a, elem, welem);
    if (rc) return rc;
    a.n = tokens * k;
    if (a.n == 0 || d == 0) return MSR_OK;
    const size_t es = elem == MSR_BF16 ? 2 : 4, ws = welem == MSR_BF16 ? 2 : 4;
    if (!rows || !w || !y || !position) { set_error("msr_combine: a pointer is NULL"); return MSR_ERR_ARG; }
    if (!aligned(rows, es) || !aligned(y, es) || !aligned(w, ws)) { set_error("msr_combine: operands must be aligned to their types"); return MSR_ERR_ALIGN; }
    const size_t rb = (size_t)a.n * (size_t)d * es, tb = (size_t)tokens * (size_t)d * es;
    if (touch(y, tb, rows, rb) || touch(y, tb, w, (size_t)a.n * ws) || touch(y, tb, position, (size_t)a.n * 4)) {
        set_error("msr_combine: y overlaps an input");
        return MSR_ERR_OVERLAP;
    }
    const bool vec = move_vec(d, d, es, rows, y, nullptr);
    const int packs = move_plan(a, elem, vec);
    MOVE_LAUNCH(combine_kernel, true);
    return check_launch("combine_kernel");
}

int msr_combine_grad(const void *dy, int64_t lddy, const void *rows, const void *w, void *drows, void *dw,
                     const int32_t *position, const int32_t *offsets, int32_t experts, int64_t tokens, int32_t k,
                     int64_t d, int32_t elem, int32_t welem, msr_stream_t stream) {
    MoveArgs a{};
    a.tok = dy; a.ldtok = lddy; a.rows = rows; a.w = w; a.out = drows; a.dw = dw; a.position = position; a.offsets = offsets;
    a.tokens = tokens; a.d = d; a.k = k; a.experts = experts; a.w32 = welem == MSR_F32;
    int rc = move_check("msr_combine_grad", a, elem, welem);
    if (rc) return rc;
    a.n = tokens * k;
    if (a.n == 0 || (!drows && !dw)) return MSR_OK;
    const size_t es = elem == MSR_BF16 ? 2 : 4, ws = welem == MSR_BF16 ? 2 : 4;
    if ((d > 0 && !dy) || (d > 0 && dw && !rows) || !w || !position || (drows && !offsets) || lddy < d || experts < 0) {
        set_error("msr_combine_grad: bad arguments");
        return MSR_ERR_ARG;
    }
    if (!aligned(dy, es) || !aligned(rows, es) || !aligned(drows, es) || !aligned(w, ws) || !aligned(dw, ws)) {
        set_error("msr_combine_grad: operands must be aligned to their types");
        return MSR_ERR_ALIGN;
    }
    const size_t rb = (size_t)a.n * (size_t)d * es, tb = ((size_t)(tokens - 1) * (size_t)lddy + (size_t)d) * es;
    const size_t wb = (size_t)a.n * ws, pb = (size_t)a.n * 4, ob = ((size_t)experts + 1) * 4;
    const void *in[5] = {dy, rows, w, position, offsets};
    const size_t ib[5] = {tb, rb, wb, pb, ob};
    bool bad = touch(drows, rb, dw, wb);
    for (int i = 0; i < 5; ++i) bad = bad || touch(drows, rb, in[i], ib[i]) || touch(dw, wb, in[i], ib[i]);
    if (bad) { set_error("msr_combine_grad: an output overlaps another operand"); return MSR_ERR_OVERLAP; }
    const bool vec = move_vec(d, lddy, es, dy, rows, drows);
    const int packs = move_plan(a, elem, vec);
    if (a.share) MOVE_LAUNCH(combine_grad_kernel, true);
    else MOVE_LAUNCH(combine_grad_kernel, false);
    return check_launch("combine_grad_kernel");
}

}  // extern "C"
