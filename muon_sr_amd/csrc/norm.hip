// Layer norm over the last dimension, rows x [rows][d]:
//     mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r,   y = h w + b
//     q = dy w,   dx = r (q - mean(q) - h mean(q h)),   dw = sum_n dy h,   db = sum_n dy
// HBM bounds both passes (x and y; x, dy and dx).  A row is held in the registers of L lanes, 8 to 64 of a wave or a whole work-group of
// 256 or 1024, read once: a mean m first, then the sums of what is left of it and of its squares, so that a mean far from zero costs no
// digits: with z = x - m and c = mean(z), h = (z - c) r and the variance is mean(z^2) - c^2.  m and c are kept as two numbers for the
// backward pass too: their sum, rounded at the size of the mean, puts every h of a row off by up to half of its ulp times r (fp32 rows of
// 768 around 1000 of deviation 1e-2, against 64 bits: dx off by 9e-5 and dw by 1.9e-3, and by 1e-7 each so).  The backward pass adds dw
// and db up in registers over the rows that a work-group takes, in order; the work-groups' sums, in fp32, are added by a second kernel, in
// order.
#include "rows.hpp"
#include "../../include/muon_sr_amd.h"

namespace msr {

// dx goes past the caches, y does not (32768 rows of 4096: gradient 157 us with cached stores, 145 so; forward 113 and 116, and
// the next product finds y).
struct NormArgs {
    const void *x, *dy, *w, *b;
    int64_t ldx, lddy, rows, d;
    void *y;                     // y, or dx
    float *mean, *rstd;          // [2][rows]: m, c; [rows]
    float *parts;                // [work-groups][2][d]: sums of dy h and of dy
    float eps;
    int32_t w32;                 // w and b are fp32
};

// N elements of w or b from column c on
template <int N>
__device__ __forceinline__ void vector_cells(const void *p, int w32, int64_t c, int64_t d, float other, float (&f)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        f[e] = other;
        if (p && c + e < d) f[e] = w32 ? static_cast<const float *>(p)[c + e] : bf16_to_f32(static_cast<const uint16_t *>(p)[c + e]);
    }
}

// Sums over the L lanes that hold a row.
template <int L>
struct RowSum {
    static constexpr int WAVES = L > 64 ? L / 64 : 1;
    float2 (*lds)[WAVES];        // [2][WAVES], used in turn
    int turn = 0;
    __device__ __forceinline__ float2 of(float x, float y) {
        if constexpr (L < 64) return make_float2(over_group<L>(x, Add{}), over_group<L>(y, Add{}));
        float2 v = wave_sum2(x, y);
        if constexpr (L > 64) {
            float2 *const at = lds[turn];
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
            __syncthreads();
            v = at[0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) v = make_float2(v.x + at[w].x, v.y + at[w].y);
        }
        return v;
    }
};
constexpr int norm_threads(int L) { return L > 256 ? L : 256; }

// U cells per lane, L lanes per row: few lanes to a short row, so that a wave holds up to eight (us, forward and gradient, a wave to a
// row and so: 131072 rows of 64 46 92, 12 16; of 128 47 94, 23 24), 1024 to a long one (rows read as often as they are needed, and so: 8000
// rows of 16384 501 1312, 122 207; 3000 fp32 rows of 16000 144 449, 84 125).
template <typename T, int U, int L>
__global__ __launch_bounds__(norm_threads(L)) void norm_kernel(NormArgs a) {
    using C = Cells<T>;
    constexpr int N = C::N, ROWS = norm_threads(L) / L;
    __shared__ float2 lds[2][RowSum<L>::WAVES];
    RowSum<L> sums{lds};
    const int lane = threadIdx.x % L, sub = threadIdx.x / L;
    const float d = (float)a.d;
    float w[U][N], b[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        vector_cells<N>(a.w, a.w32, (int64_t)(u * L + lane) * N, a.d, 1.0f, w[u]);
        vector_cells<N>(a.b, a.w32, (int64_t)(u * L + lane) * N, a.d, 0.0f, b[u]);
    }
    const int64_t step = (int64_t)gridDim.x * ROWS;
    C next[U];
    auto fetch = [&](int64_t r) __attribute__((always_inline)) {
        if (r >= a.rows) return;
#pragma unroll
        for (int u = 0; u < U; ++u) next[u].load(static_cast<const T *>(a.x) + r * a.ldx, (int64_t)(u * L + lane) * N, a.d);
    };
    int64_t n = (int64_t)blockIdx.x * ROWS + sub;
    fetch(n);
    for (; n - (L < 64 ? sub : 0) < a.rows; n += step) {   // (the same for every lane of a wave: lanes without a row go along)
        float x[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) next[u].get(x[u]);
        fetch(n + step);
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) s += x[u][e];
        float mean = sums.of(s, 0.0f).x / d;
        float z = 0.0f, q = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                x[u][e] = (int64_t)(u * L + lane) * N + e < a.d ? x[u][e] - mean : 0.0f;
                z += x[u][e];
                q = __builtin_fmaf(x[u][e], x[u][e], q);
            }
        const float2 left = sums.of(z, q);
        if (L < 64 && n >= a.rows) continue;
        const float c = left.x / d, r = 1.0f / sqrtf(fmaxf(left.y / d - c * c, 0.0f) + a.eps);
        if (lane == 0) {
            a.mean[n] = mean;
            a.mean[a.rows + n] = c;
            a.rstd[n] = r;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[N];
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = __builtin_fmaf((x[u][e] - c) * r, w[u][e], b[u][e]);
            C v;
            v.set(f);
            v.store(static_cast<T *>(a.y) + n * a.d, (int64_t)(u * L + lane) * N, a.d);
        }
    }
}

template <typename T, int U, int L>
__global__ __launch_bounds__(norm_threads(L)) void norm_grad_kernel(NormArgs a) {
    using C = Cells<T>;
    constexpr int N = C::N, ROWS = norm_threads(L) / L;
    // the next row on its way meanwhile: not where its registers, of 128 that a thread of 1024 has, cost more (us with it and without:
    // 3000 fp32 rows of 16000 236 and 156, bf16 8000 of 16384 223 and 234, fp32 4000 of 8192 69 and 71)
    constexpr bool AHEAD = L <= 256 || sizeof(T) == 2 || U * N <= 8;
    __shared__ float2 lds[2][RowSum<L>::WAVES];
    RowSum<L> sums{lds};
    const int lane = threadIdx.x % L, sub = threadIdx.x / L;
    const float inv = 1.0f / (float)a.d;
    float w[U][N], dw[U][N], db[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        vector_cells<N>(a.w, a.w32, (int64_t)(u * L + lane) * N, a.d, 1.0f, w[u]);
#pragma unroll
        for (int e = 0; e < N; ++e) dw[u][e] = db[u][e] = 0.0f;
    }
    const int64_t step = (int64_t)gridDim.x * ROWS;
    C vx[U], vy[U];
    float next_mean = 0.0f, next_c = 0.0f, next_r = 0.0f;
    auto fetch = [&](int64_t i) __attribute__((always_inline)) {
        if constexpr (L < 64) {
#pragma unroll
            for (int u = 0; u < U; ++u) vx[u].v = vy[u].v = Bytes16{};
            next_mean = next_c = next_r = 0.0f;
        }
        if (i >= a.rows) return;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vx[u].load(static_cast<const T *>(a.x) + i * a.ldx, (int64_t)(u * L + lane) * N, a.d);
            vy[u].load(static_cast<const T *>(a.dy) + i * a.lddy, (int64_t)(u * L + lane) * N, a.d);
        }
        next_mean = a.mean[i];
        next_c = a.mean[a.rows + i];
        next_r = a.rstd[i];
    };
    int64_t n = (int64_t)blockIdx.x * ROWS + sub;
    if (AHEAD) fetch(n);
    for (; n - (L < 64 ? sub : 0) < a.rows; n += step) {
        if (!AHEAD) fetch(n);
        const float mean = next_mean, c = next_c, r = next_r;
        float h[U][N], q[U][N], sq = 0.0f, sqh = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vx[u].get(h[u]);
            vy[u].get(q[u]);
#pragma unroll
            for (int e = 0; e < N; ++e) {       // (beyond the row, and without one, dy is 0, and so is what it is multiplied into)
                h[u][e] = ((h[u][e] - mean) - c) * r;
                dw[u][e] = __builtin_fmaf(q[u][e], h[u][e], dw[u][e]);
                db[u][e] += q[u][e];
                q[u][e] *= w[u][e];
                sq += q[u][e];
                sqh = __builtin_fmaf(q[u][e], h[u][e], sqh);
            }
        }
        if (AHEAD) fetch(n + step);
        const float2 m = sums.of(sq, sqh);
        const float mq = m.x * inv, mh = m.y * inv;
        if (a.y && (L >= 64 || n < a.rows)) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[N];
#pragma unroll
                for (int e = 0; e < N; ++e) f[e] = r * (q[u][e] - __builtin_fmaf(h[u][e], mh, mq));
                C v;
                v.set(f);
                v.template store<true>(static_cast<T *>(a.y) + n * a.d, (int64_t)(u * L + lane) * N, a.d);
            }
        }
    }
    if (!a.parts) return;
    float *const to = a.parts + (int64_t)blockIdx.x * 2 * a.d;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int64_t c = (int64_t)(u * L + lane) * N + e;
                if (c >= a.d) continue;
                to[c] = dw[u][e];
                to[a.d + c] = db[u][e];
            }
    } else {
        // the rows' sums, a cell of each lane at a time
        __shared__ float both[ROWS][2][L * N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < N; ++e) {
                both[sub][0][lane * N + e] = dw[u][e];
                both[sub][1][lane * N + e] = db[u][e];
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 2 * L * N; i += 256) {
                const int k = i / (L * N), c = i % (L * N);
                if ((int64_t)u * L * N + c >= a.d) continue;
                float s = both[0][k][c];
#pragma unroll
                for (int g = 1; g < ROWS; ++g) s += both[g][k][c];
                to[k * a.d + (int64_t)u * L * N + c] = s;
            }
        }
    }
}

// Rows too long for registers: a work-group per row reads it as often as it needs it (from L2 after the first time).
template <typename T>
__global__ __launch_bounds__(256) void norm_long_kernel(NormArgs a) {
    using C = Cells<T>;
    constexpr int N = C::N;
    __shared__ float2 lds[2][4];
    RowSum<256> sums{lds};
    const float d = (float)a.d;
    for (int64_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
        const T *const row = static_cast<const T *>(a.x) + n * a.ldx;
        float mean = 0.0f, r = 0.0f, left = 0.0f;     // left: the mean of x - mean
        for (int pass = 0; pass < 2; ++pass) {
            float s = 0.0f, q = 0.0f;
            for (int64_t c = (int64_t)threadIdx.x * N; c < a.d; c += 256 * N) {
                C v;
                float f[N];
                v.load(row, c, a.d);
                v.get(f);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    if (c + e >= a.d) continue;
                    const float x = f[e] - mean;
                    s += x;
                    q = __builtin_fmaf(x, x, q);
                }
            }
            const float2 sum = sums.of(s, q);
            if (pass) left = sum.x / d;
            else mean = sum.x / d;
            r = 1.0f / sqrtf(fmaxf(sum.y / d - left * left, 0.0f) + a.eps);
        }
        if (threadIdx.x == 0) {
            a.mean[n] = mean;
            a.mean[a.rows + n] = left;
            a.rstd[n] = r;
        }
        for (int64_t c = (int64_t)threadIdx.x * N; c < a.d; c += 256 * N) {
            C v;
            float f[N], w[N], b[N];
            v.load(row, c, a.d);
            v.get(f);
            vector_cells<N>(a.w, a.w32, c, a.d, 1.0f, w);
            vector_cells<N>(a.b, a.w32, c, a.d, 0.0f, b);
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = __builtin_fmaf(((f[e] - mean) - left) * r, w[e], b[e]);
            v.set(f);
            v.store(static_cast<T *>(a.y) + n * a.d, c, a.d);
        }
    }
}

// Their gradient; the work-group's sums of dw and db stay in its part of the workspace between its rows.
template <typename T>
__global__ __launch_bounds__(256) void norm_long_grad_kernel(NormArgs a) {
    using C = Cells<T>;
    constexpr int N = C::N;
    __shared__ float2 lds[2][4];
    RowSum<256> sums{lds};
    const float inv = 1.0f / (float)a.d;
    float *const to = a.parts ? a.parts + (int64_t)blockIdx.x * 2 * a.d : nullptr;
    bool first = true;
    for (int64_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
        const float mean = a.mean[n], left = a.mean[a.rows + n], r = a.rstd[n];
        float2 m = make_float2(0.0f, 0.0f);
        for (int pass = 0; pass < 2; ++pass) {
            float sq = 0.0f, sqh = 0.0f;
            for (int64_t c = (int64_t)threadIdx.x * N; c < a.d; c += 256 * N) {
                C vx, vy;
                float h[N], q[N], w[N];
                vx.load(static_cast<const T *>(a.x) + n * a.ldx, c, a.d);
                vy.load(static_cast<const T *>(a.dy) + n * a.lddy, c, a.d);
                vx.get(h);
                vy.get(q);
                vector_cells<N>(a.w, a.w32, c, a.d, 1.0f, w);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    h[e] = ((h[e] - mean) - left) * r;
                    if (!pass && to && c + e < a.d) {
                        to[c + e] = __builtin_fmaf(q[e], h[e], first ? 0.0f : to[c + e]);
                        to[a.d + c + e] = q[e] + (first ? 0.0f : to[a.d + c + e]);
                    }
                    q[e] *= w[e];
                    sq += q[e];
                    sqh = __builtin_fmaf(q[e], h[e], sqh);
                    q[e] = r * (q[e] - __builtin_fmaf(h[e], m.y, m.x));
                }
                if (pass && a.y) {
                    vx.set(q);
                    vx.store(static_cast<T *>(a.y) + n * a.d, c, a.d);
                }
            }
            if (pass) break;
            m = sums.of(sq, sqh);
            m = make_float2(m.x * inv, m.y * inv);
        }
        first = false;
    }
}

// dw and db from the work-groups' sums: 32 columns and 8 shares of the work-groups per work-group
template <typename TW>
__global__ __launch_bounds__(256) void norm_join_kernel(const float *parts, int groups, int64_t d, TW *dw, TW *db) {
    __shared__ float2 share[8][32];
    const int col = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + col;
    float2 s = make_float2(0.0f, 0.0f);
    if (c < d) {
#pragma unroll 8
        for (int g = k; g < groups; g += 8) {
            s.x += parts[(int64_t)g * 2 * d + c];
            s.y += parts[((int64_t)g * 2 + 1) * d + c];
        }
    }
    share[k][col] = s;
    __syncthreads();
    if (k > 0 || c >= d) return;
    for (int i = 1; i < 8; ++i) {
        s.x += share[i][col].x;
        s.y += share[i][col].y;
    }
    auto put = [&](TW *to, float v) __attribute__((always_inline)) {
        if constexpr (sizeof(TW) == 2) to[c] = (TW)rne_bf16(v);
        else to[c] = v;
    };
    if (dw) put(dw, s.x);
    if (db) put(db, s.y);
}

// f(cells per lane, lanes per row) of a row of d elements; false, and f is not called, for one that does not fit in registers.
template <typename T, typename F>
static bool norm_shape(int64_t d, F &&f) {
    auto is = [&](auto u, auto l) {
        if (d > (int64_t)decltype(u)::value * decltype(l)::value * Cells<T>::N) return false;
        f(u, l);
        return true;
    };
    using std::integral_constant;
    using U1 = integral_constant<int, 1>;
    using U2 = integral_constant<int, 2>;
    using U4 = integral_constant<int, 4>;
    if (is(U1{}, integral_constant<int, 8>{}) || is(U1{}, integral_constant<int, 16>{}) || is(U1{}, integral_constant<int, 32>{}) ||
        is(U1{}, integral_constant<int, 64>{}) || is(U2{}, integral_constant<int, 64>{}) || is(U1{}, integral_constant<int, 256>{}) ||
        is(U2{}, integral_constant<int, 256>{}) || is(U4{}, integral_constant<int, 256>{}) || is(U2{}, integral_constant<int, 1024>{}))
        return true;
    if constexpr (sizeof(T) == 4) return is(U4{}, integral_constant<int, 1024>{});
    return false;
}
// Work-groups of the backward pass, each of which leaves sums of dw and db: two of 256 threads per CU, or one of 1024.  Four, where their
// registers allow it, for rows that leave lanes without a cell, if each has rows enough for its sums to be few (us with two and four:
// 100000 rows of 448 70 and 54, of 512 53 and 60; 32768 of 1400 90 and 66, of 2048 77 and 82; 4096 of 384 12 and 18).
static int norm_groups(int64_t rows, int64_t d, int32_t elem) {
    int64_t at_once = 1, most = 512;
    const int n = elem == MSR_BF16 ? 8 : 4;
    auto of = [&](auto u, auto l) {
        constexpr int L = decltype(l)::value;
        at_once = norm_threads(L) / L;
        if (L > 256) most = 256;
        if (L >= 32 && L <= 256 && decltype(u)::value * n <= 8 && d < L * decltype(u)::value * n && rows >= 8 * 1024 * at_once) most = 1024;
    };
    if (elem == MSR_BF16) norm_shape<uint16_t>(d, of);
    else norm_shape<float>(d, of);
    return (int)std::min<int64_t>(std::max<int64_t>((rows + at_once - 1) / at_once, 1), most);
}

static int norm_check(const char *name, int64_t rows, int64_t d, int32_t elem, int32_t welem) {
    if (rows < 0 || rows >= (int64_t(1) << 40) || d < 0 || d > (1 << 24) || (elem != MSR_BF16 && elem != MSR_F32) || (welem != MSR_BF16 && welem != MSR_F32)) {
        set_error("%s: need fewer than 2^40 rows of at most 2^24 elements, bf16 or fp32 (got %lld x %lld, types %d and %d)", name, (long long)rows,
                  (long long)d, (int)elem, (int)welem);
        return MSR_ERR_ARG;
    }
    return MSR_OK;
}

template <typename T>
static void norm_launch(const NormArgs &a, hipStream_t s) {
    const bool held = norm_shape<T>(a.d, [&](auto u, auto l) {
        constexpr int L = decltype(l)::value, TH = norm_threads(L);
        hipLaunchKernelGGL((norm_kernel<T, decltype(u)::value, L>), dim3(grid_for(a.rows, TH / L, 256 * 2048 / TH)), dim3(TH), 0, s, a);
    });
    if (!held) hipLaunchKernelGGL(norm_long_kernel<T>, dim3(grid_for(a.rows, 1, 256 * 8)), dim3(256), 0, s, a);
}
template <typename T>
static void norm_grad_launch(const NormArgs &a, int groups, hipStream_t s) {
    const bool held = norm_shape<T>(a.d, [&](auto u, auto l) {
        constexpr int L = decltype(l)::value;
        hipLaunchKernelGGL((norm_grad_kernel<T, decltype(u)::value, L>), dim3(groups), dim3(norm_threads(L)), 0, s, a);
    });
    if (!held) hipLaunchKernelGGL(norm_long_grad_kernel<T>, dim3(groups), dim3(256), 0, s, a);
}

}  // namespace msr

using namespace msr;

extern "C" {

int msr_layer_norm(const void *x, int64_t ldx, const void *w, const void *b, float eps, int64_t rows, int64_t d, void *y, float *mean,
                   float *rstd, int32_t elem, int32_t welem, msr_stream_t stream) {
    const char *const name = "msr_layer_norm";
    int rc = norm_check(name, rows, d, elem, welem);
    if (rc || rows == 0 || d == 0) return rc;
    if (!x || !y || !mean || !rstd || ldx < d) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
    const size_t es = elem_bytes(elem), ws = elem_bytes(welem);
    if (!aligned(x, es) || !aligned(y, es) || !aligned(w, ws) || !aligned(b, ws) || !aligned(mean, 4) || !aligned(rstd, 4)) {
        set_error("%s: operands must be aligned to their types", name);
        return MSR_ERR_ALIGN;
    }
    const size_t n = (size_t)rows;
    const Range r[6] = {{y, n * (size_t)d * es}, {mean, 8 * n}, {rstd, 4 * n}, {x, rows_bytes(rows, ldx, d, es)}, {w, (size_t)d * ws}, {b, (size_t)d * ws}};
    rc = ranges_apart(name, r, 6, 3);
    if (rc) return rc;
    NormArgs a{};
    a.x = x; a.ldx = ldx; a.w = w; a.b = b; a.eps = eps; a.rows = rows; a.d = d; a.y = y; a.mean = mean; a.rstd = rstd; a.w32 = welem == MSR_F32;
    if (elem == MSR_BF16) norm_launch<uint16_t>(a, (hipStream_t)stream);
    else norm_launch<float>(a, (hipStream_t)stream);
    return check_launch("norm_kernel");
}

int msr_layer_norm_workspace_bytes(int64_t rows, int64_t d, int32_t elem, size_t *bytes) {
    const int rc = norm_check("msr_layer_norm_workspace_bytes", rows, d, elem, MSR_F32);
    if (rc) return rc;
    if (!bytes) { set_error("msr_layer_norm_workspace_bytes: a pointer is NULL"); return MSR_ERR_ARG; }
    *bytes = (size_t)norm_groups(rows, d, elem) * 2 * (size_t)d * 4;
    return MSR_OK;
}

int msr_layer_norm_grad(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *w, const float *mean, const float *rstd,
                        int64_t rows, int64_t d, void *dx, void *dw, void *db, int32_t elem, int32_t welem, void *workspace,
                        size_t workspace_bytes, msr_stream_t stream) {
    const char *const name = "msr_layer_norm_grad";
    int rc = norm_check(name, rows, d, elem, welem);
    if (rc || d == 0 || (!dx && !dw && !db)) return rc;
    if ((rows > 0 && (!dy || !x || !mean || !rstd)) || lddy < d || ldx < d) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
    const size_t es = elem_bytes(elem), ws = elem_bytes(welem);
    if (!aligned(dy, es) || !aligned(x, es) || !aligned(dx, es) || !aligned(w, ws) || !aligned(dw, ws) || !aligned(db, ws) || !aligned(mean, 4) ||
        !aligned(rstd, 4) || !aligned(workspace, 4)) {
        set_error("%s: operands must be aligned to their types", name);
        return MSR_ERR_ALIGN;
    }
    const int all = norm_groups(rows, d, elem);
    const size_t need = (size_t)all * 2 * (size_t)d * 4, n = (size_t)rows;
    if ((dw || db) && (!workspace || workspace_bytes < need)) {
        set_error("%s: workspace of %zu bytes is smaller than the %zu required", name, workspace_bytes, need);
        return MSR_ERR_WORKSPACE;
    }
    const Range r[9] = {{dx, n * (size_t)d * es}, {dw, (size_t)d * ws}, {db, (size_t)d * ws}, {workspace, dw || db ? need : 0},
                        {dy, rows_bytes(rows, lddy, d, es)}, {x, rows_bytes(rows, ldx, d, es)}, {w, (size_t)d * ws}, {mean, 8 * n}, {rstd, 4 * n}};
    rc = ranges_apart(name, r, 9, 4);
    if (rc) return rc;
    hipStream_t s = (hipStream_t)stream;
    NormArgs a{};
    a.x = x; a.ldx = ldx; a.dy = dy; a.lddy = lddy; a.w = w; a.rows = rows; a.d = d; a.y = dx; a.w32 = welem == MSR_F32;
    a.mean = const_cast<float *>(mean); a.rstd = const_cast<float *>(rstd);
    a.parts = dw || db ? static_cast<float *>(workspace) : nullptr;
    if (rows > 0) {
        if (elem == MSR_BF16) norm_grad_launch<uint16_t>(a, all, s);
        else norm_grad_launch<float>(a, all, s);
        if ((rc = check_launch("norm_grad_kernel"))) return rc;
    }
    if (!a.parts) return MSR_OK;
    const dim3 grid((unsigned)((d + 31) / 32));
    const int groups = rows > 0 ? all : 0;
    if (welem == MSR_BF16) hipLaunchKernelGGL(norm_join_kernel<uint16_t>, grid, dim3(256), 0, s, a.parts, groups, d, static_cast<uint16_t *>(dw), static_cast<uint16_t *>(db));
    else hipLaunchKernelGGL(norm_join_kernel<float>, grid, dim3(256), 0, s, a.parts, groups, d, static_cast<float *>(dw), static_cast<float *>(db));
    return check_launch("norm_join_kernel");
}

}  // extern "C"
