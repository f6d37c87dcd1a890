// Layer norm over the last dimension, rows x [rows][d]:
//     mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r,   y = h w + b
//     q = dy w,   dx = r (q - mean(q) - h mean(q h)),   dw = sum_n dy h,   db = sum_n dy
// HBM bounds both passes (x and y; x, dy and dx).  A row is held in the registers of one wave or of the four of a
// work-group, read once: a mean first, then the sums of what is left of it and of its squares, so that a mean far from zero costs no
// digits: with z = x - (that mean), mean += mean(z) and the variance is mean(z^2) - mean(z)^2.  The
// backward pass adds dw and db up in registers over the rows that a work-group takes, in order; the
// work-groups' sums, in fp32, are added by a second kernel, in order.
#include "rows.hpp"
#include "../../include/muon_sr_amd.h"

namespace msr {

// dx goes past the caches, y does not (32768 rows of 4096: gradient 157 us with cached stores, 145 so; forward 113 and 116, and
// the next product finds y).
struct NormArgs {
    const void *x, *dy, *w, *b;
    int64_t ldx, lddy, rows, d;
    void *y;                     // y, or dx
    float *mean, *rstd;          // [rows]
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

// Sums over the lanes that hold a row: a wave (W = 1), or the work-group's four.
template <int W>
struct RowSum {
    float2 (*lds)[4];            // [2][4], used in turn
    int turn = 0;
    __device__ __forceinline__ float2 of(float x, float y) {
        float2 v = wave_sum2(x, y);
        if constexpr (W > 1) {
            float2 *const at = lds[turn];
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
            __syncthreads();
            v = make_float2(((at[0].x + at[1].x) + at[2].x) + at[3].x, ((at[0].y + at[1].y) + at[2].y) + at[3].y);
        }
        return v;
    }
};

// U cells per lane; W waves per row.
template <typename T, int U, int W>
__global__ __launch_bounds__(256) void norm_kernel(NormArgs a) {
    using C = Cells<T>;
    constexpr int N = C::N, L = 64 * W;
    __shared__ float2 lds[2][4];
    RowSum<W> sums{lds};
    const int lane = threadIdx.x % L, sub = threadIdx.x / L;
    const float d = (float)a.d;
    float w[U][N], b[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        vector_cells<N>(a.w, a.w32, (int64_t)(u * L + lane) * N, a.d, 1.0f, w[u]);
        vector_cells<N>(a.b, a.w32, (int64_t)(u * L + lane) * N, a.d, 0.0f, b[u]);
    }
    const int64_t step = (int64_t)gridDim.x * (4 / W);
    int64_t n = (int64_t)blockIdx.x * (4 / W) + sub;
    C next[U];
    auto fetch = [&](int64_t r) __attribute__((always_inline)) {
        if (r >= a.rows) return;
#pragma unroll
        for (int u = 0; u < U; ++u) next[u].load(static_cast<const T *>(a.x) + r * a.ldx, (int64_t)(u * L + lane) * N, a.d);
    };
    for (fetch(n); n < a.rows; n += step) {
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
        const float c = left.x / d, r = 1.0f / sqrtf(fmaxf(left.y / d - c * c, 0.0f) + a.eps);
        mean += c;
        if (lane == 0) {
            a.mean[n] = mean;
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

template <typename T, int U, int W>
__global__ __launch_bounds__(256) void norm_grad_kernel(NormArgs a) {
    using C = Cells<T>;
    constexpr int N = C::N, L = 64 * W;
    __shared__ float2 lds[2][4];
    RowSum<W> sums{lds};
    const int lane = threadIdx.x % L, sub = threadIdx.x / L;
    const float inv = 1.0f / (float)a.d;
    float w[U][N], dw[U][N], db[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        vector_cells<N>(a.w, a.w32, (int64_t)(u * L + lane) * N, a.d, 1.0f, w[u]);
#pragma unroll
        for (int e = 0; e < N; ++e) dw[u][e] = db[u][e] = 0.0f;
    }
    const int64_t step = (int64_t)gridDim.x * (4 / W);
    int64_t n = (int64_t)blockIdx.x * (4 / W) + sub;
    C vx[U], vy[U];
    float next_mean = 0.0f, next_r = 0.0f;
    auto fetch = [&](int64_t i) __attribute__((always_inline)) {
        if (i >= a.rows) return;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vx[u].load(static_cast<const T *>(a.x) + i * a.ldx, (int64_t)(u * L + lane) * N, a.d);
            vy[u].load(static_cast<const T *>(a.dy) + i * a.lddy, (int64_t)(u * L + lane) * N, a.d);
        }
        next_mean = a.mean[i];
        next_r = a.rstd[i];
    };
    for (fetch(n); n < a.rows; n += step) {
        const float mean = next_mean, r = next_r;
        float h[U][N], q[U][N], sq = 0.0f, sqh = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vx[u].get(h[u]);
            vy[u].get(q[u]);
#pragma unroll
            for (int e = 0; e < N; ++e) {       // (beyond the row dy is 0, and so is what it is multiplied into)
                h[u][e] = (h[u][e] - mean) * r;
                dw[u][e] = __builtin_fmaf(q[u][e], h[u][e], dw[u][e]);
                db[u][e] += q[u][e];
                q[u][e] *= w[u][e];
                sq += q[u][e];
                sqh = __builtin_fmaf(q[u][e], h[u][e], sqh);
            }
        }
        fetch(n + step);
        const float2 m = sums.of(sq, sqh);
        const float mq = m.x * inv, mh = m.y * inv;
        if (a.y) {
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
    if constexpr (W > 1) {
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
        // the four waves' sums, a cell at a time
        __shared__ float both[4][2][64 * N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < N; ++e) {
                both[sub][0][lane * N + e] = dw[u][e];
                both[sub][1][lane * N + e] = db[u][e];
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 2 * 64 * N; i += 256) {
                const int k = i / (64 * N), c = i % (64 * N);
                if ((int64_t)u * L * N + c >= a.d) continue;
                to[k * a.d + (int64_t)u * L * N + c] = ((both[0][k][c] + both[1][k][c]) + both[2][k][c]) + both[3][k][c];
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
    RowSum<4> sums{lds};
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
            a.mean[n] = mean + left;
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
    RowSum<4> sums{lds};
    const float inv = 1.0f / (float)a.d;
    float *const to = a.parts ? a.parts + (int64_t)blockIdx.x * 2 * a.d : nullptr;
    bool first = true;
    for (int64_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
        const float mean = a.mean[n], r = a.rstd[n];
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
                    h[e] = (h[e] - mean) * r;
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

// Cells per lane and waves per row; 0 cells: the row does not fit in registers.
struct NormPlan {
    int u, w, groups;            // groups: work-groups of the backward pass
};
static NormPlan norm_plan(int64_t rows, int64_t d, int32_t elem) {
    NormPlan p{};
    const int64_t cells = (d + (elem == MSR_BF16 ? 7 : 3)) / (elem == MSR_BF16 ? 8 : 4);
    p.w = cells <= 64 * 2 ? 1 : 4;
    const int64_t per = (cells + 64 * p.w - 1) / (64 * p.w);
    p.u = per <= 1 ? 1 : per <= 2 ? 2 : per <= 4 ? 4 : 0;
    if (p.u == 0) p.w = 4;
    const int64_t at_once = 4 / p.w;
    p.groups = (int)std::min<int64_t>(std::max<int64_t>((rows + at_once - 1) / at_once, 1), 512);
    return p;
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
static void norm_launch(const NormArgs &a, const NormPlan &p, hipStream_t s) {
    const dim3 grid(grid_for(a.rows, 4 / p.w, 256 * 8));
    auto go = [&](auto u, auto w) { hipLaunchKernelGGL((norm_kernel<T, decltype(u)::value, decltype(w)::value>), grid, dim3(256), 0, s, a); };
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    if (p.u == 0) hipLaunchKernelGGL(norm_long_kernel<T>, dim3(grid_for(a.rows, 1, 256 * 8)), dim3(256), 0, s, a);
    else if (p.w == 1) p.u == 1 ? go(I1{}, I1{}) : go(I2{}, I1{});
    else p.u == 1 ? go(I1{}, I4{}) : p.u == 2 ? go(I2{}, I4{}) : go(I4{}, I4{});
}
template <typename T>
static void norm_grad_launch(const NormArgs &a, const NormPlan &p, hipStream_t s) {
    auto go = [&](auto u, auto w) { hipLaunchKernelGGL((norm_grad_kernel<T, decltype(u)::value, decltype(w)::value>), dim3(p.groups), dim3(256), 0, s, a); };
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    if (p.u == 0) hipLaunchKernelGGL(norm_long_grad_kernel<T>, dim3(p.groups), dim3(256), 0, s, a);
    else if (p.w == 1) p.u == 1 ? go(I1{}, I1{}) : go(I2{}, I1{});
    else p.u == 1 ? go(I1{}, I4{}) : p.u == 2 ? go(I2{}, I4{}) : go(I4{}, I4{});
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
    const Range r[6] = {{y, n * (size_t)d * es}, {mean, 4 * n}, {rstd, 4 * n}, {x, rows_bytes(rows, ldx, d, es)}, {w, (size_t)d * ws}, {b, (size_t)d * ws}};
    rc = ranges_apart(name, r, 6, 3);
    if (rc) return rc;
    NormArgs a{};
    a.x = x; a.ldx = ldx; a.w = w; a.b = b; a.eps = eps; a.rows = rows; a.d = d; a.y = y; a.mean = mean; a.rstd = rstd; a.w32 = welem == MSR_F32;
    const NormPlan p = norm_plan(rows, d, elem);
    if (elem == MSR_BF16) norm_launch<uint16_t>(a, p, (hipStream_t)stream);
    else norm_launch<float>(a, p, (hipStream_t)stream);
    return check_launch("norm_kernel");
}

int msr_layer_norm_workspace_bytes(int64_t rows, int64_t d, int32_t elem, size_t *bytes) {
    const int rc = norm_check("msr_layer_norm_workspace_bytes", rows, d, elem, MSR_F32);
    if (rc) return rc;
    if (!bytes) { set_error("msr_layer_norm_workspace_bytes: a pointer is NULL"); return MSR_ERR_ARG; }
    *bytes = (size_t)norm_plan(rows, d, elem).groups * 2 * (size_t)d * 4;
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
    const NormPlan p = norm_plan(rows, d, elem);
    const size_t need = (size_t)p.groups * 2 * (size_t)d * 4, n = (size_t)rows;
    if ((dw || db) && (!workspace || workspace_bytes < need)) {
        set_error("%s: workspace of %zu bytes is smaller than the %zu required", name, workspace_bytes, need);
        return MSR_ERR_WORKSPACE;
    }
    const Range r[9] = {{dx, n * (size_t)d * es}, {dw, (size_t)d * ws}, {db, (size_t)d * ws}, {workspace, dw || db ? need : 0},
                        {dy, rows_bytes(rows, lddy, d, es)}, {x, rows_bytes(rows, ldx, d, es)}, {w, (size_t)d * ws}, {mean, 4 * n}, {rstd, 4 * n}};
    rc = ranges_apart(name, r, 9, 4);
    if (rc) return rc;
    hipStream_t s = (hipStream_t)stream;
    NormArgs a{};
    a.x = x; a.ldx = ldx; a.dy = dy; a.lddy = lddy; a.w = w; a.rows = rows; a.d = d; a.y = dx; a.w32 = welem == MSR_F32;
    a.mean = const_cast<float *>(mean); a.rstd = const_cast<float *>(rstd);
    a.parts = dw || db ? static_cast<float *>(workspace) : nullptr;
    if (rows > 0) {
        if (elem == MSR_BF16) norm_grad_launch<uint16_t>(a, p, s);
        else norm_grad_launch<float>(a, p, s);
        if ((rc = check_launch("norm_grad_kernel"))) return rc;
    }
    if (!a.parts) return MSR_OK;
    const dim3 grid((unsigned)((d + 31) / 32));
    const int groups = rows > 0 ? p.groups : 0;
    if (welem == MSR_BF16) hipLaunchKernelGGL(norm_join_kernel<uint16_t>, grid, dim3(256), 0, s, a.parts, groups, d, static_cast<uint16_t *>(dw), static_cast<uint16_t *>(db));
    else hipLaunchKernelGGL(norm_join_kernel<float>, grid, dim3(256), 0, s, a.parts, groups, d, static_cast<float *>(dw), static_cast<float *>(db));
    return check_launch("norm_join_kernel");
}

}  // extern "C"
