// The global norm of many gradients, and clipping by it:
//     N = (sum |g|^p)^(1/p),  c = min(1, max_norm / (N + 1e-6)),  out = round(f32(g) c)
//
// The norm needs every element before the first one can be scaled, so two passes over the
// gradients are the least: 2 (or 4) bytes read, then as many read and 2 (or 4) written per
// element.  Both are bound by HBM.  Each pass takes many tensors per launch (a table in the
// kernel arguments):
//   1. norm_kernel   work-groups over tiles of all tensors, one partial sum each, to which the
//                    work-groups of the same number in later launches add theirs, so that a list of
//                    any length has at most CLIP_GRID of them (clipping 9000 tensors of 2^17: 1.90 ms,
//                    with new partial sums from each launch, which every work-group reads, 4.78)
//   2. clip_kernel   every work-group first adds the partial sums itself (8 KiB at most, from L2,
//                    in the same order everywhere), which saves a launch and its gap between the
//                    two passes
// Squares and their sums are held in 64 bits: bf16 and fp32 gradients have the same
// exponents, and the square of 1e20 does not fit 32 bits, nor does that of 1e-23.
#include <math.h>

#include <new>
#include <vector>

#include "common.hpp"
#include "vecio.hpp"
#include "../../include/muon_sr_amd.h"

namespace msr {

constexpr int CLIP_MAXT = 112;                       // tensors of one launch (32 bytes each in the arguments)
constexpr int CLIP_THREADS = 256;
constexpr int CLIP_UNROLL = 4;
constexpr int CLIP_TILE = CLIP_THREADS * 8 * CLIP_UNROLL;   // elements of a work-group's step
constexpr int CLIP_GRID = 256 * 4;                   // work-groups of a launch: 4 on each CU (of 1.3e9 bf16 elements,
                                                     // both passes: 1313 us, 5.9 TB/s; with 8 1403, with 2 1533)
constexpr float CLIP_EPS = 1e-6f;

constexpr uint32_t CLIP_G32 = MSR_CLIP_GRAD_F32, CLIP_O32 = MSR_CLIP_OUT_F32;

struct ClipArgs {
    const void *g[CLIP_MAXT];
    void *out[CLIP_MAXT];
    int64_t n[CLIP_MAXT];
    int32_t start[CLIP_MAXT + 1];                    // first tile of a tensor
    uint8_t flags[CLIP_MAXT];
    int32_t count;
};
static_assert(sizeof(ClipArgs) <= 3600, "kernel arguments");

// One element's part of the sum: |x|, x^2 (exact in 64 bits for any fp32 x), or the bits of |x|,
// whose order as integers is that of the magnitudes with NaN above infinity.
template <int P>
__device__ __forceinline__ void norm_add(double &s, float x) {
    if constexpr (P == MSR_NORM_1) s += fabs((double)x);
    else if constexpr (P == MSR_NORM_2) s = __builtin_fma((double)x, (double)x, s);
    else s = fmax(s, (double)(__float_as_uint(x) & 0x7fffffffu));
}
template <int P>
__device__ __forceinline__ double norm_join(double a, double b) {
    return P == MSR_NORM_INF ? fmax(a, b) : a + b;
}

// The sum of a value of every thread, in every thread (fixed order).
template <int P>
__device__ __forceinline__ double norm_block(double s, double *red) {
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) s = norm_join<P>(s, __shfl_xor(s, w));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = red[0];
#pragma unroll
    for (int w = 1; w < CLIP_THREADS / 64; ++w) s = norm_join<P>(s, red[w]);
    return s;
}

template <int P>
__device__ __forceinline__ float norm_root(double s) {
    if constexpr (P == MSR_NORM_1) return (float)s;
    else if constexpr (P == MSR_NORM_2) return (float)sqrt(s);
    else return __uint_as_float((uint32_t)s);
}

// 8 elements from element o on, of `valid` (<= 8) that exist; the others are 0.  Tensors start where they like: 16
// bytes go in one access at any alignment of the element type, which the hardware allows for global memory.
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(4)));
template <bool F32>
__device__ __forceinline__ void clip_load(const void *g, int64_t o, int valid, float f[8]) {
    if constexpr (F32) {
        const float *p = static_cast<const float *>(g) + o;
        if (valid == 8) {
            const f32x4_any_t x = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any_t *>(p));
            const f32x4_any_t y = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any_t *>(p + 4));
            f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
            f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = j < valid ? p[j] : 0.0f;
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(g) + o;
        if (valid == 8) {
            const u32x4_any_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any_t *>(p));
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            unpack8(w, f);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = j < valid ? bf16_to_f32(p[j]) : 0.0f;
        }
    }
}
template <bool F32>
__device__ __forceinline__ void clip_store(void *out, int64_t o, int valid, const float f[8]) {
    if constexpr (F32) {
        float *p = static_cast<float *>(out) + o;
        if (valid == 8) {
            __builtin_nontemporal_store(f32x4_any_t{f[0], f[1], f[2], f[3]}, reinterpret_cast<f32x4_any_t *>(p));
            __builtin_nontemporal_store(f32x4_any_t{f[4], f[5], f[6], f[7]}, reinterpret_cast<f32x4_any_t *>(p + 4));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < valid) p[j] = f[j];
        }
    } else {
        uint16_t *p = static_cast<uint16_t *>(out) + o;
        if (valid == 8) {
            __builtin_nontemporal_store(u32x4_any_t{rne_bf16x2(f[0], f[1]), rne_bf16x2(f[2], f[3]), rne_bf16x2(f[4], f[5]),
                                                    rne_bf16x2(f[6], f[7])}, reinterpret_cast<u32x4_any_t *>(p));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < valid) p[j] = (uint16_t)rne_bf16(f[j]);
        }
    }
}

// Chunk u of this thread in the tile at element `at`, and how many of its 8 elements exist.
__device__ __forceinline__ int64_t chunk_of(int64_t at, int u) { return at + (int64_t)(u * CLIP_THREADS + (int)threadIdx.x) * 8; }

template <int P, bool G32>
__device__ __forceinline__ void norm_tile(const void *g, int64_t at, int64_t n, double &s0, double &s1) {
    float f[CLIP_UNROLL][8];
    if (n - at >= CLIP_TILE) {
#pragma unroll
        for (int u = 0; u < CLIP_UNROLL; ++u) clip_load<G32>(g, chunk_of(at, u), 8, f[u]);
    } else {
#pragma unroll
        for (int u = 0; u < CLIP_UNROLL; ++u) clip_load<G32>(g, chunk_of(at, u), clamp_valid(n, chunk_of(at, u)), f[u]);
    }
#pragma unroll
    for (int u = 0; u < CLIP_UNROLL; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) norm_add<P>(j & 1 ? s1 : s0, f[u][j]);
}

// have: partial sums that earlier launches wrote
template <int P>
__global__ __launch_bounds__(CLIP_THREADS) void norm_kernel(ClipArgs a, double *partial, int have) {
    __shared__ double red[CLIP_THREADS / 64];
    double s0 = threadIdx.x == 0 && (int)blockIdx.x < have ? partial[blockIdx.x] : 0.0, s1 = 0.0;
    int i = 0;
    for (int t = blockIdx.x; t < a.start[a.count]; t += gridDim.x) {
        while (t >= a.start[i + 1]) ++i;
        const int64_t at = (int64_t)(t - a.start[i]) * CLIP_TILE;
        const uint32_t f = a.flags[i];
        if (f & CLIP_G32) norm_tile<P, true>(a.g[i], at, a.n[i], s0, s1);
        else norm_tile<P, false>(a.g[i], at, a.n[i], s0, s1);
    }
    const double s = norm_block<P>(norm_join<P>(s0, s1), red);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// The norm from the partial sums, in every thread.
template <int P>
__device__ __forceinline__ float norm_total(const double *partial, int parts, double *red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += CLIP_THREADS) s = norm_join<P>(s, partial[i]);
    return norm_root<P>(norm_block<P>(s, red));
}

template <int P>
__global__ __launch_bounds__(CLIP_THREADS) void norm_finish_kernel(const double *partial, int parts, float *norm_out) {
    __shared__ double red[CLIP_THREADS / 64];
    const float norm = norm_total<P>(partial, parts, red);
    if (threadIdx.x == 0) *norm_out = norm;
}

template <bool G32, bool O32>
__device__ __forceinline__ void clip_tile(const void *g, void *out, int64_t at, int64_t n, float c) {
    float f[CLIP_UNROLL][8];
    const bool full = n - at >= CLIP_TILE;
    if (full) {
#pragma unroll
        for (int u = 0; u < CLIP_UNROLL; ++u) clip_load<G32>(g, chunk_of(at, u), 8, f[u]);
    } else {
#pragma unroll
        for (int u = 0; u < CLIP_UNROLL; ++u) clip_load<G32>(g, chunk_of(at, u), clamp_valid(n, chunk_of(at, u)), f[u]);
    }
#pragma unroll
    for (int u = 0; u < CLIP_UNROLL; ++u) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[u][j] = f[u][j] * c;
        clip_store<O32>(out, chunk_of(at, u), full ? 8 : clamp_valid(n, chunk_of(at, u)), f[u]);
    }
}

template <int P>
__global__ __launch_bounds__(CLIP_THREADS) void clip_kernel(ClipArgs a, const double *partial, int parts, float max_norm,
                                                            float *norm_out) {
    __shared__ double red[CLIP_THREADS / 64];
    const float norm = norm_total<P>(partial, parts, red);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    float c = max_norm / (norm + CLIP_EPS);
    c = c >= 1.0f ? 1.0f : c;                        // NaN stays
    int i = 0;
    for (int t = blockIdx.x; t < a.start[a.count]; t += gridDim.x) {
        while (t >= a.start[i + 1]) ++i;
        if (c == 1.0f && a.out[i] == a.g[i]) continue;   // in place and nothing to cut
        const int64_t at = (int64_t)(t - a.start[i]) * CLIP_TILE, n = a.n[i];
        const uint32_t f = a.flags[i];
        if (f & CLIP_O32) clip_tile<true, true>(a.g[i], a.out[i], at, n, c);
        else if (f & CLIP_G32) clip_tile<true, false>(a.g[i], a.out[i], at, n, c);
        else clip_tile<false, false>(a.g[i], a.out[i], at, n, c);
    }
}

// The next launch's tensors from items[i] on (i moves past them); its work-groups, 0 if nothing is left.
static unsigned clip_fill(ClipArgs &a, const msr_clip_item *items, int32_t count, int32_t &i, bool outs) {
    int64_t tiles = 0;
    a.count = 0;
    for (; i < count && a.count < CLIP_MAXT; ++i) {
        const msr_clip_item &x = items[i];
        if (x.n == 0) continue;
        const int64_t more = (x.n + CLIP_TILE - 1) / CLIP_TILE;
        if (a.count && tiles + more > INT32_MAX) break;
        const int t = a.count++;
        a.g[t] = x.grad;
        a.out[t] = outs ? x.out : nullptr;
        a.n[t] = x.n;
        a.start[t] = (int32_t)tiles;
        a.flags[t] = (uint8_t)x.flags;
        tiles += more;
    }
    a.start[a.count] = (int32_t)tiles;
    return (unsigned)std::min<int64_t>(tiles, CLIP_GRID);
}

static int clip_check(const msr_clip_item *items, int32_t count, bool outs, const char *name) {
    if (count < 0 || (count > 0 && !items)) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
    for (int32_t i = 0; i < count; ++i) {
        const msr_clip_item &x = items[i];
        if (x.n < 0 || x.n > (int64_t)INT32_MAX * CLIP_TILE || (x.n > 0 && (!x.grad || (outs && !x.out))) ||
            (x.flags & ~(MSR_CLIP_GRAD_F32 | MSR_CLIP_OUT_F32)) ||
            (x.flags & (MSR_CLIP_GRAD_F32 | MSR_CLIP_OUT_F32)) == MSR_CLIP_OUT_F32) {
            set_error("%s: bad item %d", name, (int)i);
            return MSR_ERR_ARG;
        }
        if (!aligned(x.grad, x.flags & MSR_CLIP_GRAD_F32 ? 4 : 2) || (outs && !aligned(x.out, x.flags & MSR_CLIP_OUT_F32 ? 4 : 2))) {
            set_error("%s: item %d is not aligned to its type", name, (int)i);
            return MSR_ERR_ALIGN;
        }
    }
    return MSR_OK;
}

// The partial sums of a list: one per work-group of its largest norm launch.
static int clip_parts(const msr_clip_item *items, int32_t count) {
    ClipArgs a;
    int parts = 0;
    for (int32_t i = 0; i < count;) parts = std::max(parts, (int)clip_fill(a, items, count, i, false));
    return parts;
}

// Memory that one item writes may be touched by nothing else, but for its own gradient in place.
static int clip_apart(const msr_clip_item *items, int32_t count, bool outs, const float *norm_out, const void *ws, size_t ws_bytes,
                      const char *name) {
    std::vector<ItemRange> r;
    try {
        r.reserve(2 * (size_t)count + 2);
    } catch (const std::bad_alloc &) {
        set_error("%s: out of host memory", name);
        return MSR_ERR_ARG;
    }
    for (int32_t i = 0; i < count; ++i) {
        const msr_clip_item &x = items[i];
        if (x.n == 0) continue;
        const size_t gb = (x.flags & MSR_CLIP_GRAD_F32 ? 4 : 2) * (size_t)x.n, ob = (x.flags & MSR_CLIP_OUT_F32 ? 4 : 2) * (size_t)x.n;
        if (outs && partial_overlap(x.grad, gb, x.out, ob)) {
            set_error("%s: out of item %d overlaps its grad without being it", name, (int)i);
            return MSR_ERR_OVERLAP;
        }
        r.push_back({(uintptr_t)x.grad, (uintptr_t)x.grad + gb, i, false});
        if (outs) r.push_back({(uintptr_t)x.out, (uintptr_t)x.out + ob, i, true});
    }
    r.push_back({(uintptr_t)norm_out, (uintptr_t)norm_out + 4, count, true});
    r.push_back({(uintptr_t)ws, (uintptr_t)ws + ws_bytes, count + 1, true});
    if (ranges_conflict(r.data(), (int)r.size())) {
        set_error("%s: an out, the norm or the workspace overlaps another item of the list", name);
        return MSR_ERR_OVERLAP;
    }
    return MSR_OK;
}

template <int P>
static int clip_run(const msr_clip_item *items, int32_t count, bool outs, float max_norm, float *norm_out, double *partial,
                    hipStream_t s) {
    ClipArgs a;
    int parts = 0, rc;
    for (int32_t i = 0; i < count;) {
        const unsigned grid = clip_fill(a, items, count, i, false);
        if (!grid) break;
        hipLaunchKernelGGL((norm_kernel<P>), dim3(grid), dim3(CLIP_THREADS), 0, s, a, partial, parts);
        if ((rc = check_launch("norm_kernel"))) return rc;
        parts = std::max(parts, (int)grid);
    }
    if (!outs || !parts) {
        hipLaunchKernelGGL((norm_finish_kernel<P>), dim3(1), dim3(CLIP_THREADS), 0, s, partial, parts, norm_out);
        return check_launch("norm_finish_kernel");
    }
    for (int32_t i = 0; i < count;) {
        const unsigned grid = clip_fill(a, items, count, i, true);
        if (!grid) break;
        hipLaunchKernelGGL((clip_kernel<P>), dim3(grid), dim3(CLIP_THREADS), 0, s, a, partial, parts, max_norm, norm_out);
        if ((rc = check_launch("clip_kernel"))) return rc;
        norm_out = nullptr;
    }
    return MSR_OK;
}

static int clip_entry(const char *name, const msr_clip_item *items, int32_t count, bool outs, int32_t norm, float max_norm,
                      float *norm_out, void *workspace, size_t workspace_bytes, msr_stream_t stream) {
    int rc = clip_check(items, count, outs, name);
    if (rc) return rc;
    if (norm != MSR_NORM_1 && norm != MSR_NORM_2 && norm != MSR_NORM_INF) {
        set_error("%s: norm %d is not MSR_NORM_1, _2 or _INF", name, (int)norm);
        return MSR_ERR_ARG;
    }
    if (!norm_out) { set_error("%s: norm_out is NULL", name); return MSR_ERR_ARG; }
    if (!aligned(norm_out, 4) || !aligned(workspace, 8)) {
        set_error("%s: norm_out must be 4-byte and the workspace 8-byte aligned", name);
        return MSR_ERR_ALIGN;
    }
    const size_t need = (size_t)clip_parts(items, count) * sizeof(double);
    if (need && (!workspace || workspace_bytes < need)) {
        set_error("%s: workspace of %zu bytes is smaller than the %zu required", name, workspace_bytes, need);
        return MSR_ERR_WORKSPACE;
    }
    if ((rc = clip_apart(items, count, outs, norm_out, workspace, need, name))) return rc;
    double *const ws = static_cast<double *>(workspace);
    hipStream_t s = (hipStream_t)stream;
    if (norm == MSR_NORM_1) return clip_run<MSR_NORM_1>(items, count, outs, max_norm, norm_out, ws, s);
    if (norm == MSR_NORM_2) return clip_run<MSR_NORM_2>(items, count, outs, max_norm, norm_out, ws, s);
    return clip_run<MSR_NORM_INF>(items, count, outs, max_norm, norm_out, ws, s);
}

}  // namespace msr

using namespace msr;

extern "C" {

int msr_grad_norm_workspace_bytes(const msr_clip_item *items, int32_t count, size_t *bytes) {
    const int rc = clip_check(items, count, false, "msr_grad_norm_workspace_bytes");
    if (rc) return rc;
    if (!bytes) { set_error("msr_grad_norm_workspace_bytes: bytes is NULL"); return MSR_ERR_ARG; }
    *bytes = (size_t)clip_parts(items, count) * sizeof(double);
    return MSR_OK;
}

int msr_grad_norm(const msr_clip_item *items, int32_t count, int32_t norm, float *norm_out, void *workspace,
                  size_t workspace_bytes, msr_stream_t stream) {
    return clip_entry("msr_grad_norm", items, count, false, norm, 0.0f, norm_out, workspace, workspace_bytes, stream);
}

int msr_clip_grads(const msr_clip_item *items, int32_t count, int32_t norm, float max_norm, float *norm_out,
                   void *workspace, size_t workspace_bytes, msr_stream_t stream) {
    return clip_entry("msr_clip_grads", items, count, true, norm, max_norm, norm_out, workspace, workspace_bytes, stream);
}

}  // extern "C"
