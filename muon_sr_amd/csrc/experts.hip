// The experts' products over rows sorted by expert, with group sizes known only on the GPU:
//     forward   y[r]  = W[e] x[r]             m = rows of e, n = out, k = in
//     dgrad     dx[r] = W[e]^T dy[r]          m = rows of e, n = in,  k = out
//     wgrad     dw[e] = sum_r dy[r] x[r]^T    m = out,       n = in,  k = rows of e
// as tiles of the bf16 MFMA with fp32 accumulators.  The grid is an upper bound that depends on the
// number of rows alone; each work-group finds its group and tile from the offsets.
#include "gemm.hpp"
#include "../../include/muon_sr_amd.h"

namespace msr {

enum : int { EX_FWD = 0, EX_DGRAD = 1, EX_WGRAD = 2 };

struct ExpertArgs {
    const uint16_t *P;           // x (forward), dy (dgrad, wgrad): the operand of m
    int64_t ldp;
    const uint16_t *Q;           // W (forward, dgrad), x (wgrad): the operand of n
    int64_t ldq;
    uint16_t *D;                 // y, dx [rows][n], or dw / acc [experts][m][n]
    const int32_t *offsets;
    int64_t rows;
    int32_t experts, M, N, K;    // M: wgrad only; K: not wgrad
    int32_t zero_init;
    Noise ns;
};

// First row of group e: experts, then the rows without one (e = experts).
__device__ __forceinline__ int group_row(const ExpertArgs &a, int e) {
    return e <= 0 ? 0 : e > a.experts ? (int)a.rows : min(max(a.offsets[e], 0), (int)a.rows);
}

constexpr int XT = 64, XK = 32, XP = XK + 8;    // tile, k per slab, LDS row pitch

// MODE: noise mode of the accumulation, or -1 for a plain store.
template <int KIND, int MODE>
__global__ __launch_bounds__(256) void experts_kernel(ExpertArgs a) {
    __shared__ uint16_t lp[XT * XP], lq[XT * XP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
    const int n0 = blockIdx.x * XT;
    int e = 0, m0 = 0, M, K, lo = 0, hi = 0;
    if constexpr (KIND == EX_WGRAD) {
        e = blockIdx.z;
        m0 = blockIdx.y * XT;
        lo = group_row(a, e);
        hi = max(lo, group_row(a, e + 1));
        M = a.M;
        K = hi - lo;
    } else {
        int t = blockIdx.y;
        for (; e <= a.experts; ++e) {
            lo = group_row(a, e);
            hi = max(lo, group_row(a, e + 1));
            const int tiles = (hi - lo + XT - 1) / XT;
            if (t < tiles) break;
            t -= tiles;
        }
        if (e > a.experts) return;
        m0 = t * XT;
        M = hi - lo;
        K = e < a.experts ? a.K : 0;
    }
    const uint16_t *P = a.P + (int64_t)lo * a.ldp;
    const uint16_t *Q = KIND == EX_WGRAD ? a.Q + (int64_t)lo * a.ldq : a.Q + (int64_t)e * a.N * a.K;
    f32x16_t acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    for (int k0 = 0; k0 < K; k0 += XK) {
        for (int i = tid; i < XT * XK; i += 256) {
            const int r = KIND == EX_WGRAD ? i % XT : i / XK, k = KIND == EX_WGRAD ? i / XT : i % XK;
            uint16_t v = 0;
            if (m0 + r < M && k0 + k < K)
                v = KIND == EX_WGRAD ? P[(int64_t)(k0 + k) * a.ldp + m0 + r] : P[(int64_t)(m0 + r) * a.ldp + k0 + k];
            lp[r * XP + k] = v;
            const int c = KIND == EX_FWD ? i / XK : i % XT, kq = KIND == EX_FWD ? i % XK : i / XT;
            v = 0;
            if (n0 + c < a.N && k0 + kq < K)
                v = KIND == EX_FWD ? Q[(int64_t)(n0 + c) * a.K + k0 + kq]
                                   : Q[(int64_t)(k0 + kq) * (KIND == EX_WGRAD ? a.ldq : a.N) + n0 + c];
            lq[c * XP + kq] = v;
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < XK; ks += 16) {
            const bf16x8_t p = *reinterpret_cast<const bf16x8_t *>(lp + (wm * 32 + (lane & 31)) * XP + ks + 8 * (lane >> 5));
            const bf16x8_t q = *reinterpret_cast<const bf16x8_t *>(lq + (wn * 32 + (lane & 31)) * XP + ks + 8 * (lane >> 5));
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q, p, acc, 0, 0, 0);
        }
        __syncthreads();
    }
    const int m = m0 + wm * 32 + (lane & 31);
    if (m >= M) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int n = n0 + wn * 32 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
        if (n >= a.N) continue;
        const uint32_t v = rne_bf16(acc[i]);
        if constexpr (KIND == EX_WGRAD) {
            const int64_t o = ((int64_t)e * M + m) * a.N + n;
            if constexpr (MODE >= 0) {
                const float old = a.zero_init ? 0.0f : bf16_to_f32(a.D[o]);
                a.D[o] = (uint16_t)sr_bf16(old + bf16_to_f32(v), noise1<MODE>(a.ns, o));
            } else {
                a.D[o] = (uint16_t)v;
            }
        } else {
            a.D[((int64_t)lo + m) * a.N + n] = (uint16_t)v;
        }
    }
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
    if (!offsets || (rows > 0 && (!p || !w || !out)) || ldp < width) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
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
    a.rows = rows; a.experts = experts; a.N = (int)outw; a.K = (int)width;
    const dim3 grid((unsigned)((outw + XT - 1) / XT), (unsigned)(rows / XT + experts + 1));
    if (kind == EX_FWD) hipLaunchKernelGGL((experts_kernel<EX_FWD, -1>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((experts_kernel<EX_DGRAD, -1>), grid, dim3(256), 0, s, a);
    return check_launch(name);
}

static int experts_weights(const char *name, uint16_t *d, const uint16_t *x, int64_t ldx, const uint16_t *dy, int64_t lddy,
                           const int32_t *offsets, int64_t rows, int32_t experts, int64_t in_f, int64_t out_f, int mode,
                           uint32_t seed, int32_t zero_init, const uint16_t *inject, hipStream_t s) {
    if (!d || !offsets || (rows > 0 && (!x || !dy)) || ldx < in_f || lddy < out_f) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
    if (!aligned(d, 16) || !aligned(x, 16) || !aligned(dy, 16) || !aligned(offsets, 4) || ldx % 8 || lddy % 8) {
        set_error("%s: operands must be 16-byte aligned with row strides a multiple of 8", name);
        return MSR_ERR_ALIGN;
    }
    const Span in[3] = {{x, row_bytes(rows, ldx, in_f)}, {dy, row_bytes(rows, lddy, out_f)}, {offsets, 4 * ((size_t)experts + 1)}};
    const int rc = experts_spans(name, {d, 2 * (size_t)experts * (size_t)(in_f * out_f)}, in, 3);
    if (rc) return rc;
    ExpertArgs a{};
    a.P = dy; a.ldp = lddy; a.Q = x; a.ldq = ldx; a.D = d; a.offsets = offsets;
    a.rows = rows; a.experts = experts; a.M = (int)out_f; a.N = (int)in_f; a.zero_init = zero_init != 0;
    a.ns.key = seed_key(seed, 0);
    a.ns.inject = inject;
    const dim3 grid((unsigned)((in_f + XT - 1) / XT), (unsigned)((out_f + XT - 1) / XT), (unsigned)experts);
    if (mode < 0) hipLaunchKernelGGL((experts_kernel<EX_WGRAD, -1>), grid, dim3(256), 0, s, a);
    else MSR_DISPATCH_NOISE(mode, MODE, hipLaunchKernelGGL((experts_kernel<EX_WGRAD, MODE>), grid, dim3(256), 0, s, a));
    return check_launch(name);
}

}  // namespace msr

using namespace msr;

extern "C" {

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
