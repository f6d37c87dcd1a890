// A router's balance loss: for logits [tokens][experts], the experts chosen for each token ids [tokens][k] and the n
// tokens that count,
//     p[t] = softmax(logits[t]),   c[e] = slots of these tokens with expert e,   f[e] = c[e] / (n k)
//     loss = experts / n sum_e f[e] sum_t p[t][e]
//     dlogits[t][e] = dloss p[t][e] (u[e] - sum_j u[j] p[t][j]),   u[e] = experts / n f[e]
// Both passes read the logits once; the probabilities are not stored, but the log of each token's sum is.  A token is held by
// L lanes, V experts each, so that a wave sums its tokens' probabilities in registers; the work-groups' sums (fp32) and counts are
// added in order by a second kernel.  Logits of -inf have probability 0, and a token that has no others counts with 0
// everywhere.
#include "rows.hpp"
#include "../../include/muon_sr_amd.h"

namespace msr {

constexpr int BAL_WGS = 256;

struct BalanceArgs {
    const void *logits;
    int64_t ld, tokens;
    const void *ids;
    const uint8_t *mask;         // [tokens], or null: every token counts
    float *lse;                  // [tokens]
    float *sums;                 // [work-groups][experts]
    int32_t *counts;             // [work-groups][experts + 1]: slots, and the tokens that count
    const float *dloss, *slope;  // one; u [experts]
    void *out;                   // dlogits [tokens][experts]
    int32_t experts, k, i64;
};

template <int L>
__device__ __forceinline__ float group_max(float x) {
#pragma unroll
    for (int w = 1; w < L; w <<= 1) x = fmaxf(x, __shfl_xor(x, w));
    return x;
}
template <int L>
__device__ __forceinline__ float group_sum(float x) {
    if constexpr (L == 64) return wave_sum(x);
#pragma unroll
    for (int w = 1; w < L; w <<= 1) x += __shfl_xor(x, w);
    return x;
}
template <typename T>
__device__ __forceinline__ float logit(const T *row, int e) {
    if constexpr (sizeof(T) == 2) return bf16_to_f32(row[e]);
    else return row[e];
}

// expert e is element e / L of lane e % L of its token's L lanes
template <typename T, int L, int V>
__global__ __launch_bounds__(256) void balance_kernel(BalanceArgs a) {
    constexpr int TOK = 256 / L;                      // tokens of a work-group at a time
    __shared__ float part[4][MSR_EXPERTS_MAX];
    __shared__ int hist[MSR_EXPERTS_MAX + 1];
    const int tid = threadIdx.x, sub = tid / L, l = tid % L;
    for (int e = tid; e <= a.experts; e += 256) hist[e] = 0;
    __syncthreads();
    float sum[V] = {};
    int counted = 0;
    for (int64_t t0 = (int64_t)blockIdx.x * TOK; t0 < a.tokens; t0 += (int64_t)gridDim.x * TOK) {
        const int64_t t = t0 + sub;
        const bool on = t < a.tokens && (!a.mask || a.mask[t]);
        const T *const row = static_cast<const T *>(a.logits) + t * a.ld;
        float x[V], m = -INFINITY, s = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            x[v] = on && v * L + l < a.experts ? logit(row, v * L + l) : -INFINITY;
            m = fmaxf(m, x[v]);
        }
        m = group_max<L>(m);
        const float at = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            x[v] = __builtin_amdgcn_exp2f((x[v] - at) * 1.4426950408889634f);
            s += x[v];
        }
        s = group_sum<L>(s);
        const float inv = s == 0.0f ? 0.0f : 1.0f / s;
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] = __builtin_fmaf(x[v], inv, sum[v]);
        if (on && l == 0) {
            a.lse[t] = s == 0.0f ? INFINITY : at + logf(s);      // exp(logit - lse) is 0 where there is no probability
            ++counted;
        }
        if (on)
            for (int j = l; j < a.k; j += L) {
                const int64_t e = a.i64 ? static_cast<const int64_t *>(a.ids)[t * a.k + j] : static_cast<const int32_t *>(a.ids)[t * a.k + j];
                if (e >= 0 && e < a.experts) atomicAdd(&hist[e], 1);
            }
    }
    if (counted) atomicAdd(&hist[a.experts], counted);
    // the sums over a wave's groups of lanes, then over the waves
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int w = L; w < 64; w <<= 1) sum[v] += __shfl_xor(sum[v], w);
        if ((tid & 63) < L && v * L + l < a.experts) part[tid >> 6][v * L + l] = sum[v];
    }
    __syncthreads();
    for (int e = tid; e <= a.experts; e += 256) {
        a.counts[(int64_t)blockIdx.x * (a.experts + 1) + e] = hist[e];
        if (e < a.experts) a.sums[(int64_t)blockIdx.x * a.experts + e] = ((part[0][e] + part[1][e]) + part[2][e]) + part[3][e];
    }
}

// One work-group: every expert's count and u, and the loss
__global__ __launch_bounds__(1024) void balance_join_kernel(const float *sums, const int32_t *parts, int groups, int experts, int k, float *loss,
                                                            int32_t *counts, float *slope) {
    __shared__ int all[MSR_EXPERTS_MAX + 1];
    __shared__ float probs[1024];
    __shared__ double wave_part[16];
    const int tid = threadIdx.x, E1 = experts + 1;
    for (int e = tid; e < E1; e += 1024) all[e] = 0;
    // a thread per expert and share of the work-groups
    const int shares = max(1, 1024 / E1), e = tid % E1, share = tid / E1;
    __syncthreads();
    if (shares == 1) {                                   // E1 may be 1025
        for (int i = tid; i < E1; i += 1024) {
            int c = 0;
            for (int g = 0; g < groups; ++g) c += parts[(int64_t)g * E1 + i];
            all[i] = c;
        }
    } else if (share < shares) {
        int c = 0;
#pragma unroll 8
        for (int g = share; g < groups; g += shares) c += parts[(int64_t)g * E1 + e];
        atomicAdd(&all[e], c);
    }
    // sums: a thread per expert and share, added in order
    const int lanes = max(1, 1024 / experts), x = tid % experts, part = tid / experts;
    float s = 0.0f;
    if (part < lanes) {
#pragma unroll 8
        for (int g = part; g < groups; g += lanes) s += sums[(int64_t)g * experts + x];
    }
    probs[tid] = s;
    __syncthreads();
    double mine = 0.0;
    if (tid < experts) {
        for (int i = 1; i < lanes; ++i) s += probs[i * experts + tid];
        const double n = max(all[experts], 1), f = all[tid] / (n * k);
        counts[tid] = all[tid];
        slope[tid] = (float)(f * experts / n);
        mine = f * s * experts / n;
    }
    for (int w = 32; w; w >>= 1) mine += __shfl_xor(mine, w);
    if ((tid & 63) == 0) wave_part[tid >> 6] = mine;
    __syncthreads();
    if (tid) return;
    for (int w = 1; w < 16; ++w) mine += wave_part[w];
    loss[0] = (float)mine;
}

template <typename T, int L, int V>
__global__ __launch_bounds__(256) void balance_grad_kernel(BalanceArgs a) {
    constexpr int TOK = 256 / L;
    const int sub = threadIdx.x / L, l = threadIdx.x % L;
    const float up = a.dloss[0];
    float u[V];
#pragma unroll
    for (int v = 0; v < V; ++v) u[v] = v * L + l < a.experts ? a.slope[v * L + l] : 0.0f;
    for (int64_t t = (int64_t)blockIdx.x * TOK + sub; t < a.tokens; t += (int64_t)gridDim.x * TOK) {
        const bool on = !a.mask || a.mask[t];
        const T *const row = static_cast<const T *>(a.logits) + t * a.ld;
        const float lse = on ? a.lse[t] : 0.0f;
        float p[V], dot = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            p[v] = on && v * L + l < a.experts ? __builtin_amdgcn_exp2f((logit(row, v * L + l) - lse) * 1.4426950408889634f) : 0.0f;
            dot = __builtin_fmaf(p[v], u[v], dot);
        }
        dot = group_sum<L>(dot);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (v * L + l >= a.experts) continue;
            const float d = on ? up * (p[v] * (u[v] - dot)) : 0.0f;
            T *const to = static_cast<T *>(a.out) + t * a.experts + v * L + l;
            if constexpr (sizeof(T) == 2) *to = (T)rne_bf16(d);
            else *to = d;
        }
    }
}

static int balance_groups(int64_t tokens) { return (int)std::min<int64_t>(std::max<int64_t>((tokens + 15) / 16, 1), BAL_WGS); }

// lanes per token and experts per lane
template <typename F>
static void balance_shape(int experts, F &&f) {
    using std::integral_constant;
    if (experts <= 8) f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    else if (experts <= 16) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (experts <= 32) f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else if (experts <= 64) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (experts <= 128) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (experts <= 256) f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    else if (experts <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    else f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

static int balance_check(const char *name, int64_t tokens, int32_t experts, int32_t k, int32_t elem) {
    if (tokens < 0 || k < 1 || experts < 1 || experts > MSR_EXPERTS_MAX || tokens >= (int64_t(1) << 30) / k || (elem != MSR_BF16 && elem != MSR_F32)) {
        set_error("%s: need tokens * k < 2^30, 1 to %d experts and bf16 or fp32 logits (got %lld x %d, %d experts, type %d)", name, MSR_EXPERTS_MAX,
                  (long long)tokens, (int)k, (int)experts, (int)elem);
        return MSR_ERR_ARG;
    }
    return MSR_OK;
}

}  // namespace msr

using namespace msr;

extern "C" {

int msr_balance_workspace_bytes(int64_t tokens, int32_t experts, size_t *bytes) {
    const int rc = balance_check("msr_balance_workspace_bytes", tokens, experts, 1, MSR_F32);
    if (rc) return rc;
    if (!bytes) { set_error("msr_balance_workspace_bytes: a pointer is NULL"); return MSR_ERR_ARG; }
    *bytes = (size_t)balance_groups(tokens) * (size_t)(2 * experts + 1) * 4;
    return MSR_OK;
}

int msr_balance_loss(const void *logits, int64_t ld, const void *ids, int32_t ids_i64, const uint8_t *mask, int64_t tokens, int32_t experts,
                     int32_t k, float *loss, int32_t *counts, float *lse, float *slope, int32_t elem, void *workspace, size_t workspace_bytes,
                     msr_stream_t stream) {
    const char *const name = "msr_balance_loss";
    int rc = balance_check(name, tokens, experts, k, elem);
    if (rc) return rc;
    if (!loss || !counts || !slope || (tokens > 0 && (!logits || !ids || !lse)) || ld < experts) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
    const size_t es = elem_bytes(elem), is = ids_i64 ? 8 : 4;
    if (!aligned(logits, es) || !aligned(ids, is) || !aligned(loss, 4) || !aligned(counts, 4) || !aligned(lse, 4) || !aligned(slope, 4) || !aligned(workspace, 4)) {
        set_error("%s: operands must be aligned to their types", name);
        return MSR_ERR_ALIGN;
    }
    const int groups = balance_groups(tokens);
    const size_t need = (size_t)groups * (size_t)(2 * experts + 1) * 4, n = (size_t)tokens;
    if (!workspace || workspace_bytes < need) {
        set_error("%s: workspace of %zu bytes is smaller than the %zu required", name, workspace_bytes, need);
        return MSR_ERR_WORKSPACE;
    }
    const Range r[8] = {{loss, 4}, {counts, 4 * (size_t)experts}, {lse, 4 * n}, {slope, 4 * (size_t)experts}, {workspace, need},
                        {logits, rows_bytes(tokens, ld, experts, es)}, {ids, n * (size_t)k * is}, {mask, n}};
    rc = ranges_apart(name, r, 8, 5);
    if (rc) return rc;
    hipStream_t s = (hipStream_t)stream;
    BalanceArgs a{};
    a.logits = logits; a.ld = ld; a.tokens = tokens; a.ids = ids; a.i64 = ids_i64 != 0; a.mask = mask; a.lse = lse; a.experts = experts; a.k = k;
    a.sums = static_cast<float *>(workspace);
    a.counts = reinterpret_cast<int32_t *>(a.sums + (size_t)groups * (size_t)experts);
    balance_shape(experts, [&](auto l, auto v) {
        if (elem == MSR_BF16) hipLaunchKernelGGL((balance_kernel<uint16_t, decltype(l)::value, decltype(v)::value>), dim3(groups), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((balance_kernel<float, decltype(l)::value, decltype(v)::value>), dim3(groups), dim3(256), 0, s, a);
    });
    if ((rc = check_launch("balance_kernel"))) return rc;
    hipLaunchKernelGGL(balance_join_kernel, dim3(1), dim3(1024), 0, s, a.sums, a.counts, groups, experts, k, loss, counts, slope);
    return check_launch("balance_join_kernel");
}

int msr_balance_grad(const void *logits, int64_t ld, const uint8_t *mask, const float *lse, const float *slope, const float *dloss,
                     int64_t tokens, int32_t experts, void *dlogits, int32_t elem, msr_stream_t stream) {
    const char *const name = "msr_balance_grad";
    int rc = balance_check(name, tokens, experts, 1, elem);
    if (rc || tokens == 0) return rc;
    if (!logits || !lse || !slope || !dloss || !dlogits || ld < experts) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
    const size_t es = elem_bytes(elem), n = (size_t)tokens;
    if (!aligned(logits, es) || !aligned(dlogits, es) || !aligned(lse, 4) || !aligned(slope, 4) || !aligned(dloss, 4)) {
        set_error("%s: operands must be aligned to their types", name);
        return MSR_ERR_ALIGN;
    }
    const Range r[6] = {{dlogits, n * (size_t)experts * es}, {logits, rows_bytes(tokens, ld, experts, es)}, {mask, n}, {lse, 4 * n},
                        {slope, 4 * (size_t)experts}, {dloss, 4}};
    rc = ranges_apart(name, r, 6, 1);
    if (rc) return rc;
    BalanceArgs a{};
    a.logits = logits; a.ld = ld; a.tokens = tokens; a.mask = mask; a.lse = const_cast<float *>(lse); a.slope = slope; a.dloss = dloss;
    a.out = dlogits; a.experts = experts;
    balance_shape(experts, [&](auto l, auto v) {
        const dim3 grid(grid_for(tokens, 256 / decltype(l)::value, 256 * 8));
        if (elem == MSR_BF16) hipLaunchKernelGGL((balance_grad_kernel<uint16_t, decltype(l)::value, decltype(v)::value>), grid, dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((balance_grad_kernel<float, decltype(l)::value, decltype(v)::value>), grid, dim3(256), 0, (hipStream_t)stream, a);
    });
    return check_launch("balance_grad_kernel");
}

}  // extern "C"
