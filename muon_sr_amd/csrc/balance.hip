// A router's balance loss: for logits [tokens][experts], the experts chosen for each token ids [tokens][k] and the n
// tokens that count,
//     p[t] = softmax(logits[t]),   c[e] = slots of these tokens with expert e,   f[e] = c[e] / (n k)
//     loss = experts / n sum_e f[e] sum_t p[t][e]
//     dlogits[t][e] = dloss p[t][e] (u[e] - sum_j u[j] p[t][j]),   u[e] = experts / n f[e]
// Both passes read the logits once; the probabilities are not stored, but each token's largest logit m and 1 / s, s = sum exp(logit - m), are:
// both passes form p = exp(logit - m) / s by the same instructions.  (m + log s in one number is rounded at the size of the logits, and all p of a
// token are off by a common factor, which u[e] - sum_j u[j] p[j] multiplies where the load is nearly even: 64 experts, u spread by 1 %,
// logits of deviation 1 around 1000, dlogits off by 2e-3, and by 8e-6 so wherever they are.)  A token is held by
// L lanes, U cells of 16 bytes each, so that a wave sums the probabilities of 64 / L tokens at a time in registers, the next
// tokens' logits on their way; the work-groups' sums (fp32) and counts are added in order by a second kernel.  Logits of -inf have probability 0, and a token that has no others counts with 0
// everywhere.
#include "rows.hpp"
#include "../../include/muon_sr_amd.h"

namespace msr {

constexpr int BAL_WGS = 256, BAL_THREADS = 1024;   // at most: one work-group to a CU, whose sums the second kernel adds

struct BalanceArgs {
    const void *logits;
    int64_t ld, tokens;
    const void *ids;
    const uint8_t *mask;         // [tokens], or null: every token counts
    float *stats;                // [2][tokens]: m (0 of a token without probabilities), 1 / s (0 of it)
    float *sums;                 // [work-groups][experts]
    int32_t *counts;             // [work-groups][experts + 1]: slots, and the tokens that count
    const float *dloss, *slope;  // one; u [experts]
    void *out;                   // dlogits [tokens][experts]
    int32_t experts, k, i64;
};

constexpr float LOG2E = 1.4426950408889634f;

// Work-group b's tokens: [b per, (b + 1) per).  blockDim.x: 256 or 1024.
template <typename T, int L, int U>
__global__ __launch_bounds__(BAL_THREADS) void balance_kernel(BalanceArgs a, int64_t per) {
    using C = Cells<T>;
    constexpr int N = C::N;
    __shared__ float part[U * N * L][17];   // [experts][waves]
    __shared__ int hist[MSR_EXPERTS_MAX + 1];
    const int tid = threadIdx.x, sub = tid / L, l = tid % L, toks = blockDim.x / L, waves = blockDim.x / 64;
    for (int e = tid; e <= a.experts; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * per, last = min(first + per, a.tokens);
    // the counts
    int counted = 0;
    if (a.mask)
        for (int64_t t = first + tid; t < last; t += blockDim.x) counted += a.mask[t] != 0;
    else if (tid == 0 && last > first)
        counted = (int)(last - first);
    if (counted) atomicAdd(&hist[a.experts], counted);
    constexpr int SLOTS = 4;                          // whose loads are in flight together
    for (int64_t i0 = first * a.k + tid; i0 < last * a.k; i0 += SLOTS * blockDim.x) {
        int64_t e[SLOTS];
        bool on[SLOTS];
#pragma unroll
        for (int y = 0; y < SLOTS; ++y) {
            const int64_t i = i0 + y * blockDim.x;
            on[y] = i < last * a.k;
            e[y] = -1;
            if (on[y]) {
                e[y] = a.i64 ? static_cast<const int64_t *>(a.ids)[i] : static_cast<const int32_t *>(a.ids)[i];
                if (a.mask) on[y] = a.mask[(uint32_t)i / (uint32_t)a.k];
            }
        }
#pragma unroll
        for (int y = 0; y < SLOTS; ++y)
            if (on[y] && e[y] >= 0 && e[y] < a.experts) atomicAdd(&hist[e[y]], 1);
    }
    // the probabilities
    float sum[U][N] = {};
    // A tokens ahead, in turn (131071 tokens of 256 experts: 43 us with one, 40 with two, 39 with four)
    constexpr int A = U == 1 ? 4 : 2;
    C next[A][U];
    bool next_on[A] = {};
    auto fetch = [&](int64_t t, auto I) __attribute__((always_inline)) {
        constexpr int i = decltype(I)::value;
        next_on[i] = t < last && (!a.mask || a.mask[t]);
        if (!next_on[i]) return;
#pragma unroll
        for (int u = 0; u < U; ++u) next[i][u].load(static_cast<const T *>(a.logits) + t * a.ld, (u * L + l) * N, a.experts);
    };
    auto token = [&](int64_t t, auto I) __attribute__((always_inline)) {
        constexpr int i = decltype(I)::value;
        const bool on = next_on[i];
        float x[U][N], m = -INFINITY, s = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            next[i][u].get(x[u]);
            // (a select for each element: with a branch around them clang 22.0.0 of ROCm 7.2.0 loses the -inf of element 0 in lanes whose first
            // element is absent)
            const int held = on ? a.experts - (u * L + l) * N : 0;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                x[u][e] = e < held ? x[u][e] : -INFINITY;
                m = fmaxf(m, x[u][e]);
            }
        }
        fetch(t + A * toks, I);
        m = over_group<L>(m, Max{});
        const float at = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                x[u][e] = __builtin_amdgcn_exp2f((x[u][e] - at) * LOG2E);
                s += x[u][e];
            }
        s = over_group<L>(s, Add{});
        // (the instruction for 1 / s is within an ulp, one step of Newton's rounds it)
        const float near = __builtin_amdgcn_rcpf(s), inv = s == 0.0f ? 0.0f : __builtin_fmaf(__builtin_fmaf(-s, near, 1.0f), near, near);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) sum[u][e] = __builtin_fmaf(x[u][e], inv, sum[u][e]);
        if (on && l == 0) {
            a.stats[t] = at;
            a.stats[a.tokens + t] = inv;
        }
    };
    auto each = [&](auto &&f) __attribute__((always_inline)) {
        f(std::integral_constant<int, 0>{});
        f(std::integral_constant<int, 1>{});
        if constexpr (A > 2) {
            f(std::integral_constant<int, 2>{});
            f(std::integral_constant<int, 3>{});
        }
    };
    each([&](auto I) __attribute__((always_inline)) { fetch(first + sub + decltype(I)::value * toks, I); });
    for (int64_t t0 = first; t0 < last; t0 += A * toks)
        each([&](auto I) __attribute__((always_inline)) {
            if (t0 + decltype(I)::value * toks < last) token(t0 + sub + decltype(I)::value * toks, I);
        });
    // over a wave's groups of lanes, then over the waves
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float v = sum[u][e];
#pragma unroll
            for (int w = L; w < 64; w <<= 1) v += __shfl_xor(v, w);
            if ((tid & 63) < L) part[(u * L + l) * N + e][tid >> 6] = v;
        }
    __syncthreads();
    for (int e = tid; e <= a.experts; e += blockDim.x) {
        a.counts[(int64_t)blockIdx.x * (a.experts + 1) + e] = hist[e];
        if (e == a.experts) continue;
        float v = part[e][0];
        for (int w = 1; w < waves; ++w) v += part[e][w];
        a.sums[(int64_t)blockIdx.x * a.experts + e] = v;
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
#pragma unroll 16
        for (int g = share; g < groups; g += shares) c += parts[(int64_t)g * E1 + e];
        atomicAdd(&all[e], c);
    }
    // sums: a thread per expert and share, added in order
    const int lanes = max(1, 1024 / experts), x = tid % experts, part = tid / experts;
    float s = 0.0f;
    if (part < lanes) {
#pragma unroll 16
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

template <typename T, int L, int U>
__global__ __launch_bounds__(256) void balance_grad_kernel(BalanceArgs a) {
    using C = Cells<T>;
    constexpr int N = C::N, TOK = 256 / L;
    const int sub = threadIdx.x / L, l = threadIdx.x % L;
    const float up = a.dloss[0];
    float slope[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) slope[u][e] = (u * L + l) * N + e < a.experts ? a.slope[(u * L + l) * N + e] : 0.0f;
    for (int64_t t = (int64_t)blockIdx.x * TOK + sub; t < a.tokens; t += (int64_t)gridDim.x * TOK) {
        const bool on = !a.mask || a.mask[t];
        float p[U][N] = {}, dot = 0.0f;
        C v[U];
        if (on) {
            const float at = a.stats[t], inv = a.stats[a.tokens + t];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u].load(static_cast<const T *>(a.logits) + t * a.ld, (u * L + l) * N, a.experts);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                v[u].get(p[u]);
#pragma unroll
                for (int e = 0; e < N; ++e) {           // (what is beyond the experts is not stored, and its slope is 0)
                    p[u][e] = (u * L + l) * N + e < a.experts ? __builtin_amdgcn_exp2f((p[u][e] - at) * LOG2E) * inv : 0.0f;
                    dot = __builtin_fmaf(p[u][e], slope[u][e], dot);
                }
            }
        }
        dot = over_group<L>(dot, Add{});
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float d[N];
#pragma unroll
            for (int e = 0; e < N; ++e) d[e] = on ? up * (p[u][e] * (slope[u][e] - dot)) : 0.0f;
            v[u].set(d);
            v[u].store(static_cast<T *>(a.out) + t * a.experts, (u * L + l) * N, a.experts);
        }
    }
}

// Cells of a row, lanes per token and cells per lane
template <typename T, typename F>
static void balance_lanes(int experts, F &&f) {
    using std::integral_constant;
    const int cells = (experts + Cells<T>::N - 1) / Cells<T>::N;
    if (cells <= 8) f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    else if (cells <= 16) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (cells <= 32) f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else if (cells <= 64) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (cells <= 128) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if constexpr (sizeof(T) == 4) f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
}
// f(type, lanes, cells per lane)
template <typename F>
static void balance_shape(int32_t elem, int experts, F &&f) {
    if (elem == MSR_BF16) balance_lanes<uint16_t>(experts, [&](auto l, auto u) { f(uint16_t{}, l, u); });
    else balance_lanes<float>(experts, [&](auto l, auto u) { f(float{}, l, u); });
}

// Work-groups of 256 threads while they leave CUs idle, 1024 beyond; the tokens of each.
struct BalancePlan {
    int groups, threads;
    int64_t per;
};
static BalancePlan balance_plan(int64_t tokens, int32_t experts, int32_t elem) {
    int lanes = 64;
    balance_shape(elem, experts, [&](auto, auto l, auto) { lanes = decltype(l)::value; });
    BalancePlan p{};
    p.threads = tokens <= (int64_t)BAL_WGS * 256 / lanes ? 256 : BAL_THREADS;
    const int64_t at_once = p.threads / lanes, rounds = (tokens + at_once * BAL_WGS - 1) / (at_once * BAL_WGS);
    p.per = std::max<int64_t>(rounds, 1) * at_once;
    p.groups = (int)std::max<int64_t>((tokens + p.per - 1) / p.per, 1);
    return p;
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
    const int rc = balance_check("msr_balance_workspace_bytes", tokens, experts, 1, MSR_F32);   // (as much for either type)
    if (rc) return rc;
    if (!bytes) { set_error("msr_balance_workspace_bytes: a pointer is NULL"); return MSR_ERR_ARG; }
    *bytes = (size_t)std::max(balance_plan(tokens, experts, MSR_BF16).groups, balance_plan(tokens, experts, MSR_F32).groups) * (size_t)(2 * experts + 1) * 4;
    return MSR_OK;
}

int msr_balance_loss(const void *logits, int64_t ld, const void *ids, int32_t ids_i64, const uint8_t *mask, int64_t tokens, int32_t experts,
                     int32_t k, float *loss, int32_t *counts, float *stats, float *slope, int32_t elem, void *workspace, size_t workspace_bytes,
                     msr_stream_t stream) {
    const char *const name = "msr_balance_loss";
    int rc = balance_check(name, tokens, experts, k, elem);
    if (rc) return rc;
    if (!loss || !counts || !slope || (tokens > 0 && (!logits || !ids || !stats)) || ld < experts) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
    const size_t es = elem_bytes(elem), is = ids_i64 ? 8 : 4;
    if (!aligned(logits, es) || !aligned(ids, is) || !aligned(loss, 4) || !aligned(counts, 4) || !aligned(stats, 4) || !aligned(slope, 4) || !aligned(workspace, 4)) {
        set_error("%s: operands must be aligned to their types", name);
        return MSR_ERR_ALIGN;
    }
    const BalancePlan p = balance_plan(tokens, experts, elem);
    const int groups = p.groups;
    const size_t need = (size_t)groups * (size_t)(2 * experts + 1) * 4, n = (size_t)tokens;
    if (!workspace || workspace_bytes < need) {
        set_error("%s: workspace of %zu bytes is smaller than the %zu required", name, workspace_bytes, need);
        return MSR_ERR_WORKSPACE;
    }
    const Range r[8] = {{loss, 4}, {counts, 4 * (size_t)experts}, {stats, 8 * n}, {slope, 4 * (size_t)experts}, {workspace, need},
                        {logits, rows_bytes(tokens, ld, experts, es)}, {ids, n * (size_t)k * is}, {mask, n}};
    rc = ranges_apart(name, r, 8, 5);
    if (rc) return rc;
    hipStream_t s = (hipStream_t)stream;
    BalanceArgs a{};
    a.logits = logits; a.ld = ld; a.tokens = tokens; a.ids = ids; a.i64 = ids_i64 != 0; a.mask = mask; a.stats = stats; a.experts = experts; a.k = k;
    a.sums = static_cast<float *>(workspace);
    a.counts = reinterpret_cast<int32_t *>(a.sums + (size_t)groups * (size_t)experts);
    balance_shape(elem, experts, [&](auto t, auto l, auto u) {
        hipLaunchKernelGGL((balance_kernel<decltype(t), decltype(l)::value, decltype(u)::value>), dim3(groups), dim3(p.threads), 0, s, a, p.per);
    });
    if ((rc = check_launch("balance_kernel"))) return rc;
    hipLaunchKernelGGL(balance_join_kernel, dim3(1), dim3(1024), 0, s, a.sums, a.counts, groups, experts, k, loss, counts, slope);
    return check_launch("balance_join_kernel");
}

int msr_balance_grad(const void *logits, int64_t ld, const uint8_t *mask, const float *stats, const float *slope, const float *dloss,
                     int64_t tokens, int32_t experts, void *dlogits, int32_t elem, msr_stream_t stream) {
    const char *const name = "msr_balance_grad";
    int rc = balance_check(name, tokens, experts, 1, elem);
    if (rc || tokens == 0) return rc;
    if (!logits || !stats || !slope || !dloss || !dlogits || ld < experts) { set_error("%s: bad arguments", name); return MSR_ERR_ARG; }
    const size_t es = elem_bytes(elem), n = (size_t)tokens;
    if (!aligned(logits, es) || !aligned(dlogits, es) || !aligned(stats, 4) || !aligned(slope, 4) || !aligned(dloss, 4)) {
        set_error("%s: operands must be aligned to their types", name);
        return MSR_ERR_ALIGN;
    }
    const Range r[6] = {{dlogits, n * (size_t)experts * es}, {logits, rows_bytes(tokens, ld, experts, es)}, {mask, n}, {stats, 8 * n},
                        {slope, 4 * (size_t)experts}, {dloss, 4}};
    rc = ranges_apart(name, r, 6, 1);
    if (rc) return rc;
    BalanceArgs a{};
    a.logits = logits; a.ld = ld; a.tokens = tokens; a.mask = mask; a.stats = const_cast<float *>(stats); a.slope = slope; a.dloss = dloss;
    a.out = dlogits; a.experts = experts;
    balance_shape(elem, experts, [&](auto t, auto l, auto u) {
        const dim3 grid(grid_for(tokens, 256 / decltype(l)::value, 256 * 8));
        hipLaunchKernelGGL((balance_grad_kernel<decltype(t), decltype(l)::value, decltype(u)::value>), grid, dim3(256), 0, (hipStream_t)stream, a);
    });
    return check_launch("balance_grad_kernel");
}

}  // extern "C"
