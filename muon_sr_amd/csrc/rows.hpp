// Pieces of rows of bf16 or fp32 elements held in registers, sums over a wave, and the host's overlap check.
// Used by the embedding, the norm, the router's balance loss and the head.
#pragma once

#include <type_traits>

#include "common.hpp"
#include "vecio.hpp"

namespace msr {

struct __attribute__((packed, aligned(2))) Bytes16 { uint32_t w[4]; };   // 16 bytes at any address of an element type
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ void st_nt16(void *p, const Bytes16 &v) {
    __builtin_nontemporal_store(u32x4_any_t{v.w[0], v.w[1], v.w[2], v.w[3]}, static_cast<u32x4_any_t *>(p));
}

// 16 bytes of a row: N elements from column c on, those from d on zero and not stored.  Rows may begin at any element:
// global accesses of 16 bytes need no more alignment than that.
template <typename T>
struct Cells {
    static constexpr int N = 16 / (int)sizeof(T);
    Bytes16 v;
    __device__ __forceinline__ void load(const T *row, int64_t c, int64_t d) {
        if (c + N <= d) {
            v = *reinterpret_cast<const Bytes16 *>(row + c);
        } else if (c >= d) {             // (of a row of whole cells no lane goes through its elements)
            v = Bytes16{};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 2) {
                    const uint32_t lo = c + 2 * i < d ? row[c + 2 * i] : 0u, hi = c + 2 * i + 1 < d ? row[c + 2 * i + 1] : 0u;
                    v.w[i] = lo | hi << 16;
                } else {
                    v.w[i] = c + i < d ? __float_as_uint(row[c + i]) : 0u;
                }
            }
        }
    }
    // NT: past the caches
    template <bool NT = false>
    __device__ __forceinline__ void store(T *row, int64_t c, int64_t d) const {
        if (c + N <= d) {
            if constexpr (NT) st_nt16(row + c, v);
            else *reinterpret_cast<Bytes16 *>(row + c) = v;
        } else if (c < d) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 2) {
                    if (c + 2 * i < d) row[c + 2 * i] = (uint16_t)v.w[i];
                    if (c + 2 * i + 1 < d) row[c + 2 * i + 1] = (uint16_t)(v.w[i] >> 16);
                } else {
                    if (c + i < d) row[c + i] = __uint_as_float(v.w[i]);
                }
            }
        }
    }
    __device__ __forceinline__ void get(float (&f)[N]) const {
        if constexpr (sizeof(T) == 2) {
            unpack8(v.w, f);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v.w[i]);
        }
    }
    __device__ __forceinline__ void set(const float (&f)[N]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2) v.w[i] = rne_bf16x2(f[2 * i], f[2 * i + 1]);
            else v.w[i] = __float_as_uint(f[i]);
        }
    }
};

// x of the lane CTRL turns to within a row of 16 (DPP row_ror)
template <int CTRL>
__device__ __forceinline__ float turned(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row16_sum(float v) {
    v += turned<0x121>(v);
    v += turned<0x122>(v);
    v += turned<0x124>(v);
    return v + turned<0x128>(v);
}
// The sums of two values over the wave, in every lane
__device__ __forceinline__ float2 wave_sum2(float x, float y) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    float v = __uint_as_float(h[0]) + __uint_as_float(h[1]);            // lanes 0 to 31: x, the others: y
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = row16_sum(__uint_as_float(q[0]) + __uint_as_float(q[1]));
    return make_float2(__uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 0)),
                       __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 32)));
}

// Sums and maxima over groups of L = 8, 16, 32 or 64 lanes, in every lane of the group
struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
template <int L, typename Op>
__device__ __forceinline__ float over_group(float x, Op op) {
    x = op(x, turned<0xB1>(x));                        // quad_perm [1, 0, 3, 2]
    x = op(x, turned<0x4E>(x));                        // quad_perm [2, 3, 0, 1]
    x = op(x, turned<0x141>(x));                       // row_half_mirror
    if constexpr (L >= 16) x = op(x, turned<0x140>(x));   // row_mirror
    if constexpr (L >= 32) {
        const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = op(__uint_as_float(q[0]), __uint_as_float(q[1]));
    }
    if constexpr (L >= 64) {
        const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = op(__uint_as_float(h[0]), __uint_as_float(h[1]));
    }
    return x;
}

// A call's memory ranges, the first `outs` of them written: those overlap none of the others and not one another.
struct Range {
    const void *p;
    size_t n;
};
inline int ranges_apart(const char *name, const Range *r, int n, int outs) {
    for (int i = 0; i < outs; ++i)
        for (int j = i + 1; j < n; ++j) {
            const uintptr_t u = (uintptr_t)r[i].p, v = (uintptr_t)r[j].p;
            if (u && v && r[i].n && r[j].n && u < v + r[j].n && v < u + r[i].n) {
                set_error("%s: operands overlap (%d and %d)", name, i, j);
                return MSR_ERR_OVERLAP;
            }
        }
    return MSR_OK;
}
// rows of ld elements of `size` bytes, of which `width` count
inline size_t rows_bytes(int64_t rows, int64_t ld, int64_t width, size_t size) {
    return rows > 0 ? size * ((size_t)(rows - 1) * (size_t)ld + (size_t)width) : 0;
}
inline size_t elem_bytes(int32_t elem) { return elem == MSR_BF16 ? 2 : 4; }

}  // namespace msr
