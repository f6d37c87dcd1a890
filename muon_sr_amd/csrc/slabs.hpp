// T x T tiles of the bf16 MFMA with fp32 accumulators whose operands are read in the layout that their tensors have:
// K-contiguous ("row-major"), one 16-byte LDS read per fragment, or K-major, two transposing 8-byte reads.  K goes
// through a ring of LDS stages in slabs, filled by buffer loads that write LDS directly, slabs ahead.  What a slab has beyond
// its operand's rows or beyond K is beyond its buffer resource (or is sent there), where loads give zeros, so the main loop has
// no bounds of its own.  Used by the experts' products (experts.hip) and the head's (head.hip).
#pragma once

#include <type_traits>

#include "gemm.hpp"

namespace msr {

constexpr uint32_t X_NONE = 0x80000000u;     // byte offset beyond every buffer resource

// 16 bytes per lane from byte `off` of a resource of `bytes` bytes at `base` (both wave-uniform; zeros from
// beyond it) to 1 KiB of LDS.
__device__ __forceinline__ void load_lds16(const void *base, uint32_t bytes, char *lds, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, 0x00020000),
                                             (lds_void_t *)lds, 16, off, 0, 0, 0);
}

// One operand's slab of T rows (row-major) or T columns (K-major) x BK k, and the loads of one of
// NW waves: load i fills the 1 KiB block i NW + wave, lane l its bytes 16 l to 16 l + 15.
//  * row-major: rows of 2 BK bytes, 16-byte chunk c of row r at c ^ ((r >> 1) & 7) (BK = 64) or c ^ ((r >> 2) & 3)
//    (BK = 32), so that the 16 rows of a quarter of a fragment read cover all banks;
//  * K-major: rows of k of 2 T bytes, chunk c of row k at c ^ 4 (k & 3) (T >= 128) or c ^ 4 ((k >> 1) & 1)
//    (T = 64), so that the four rows of a transposing read fall in different banks.
template <int T, int NW, bool KM, int BK>
struct Slab {
    static constexpr int BYTES = T * BK * 2, LOADS = BYTES / (1024 * NW);
    static constexpr int CH = KM ? T / 8 : BK / 8;                              // chunks of a row
    static_assert(BYTES % (1024 * NW) == 0, "whole loads");
    static __device__ __forceinline__ int swizzle(int row) {
        if (KM) return T >= 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
        return BK == 64 ? (row >> 1) & 7 : (row >> 2) & 3;
    }
    uint32_t at[LOADS];          // byte offset of each load's chunk in the slab
    int chunk;                   // logical chunk, the same in every load (rows step by whole periods)
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld) {
        const int row0 = (wave * 64 + lane) / CH;
        chunk = ((wave * 64 + lane) % CH) ^ swizzle(row0);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) at[i] = (uint32_t)((row0 + i * (NW * 64 / CH)) * (uint32_t)ld * 2u + chunk * 16u);
    }
    // The slab at k0 (zeros from K on): `base` its operand's tile at k = 0; `rows` the tile's valid rows
    // (row-major: at most T); `width` the valid columns from the tile's first one on (K-major).
    __device__ __forceinline__ void load(char *lds, int wave, const uint16_t *base, int64_t ld, int rows, int width, int k0,
                                         int K) const {
        const int left = K - k0;
        const int64_t first = left <= 0 ? 0 : KM ? (int64_t)k0 * ld : k0;
        uint32_t bytes = KM ? (uint32_t)(min(left, BK) - 1) * (uint32_t)ld * 2u + (uint32_t)width * 2u
                            : (uint32_t)(rows - 1) * (uint32_t)ld * 2u + (uint32_t)left * 2u;
        if (left <= 0) bytes = 0;
        const bool in = KM || chunk * 8 < left;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) load_lds16(base + first, bytes, lds + (i * NW + wave) * 1024, in ? at[i] : X_NONE);
    }
};

// Fragment reads of a wave: rows (columns) w0 + 32 f + lane % 32, k = 16 ks + 8 (lane / 32) + 0..7.
// K-major: two transposing reads of 4 k each; in a read, lane i of a 16-lane group fetches row k = i / 4,
// columns 4 (i % 4) .. +3 of its group's 16 and returns element i % 4 of 4 lanes' rows.
template <int T, bool KM, int BK>
struct Frags {
    uint32_t base;
    int c0, x;
    __device__ __forceinline__ void init(int lane, int w0) {
        if constexpr (KM) {
            const int G = lane >> 4, i = lane & 15;
            base = (uint32_t)((8 * (G >> 1) + (i >> 2)) * (2 * T) + (i & 1) * 8);
            c0 = w0 / 8 + 2 * (G & 1) + ((i >> 1) & 1);
            x = Slab<T, 4, true, BK>::swizzle(i >> 2);
        } else {
            const int r = lane & 31;
            base = (uint32_t)((w0 + r) * (2 * BK));
            c0 = lane >> 5;
            x = Slab<T, 4, false, BK>::swizzle(r);
        }
    }
    __device__ __forceinline__ bf16x8_t read(const char *lds, int ks, int f) const {
        if constexpr (KM) {
            const char *p = lds + base + ks * 16 * (2 * T) + (uint32_t)(((c0 + 4 * f) ^ x) * 16);
            const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(p));
            const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(p + 4 * (2 * T)));
            return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            return *reinterpret_cast<const bf16x8_t *>(lds + base + f * 32 * (2 * BK) + ((2 * ks + c0) ^ x) * 16);
        }
    }
};

// T: tile; NW waves in a 2 x NW / 2 grid.
template <int T>
struct Shape {
    static constexpr int NW = T == 256 ? 8 : 4, WN = NW / 2;
    static constexpr int TM = T / 2, TN = T / WN, FM = TM / 32, FN = TN / 32;   // a wave's sub-tile and its 32-wide blocks
};

// One wave's part of a T x T tile of P Q^T.  P's T rows (columns, PK) are the tile's m, Q's its n.  lane l holds
// D[m = l % 32][n = 8 r + 4 (l / 32) + q] of each 32 x 32 block in acc[..][..][4 r + q].  BK: k per slab; S: LDS stages.
template <int T, int BK, int S, bool PK, bool QK>
struct Product {
    using SH = Shape<T>;
    using SP = Slab<T, SH::NW, PK, BK>;
    using SQ = Slab<T, SH::NW, QK, BK>;
    static constexpr int FM = SH::FM, FN = SH::FN, NS = BK / 16, LPS = SP::LOADS + SQ::LOADS;   // substeps of a slab, a wave's loads for it
    static_assert(NS % 2 == 0 && (S - 1) * LPS < 64, "fragment sets alternate; vmcnt is 6 bits");
    SP sp;
    SQ sq;
    Frags<T, PK, BK> rp;
    Frags<T, QK, BK> rq;
    f32x16_t acc[FM][FN];
    int wave;
    __device__ __forceinline__ void init(int wave_, int lane, int64_t ldp, int64_t ldq) {
        wave = wave_;
        sp.init(wave, lane, ldp);
        sq.init(wave, lane, ldq);
        rp.init(lane, wave / SH::WN * SH::TM);
        rq.init(lane, wave % SH::WN * SH::TN);
        clear();
    }

    // One operand's tile: its address at k = 0, row stride, valid rows (row-major: at most T) or valid columns
    // from the tile's first one on (K-major), and the end of its K.
    struct Side {
        const uint16_t *base;
        int64_t ld;
        int rows, width, kend;
    };

    // acc += the products over `slabs` slabs from k = kb on.  lds_p, lds_q: the LDS of a stage (an
    // integral_constant); one variable per stage and operand, so that the compiler knows that fragment reads of one
    // stage do not alias the loads into the others.  AHEAD: the first slabs are on their way (by ahead, with the same
    // arguments, after a barrier behind the last use of the stages).
    template <bool AHEAD = false, class LP, class LQ>
    __device__ __forceinline__ void run(LP lds_p, LQ lds_q, const Side &p, const Side &q, int kb, int slabs) {
        auto load = [&](auto ST, int k0) __attribute__((always_inline)) {
            sp.load(lds_p(ST), wave, p.base, p.ld, p.rows, p.width, kb + k0, p.kend);
            sq.load(lds_q(ST), wave, q.base, q.ld, q.rows, q.width, kb + k0, q.kend);
        };
        bf16x8_t fp[2][FM], fq[2][FN];
        auto read = [&](auto ST, int ks, int b) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < FM; ++i) fp[b][i] = rp.read(lds_p(ST), ks, i);
#pragma unroll
            for (int j = 0; j < FN; ++j) fq[b][j] = rq.read(lds_q(ST), ks, j);
        };
        auto mult = [&](int b) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fq[b][j], fp[b][i], acc[i][j], 0, 0, 0);
        };
        // The slab at k0 in stage ST, whose first fragments are read: the slab S - 1 ahead is loaded into the
        // stage that the barrier before freed; each substep's MFMAs run beside the next one's fragment reads, the
        // last substep's beside those of the next slab (unused after the last slab).  Beyond K there are slabs of
        // zeros without memory accesses, so that the counted wait is the same for every slab.
        auto slab = [&](auto ST, int k0) __attribute__((always_inline)) {
            constexpr int st = decltype(ST)::value;
            using NX = std::integral_constant<int, (st + 1) % S>;
            load(std::integral_constant<int, (st + S - 1) % S>{}, k0 + (S - 1) * BK);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks + 1 < NS; ++ks) {
                read(ST, ks + 1, (ks + 1) & 1);
                mult(ks & 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            wait_vm<(S - 2) * LPS>();                                       // own loads of the next slab landed
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // everyone's; this stage is read
            read(NX{}, 0, 0);
            mult(1);
            __builtin_amdgcn_sched_barrier(0);
        };
        if (slabs <= 0) return;
        // the first slab's stage is the one from which the last slab is in stage S - 1
        const int r = slabs % S;
        auto begin = [&](auto ST) __attribute__((always_inline)) {
            constexpr int st = decltype(ST)::value;
            if constexpr (!AHEAD) {
                load(std::integral_constant<int, st>{}, 0);
                if constexpr (S > 2) load(std::integral_constant<int, (st + 1) % S>{}, BK);
                if constexpr (S > 3) load(std::integral_constant<int, (st + 2) % S>{}, 2 * BK);
            }
            wait_vm<(S - 2) * LPS>();
            asm volatile("s_barrier" ::: "memory");
            read(ST, 0, 0);
        };
        using I0 = std::integral_constant<int, 0>;
        using I1 = std::integral_constant<int, 1>;
        using I2 = std::integral_constant<int, 2>;
        using I3 = std::integral_constant<int, 3>;
        if (r == 0) begin(I0{});
        else if (r == 1) begin(std::integral_constant<int, S - 1>{});
        else if constexpr (S > 2) {
            if (r == 2) begin(std::integral_constant<int, S - 2>{});
            else if constexpr (S > 3) begin(I1{});
        }
        int k0 = 0;
        if constexpr (S > 3) {
            if (r == 3) { slab(I1{}, k0); k0 += BK; }
        }
        if constexpr (S > 2) {
            if (r >= 2) { slab(std::integral_constant<int, S - 2>{}, k0); k0 += BK; }
        }
        if (r >= 1) { slab(std::integral_constant<int, S - 1>{}, k0); k0 += BK; }
#pragma clang loop unroll(disable)
        for (; k0 < slabs * BK; k0 += S * BK) {
            slab(I0{}, k0);
            slab(I1{}, k0 + BK);
            if constexpr (S > 2) slab(I2{}, k0 + 2 * BK);
            if constexpr (S > 3) slab(I3{}, k0 + 3 * BK);
        }
    }

    // The first slab of a product of two stages, into the stage that run takes it from.
    template <class LP, class LQ>
    __device__ __forceinline__ void ahead(LP lds_p, LQ lds_q, const Side &p, const Side &q, int kb, int slabs) {
        static_assert(S == 2, "one slab ahead");
        auto load = [&](auto ST) __attribute__((always_inline)) {
            sp.load(lds_p(ST), wave, p.base, p.ld, p.rows, p.width, kb, p.kend);
            sq.load(lds_q(ST), wave, q.base, q.ld, q.rows, q.width, kb, q.kend);
        };
        if (slabs % S) load(std::integral_constant<int, 1>{});
        else load(std::integral_constant<int, 0>{});
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int x = 0; x < 16; ++x) acc[i][j][x] = 0.0f;
    }
};

}  // namespace msr
