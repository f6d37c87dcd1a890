// Embedding: y[i] = s W[id[i]], and its gradient by sorted tokens,
//     dW[v] = s sum_{i: id[i] = v} dy[i],   stored whole (0 for words without a token) or added to an accumulator with SR.
// An id outside [0, vocab) has no word: its y is 0 and it gives no gradient.  The padding id gives none either.
//
// The tokens are sorted by word, earlier tokens first: runs of SORT_RUN tokens by one work-group each (a radix sort in
// LDS), then merged, MERGE_WAYS runs at a time.  Waves then take 16 or 32 sorted tokens each and add up the rows of one word after
// the other in fp32, so that no sum depends on a race.  A word whose tokens lie in one chunk is finished there; of a word that
// crosses chunks each leaves a part, which join_rows_kernel adds up, in an order that the ids alone give.  Rows of dW without a token
// are written by the launch of the sums, found by a search in the sorted tokens.  Up to FEW tokens are not sorted: the wave of a
// word's first token finds the others itself, one launch instead of three.
#include "rows.hpp"
#include "../../include/muon_sr_amd.h"

namespace msr {

constexpr int SORT_THREADS = 1024, SORT_EACH = 2, SORT_RUN = SORT_THREADS * SORT_EACH;
constexpr int SORT_LOG = 11, MERGE_LOG = 5, MERGE_WAYS = 1 << MERGE_LOG;
static_assert(SORT_RUN == 1 << SORT_LOG, "runs are searched by halves");
constexpr int SORT_WAVES = SORT_THREADS / 64, SORT_BITS = 9;    // bits of a pass at most
// Sorted tokens of a wave: 32 where the words are many, whose zeroing is most of a whole dW's work, else 16, which shortens each wave's
// chain of rows (us of sums and join with 32 and with 16: 16384 tokens, 128256 words of 4096, all of dW written, 216 and 235; 32000 words
// of 2048, written 38 and 45, accumulated 40 and 34).  The same for a stored gradient and an accumulated one: their sums have the same
// bits.
constexpr int CHUNK_MIN = 16, CHUNK_MAX = 32;
// Tokens that are not sorted, at most.  us of accumulating 500 tokens, sorted and not: of 2000 words of 512 20 and 9; of 4096, half of them
// padding, 23 and 31; all of one word, which one wave adds up, FEW_AHEAD rows in flight, 18 and 55.  1000 tokens of one word would take
// 110 us of a pass (sorted 50).
constexpr int FEW = 512, FEW_AHEAD = 16;

// Rows are written past the caches: a batch's y, and a whole dW, are larger than they (16384 tokens, 128256 words of 4096: lookup
// 52 us with cached stores, 36 so; gradient 218 and 213).
struct EmbedArgs {
    const void *ids;
    const void *w;               // [vocab][d]
    void *out;                   // y, dW or the accumulator
    const void *dy;              // [n] rows of lddy elements
    int64_t lddy;
    uint64_t *sorted;            // word << 32 | token; a token without a word has word = vocab
    float *parts;                // [chunks][2][d]: what a chunk adds to the word it shares with the one before, and begins for the one after
    int64_t n, d, padding;
    int32_t vocab, i64, zero_init, bits, chunk;
    float scale;
    Noise ns;
};

__device__ __forceinline__ int word_at(const EmbedArgs &a, int64_t i) {
    const int64_t v = a.i64 ? static_cast<const int64_t *>(a.ids)[i] : static_cast<const int32_t *>(a.ids)[i];
    return v >= 0 && v < a.vocab ? (int)v : -1;
}

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------

constexpr int LOOK_U = 4;        // 16-byte cells of a lane: a wave moves 4 KiB of a row

template <typename T>
__global__ __launch_bounds__(256) void lookup_kernel(EmbedArgs a) {
    using C = Cells<T>;
    constexpr int WIDTH = 64 * C::N * LOOK_U;
    const int lane = threadIdx.x & 63;
    const int64_t pieces = (a.d + WIDTH - 1) / WIDTH, jobs = a.n * pieces;
    for (int64_t j = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); j < jobs; j += (int64_t)gridDim.x * 4) {
        const int64_t i = pieces == 1 ? j : j / pieces, c0 = (j - i * pieces) * WIDTH + lane * C::N;
        const int v = __builtin_amdgcn_readfirstlane(word_at(a, i));
        C x[LOOK_U];
#pragma unroll
        for (int u = 0; u < LOOK_U; ++u) {
            const int64_t c = c0 + u * 64 * C::N;
            if (v >= 0 && c < a.d) x[u].load(static_cast<const T *>(a.w) + (int64_t)v * a.d, c, a.d);
            else x[u].v = Bytes16{};
        }
#pragma unroll
        for (int u = 0; u < LOOK_U; ++u) {
            const int64_t c = c0 + u * 64 * C::N;
            if (c >= a.d) continue;
            if (a.scale != 1.0f) {
                float f[C::N];
                x[u].get(f);
#pragma unroll
                for (int e = 0; e < C::N; ++e) f[e] *= a.scale;
                x[u].set(f);
            }
            x[u].template store<true>(static_cast<T *>(a.out) + i * a.d, c, a.d);
        }
    }
}

// ---------------------------------------------------------------------------
// tokens sorted by word
// ---------------------------------------------------------------------------

// One run: passes over the bits of the word, lowest first.  In a pass each wave ranks its 64 x rounds tokens 64 at a
// time by ballots, as every lane with the same digit before it counts; the counts of the waves and digits, added up
// in order, give each its place.
__global__ __launch_bounds__(SORT_THREADS) void sort_kernel(EmbedArgs a) {
    __shared__ uint32_t words[SORT_RUN];
    __shared__ uint16_t tokens[SORT_RUN];                        // their numbers in the run
    __shared__ uint16_t at[SORT_WAVES << SORT_BITS];             // [SORT_WAVES][digits]
    __shared__ int wave_sum[SORT_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t first = (int64_t)blockIdx.x * SORT_RUN;
    const int n = (int)min((int64_t)SORT_RUN, a.n - first), rounds = (n + SORT_THREADS - 1) / SORT_THREADS, run = 64 * rounds;
    const int passes = (a.bits + SORT_BITS - 1) / SORT_BITS, bits = (a.bits + passes - 1) / passes, digits = 1 << bits;
    uint32_t word[SORT_EACH];
    uint32_t token[SORT_EACH];       // and, above bit 15, its rank in a pass
#pragma unroll
    for (int r = 0; r < SORT_EACH; ++r) {
        const int i = wave * run + r * 64 + lane;
        token[r] = i;
        word[r] = ~0u;
        if (r < rounds && i < n) {
            const int v = word_at(a, first + i);
            word[r] = v < 0 || v == a.padding ? a.vocab : v;
        }
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * bits;
        for (int i = tid; i < SORT_WAVES * digits; i += SORT_THREADS) at[i] = 0;
        __syncthreads();
        uint16_t *const mine = at + wave * digits;
#pragma unroll
        for (int r = 0; r < SORT_EACH; ++r) {
            const bool on = r < rounds && wave * run + r * 64 + lane < n;   // (the places behind the last token are never filled)
            if (r >= rounds) continue;
            const int digit = (word[r] >> shift) & (digits - 1);
            uint64_t same = __ballot(on);
            for (int b = 0; b < bits; ++b) {
                const uint64_t m = __ballot((digit >> b) & 1);
                same &= (digit >> b) & 1 ? m : ~m;
            }
            const int before = __popcll(same & ((1ull << lane) - 1));
            const uint32_t rank = on ? mine[digit] + before : 0;
            token[r] = (token[r] & 0xffffu) | rank << 16;
            // a wave's LDS accesses execute in order: every lane has read the count before the last one of a
            // digit moves it on
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (on && (same >> lane) == 1) mine[digit] = (uint16_t)(rank + 1);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        __syncthreads();
        // digit `tid`: its tokens in the waves before each, after those of lower digits
        int count = 0, c[SORT_WAVES];
        if (tid < digits) {
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) c[w] = at[w * digits + tid];
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) count += c[w];
        }
        const int to = wave_scan(count);
        if (lane == 63) wave_sum[wave] = to;
        __syncthreads();
        int from = to - count;
        for (int w = 0; w < wave; ++w) from += wave_sum[w];
        if (tid < digits) {
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) {
                at[w * digits + tid] = (uint16_t)from;
                from += c[w];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SORT_EACH; ++r) {
            if (r < rounds && wave * run + r * 64 + lane < n) {
                const int to_at = mine[(word[r] >> shift) & (digits - 1)] + (int)(token[r] >> 16);
                words[to_at] = word[r];
                tokens[to_at] = (uint16_t)token[r];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SORT_EACH; ++r) {
            const int i = wave * run + r * 64 + lane;
            if (r < rounds && i < n) {
                word[r] = words[i];
                token[r] = tokens[i];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < SORT_EACH; ++r) {
        const int i = wave * run + r * 64 + lane;
        if (r < rounds && i < n) a.sorted[first + i] = (uint64_t)word[r] << 32 | (uint64_t)(first + token[r]);
    }
}

// How many of the n ascending keys are below `key`
__device__ __forceinline__ int64_t below(const uint64_t *keys, int64_t n, uint64_t key) {
    int64_t lo = 0;
    while (n > 0) {
        const int64_t half = n >> 1;
        if (keys[lo + half] < key) {
            lo += half + 1;
            n -= half + 1;
        } else {
            n = half;
        }
    }
    return lo;
}

// Runs of `run` keys (a power of two), MERGE_WAYS at a time, merged: a key's place is its own number in its run plus how many of
// each other are below it.  A search in memory is a chain of loads, so every work-group holds each stride-th key of its group of
// runs in LDS, searches there first and in memory among the last `stride` only, in four runs at once; the searches are chains all the same,
// so four threads share those of a key (us with the whole search in memory by one thread, with the LDS, and so: 16384 tokens 17, 12, 7;
// 60000 tokens 45 with the LDS, 16 so).
constexpr int MERGE_HELD = 8192, MERGE_KEYS = 256, MERGE_SHARES = 4;
__global__ __launch_bounds__(MERGE_KEYS * MERGE_SHARES) void merge_kernel(const uint64_t *in, uint64_t *out, int64_t n, int log_run) {
    constexpr int AT_ONCE = 4, THREADS = MERGE_KEYS * MERGE_SHARES;
    __shared__ uint64_t held[MERGE_HELD];
    __shared__ int64_t below[MERGE_SHARES][MERGE_KEYS];
    const int share = threadIdx.x / MERGE_KEYS, own = threadIdx.x % MERGE_KEYS;
    const int64_t i = (int64_t)blockIdx.x * MERGE_KEYS + own, run = (int64_t)1 << log_run;
    const int log_group = log_run + MERGE_LOG;
    const int64_t first = ((int64_t)blockIdx.x * MERGE_KEYS) >> log_group << log_group, end = min(first + ((int64_t)1 << log_group), n);
    const uint64_t key = i < n ? in[i] : 0;
    int log_stride = 3;
    while ((end - first) >> log_stride > MERGE_HELD) ++log_stride;
    const int log_per = log_run - log_stride, keys = (int)((end - first) >> log_stride), all = (int)((end - first + run - 1) >> log_run) << log_per;
    for (int k = threadIdx.x; k < min(all, MERGE_HELD); k += THREADS) held[k] = k < keys ? in[first + ((int64_t)(k + 1) << log_stride) - 1] : ~0ull;
    __syncthreads();
    const int64_t mine = i >> log_run << log_run;
    int64_t place = 0;
    for (int64_t r0 = first + share * run; r0 < end; r0 += AT_ONCE * MERGE_SHARES * run) {
        int64_t lo[AT_ONCE], len[AT_ONCE];
        int k[AT_ONCE] = {};
        const int base = (int)((r0 - first) >> log_run) << log_per;
#pragma unroll
        for (int y = 0; y < AT_ONCE; ++y) {
            const int64_t r = r0 + y * MERGE_SHARES * run;
            len[y] = r == mine || i >= n ? 0 : max((int64_t)0, min(run, end - r));
        }
        for (int step = 1 << log_per; step; step >>= 1) {
#pragma unroll
            for (int y = 0; y < AT_ONCE; ++y)
                if (k[y] + step <= (int)(len[y] >> log_stride) && held[base + (y * MERGE_SHARES << log_per) + k[y] + step - 1] < key) k[y] += step;
        }
#pragma unroll
        for (int y = 0; y < AT_ONCE; ++y) lo[y] = (int64_t)k[y] << log_stride;
        for (int64_t step = (int64_t)1 << (log_stride - 1); step; step >>= 1) {
#pragma unroll
            for (int y = 0; y < AT_ONCE; ++y)
                if (lo[y] + step <= len[y] && in[r0 + y * MERGE_SHARES * run + lo[y] + step - 1] < key) lo[y] += step;
        }
#pragma unroll
        for (int y = 0; y < AT_ONCE; ++y) place += lo[y];
    }
    below[share][own] = place;
    __syncthreads();
    if (share || i >= n) return;
    for (int s = 1; s < MERGE_SHARES; ++s) place += below[s][own];
    out[first + (i - mine) + place] = key;
}

// ---------------------------------------------------------------------------
// sums
// ---------------------------------------------------------------------------

constexpr int SUM_AHEAD = 4, JOIN_AHEAD = 8;     // rows, and parts, whose loads are in flight together

// What is done with the sum of a word's rows, N columns from c on: stored in T (MODE -1), or added to the bf16 accumulator
// with SR as round(scale sum) would be by msr_sr_accum.
template <typename T, int MODE>
__device__ __forceinline__ void finish(const EmbedArgs &a, int v, int64_t c, const float (&sum)[Cells<T>::N]) {
    using C = Cells<T>;
    C x;
    float f[C::N];
#pragma unroll
    for (int e = 0; e < C::N; ++e) f[e] = sum[e] * a.scale;
    x.set(f);
    T *const row = static_cast<T *>(a.out) + (int64_t)v * a.d;
    if constexpr (MODE >= 0) {
        const int64_t o0 = (int64_t)v * a.d + c;
        const int valid = (int)min((int64_t)8, a.d - c);
        C old;
        old.v = Bytes16{};
        if (!a.zero_init) old.load(row, c, a.d);
        uint32_t rn[8], o[4];
        if (o0 % 8 == 0) {
            noise8<MODE>(a.ns, o0, valid, rn);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) rn[e] = e < valid ? noise1<MODE>(a.ns, o0 + e) : 0u;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
            o[q] = pack2(sr_bf16(bf16_lo(old.v.w[q]) + bf16_lo(x.v.w[q]), rn[2 * q]), sr_bf16(bf16_hi(old.v.w[q]) + bf16_hi(x.v.w[q]), rn[2 * q + 1]));
        x.v = Bytes16{{o[0], o[1], o[2], o[3]}};
    }
    x.template store<true>(row, c, a.d);
}

// Words that a wave looks up and zeroes where no token has them: 64, or 8 where that leaves waves idle (512 words of 256: 18 us
// and 8).
constexpr int zero_words(int64_t vocab, int64_t pieces) { return vocab * pieces >= 64 * 4096 ? 64 : 8; }

template <typename T>
__device__ __forceinline__ void zero_rows(const EmbedArgs &a, int64_t v0, uint64_t none, int64_t c) {
    Cells<T> zero;
    zero.v = Bytes16{};
    for (; none; none &= none - 1)
        if (c < a.d) zero.template store<true>(static_cast<T *>(a.out) + (v0 + __builtin_ctzll(none)) * a.d, c, a.d);
}

// floats [c, c + N) of a part of d
template <int N>
__device__ __forceinline__ void load_part(const float *part, int64_t c, int64_t d, float (&f)[N]) {
    Cells<float> x[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) x[i].load(part, c + 4 * i, d);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = __uint_as_float(x[e / 4].v.w[e % 4]);
}
template <int N>
__device__ __forceinline__ void store_part(float *part, int64_t c, int64_t d, const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        Cells<float> x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x.v.w[e] = __float_as_uint(f[4 * i + e]);
        x.store(part, c + 4 * i, d);
    }
}

// Job j: chunk j / pieces of the sorted tokens and a piece of 64 cells of their rows; behind those, `words` words that
// are looked up and, where no token has them, zeroed.
template <typename T, int MODE>
__global__ __launch_bounds__(256) void sums_kernel(EmbedArgs a, int64_t sum_jobs, int64_t zero_jobs, int words) {
    using C = Cells<T>;
    constexpr int WIDTH = 64 * C::N;
    const int lane = threadIdx.x & 63;
    int64_t j = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t pieces = (a.d + WIDTH - 1) / WIDTH;
    if (j >= sum_jobs) {
        j -= sum_jobs;
        if (j >= zero_jobs) return;
        const int64_t v0 = j / pieces * words, v = v0 + lane;
        bool hit = lane >= words || v >= a.vocab;
        if (!hit) {
            const int64_t at = below(a.sorted, a.n, (uint64_t)v << 32);
            hit = at < a.n && (int64_t)(a.sorted[at] >> 32) == v;
        }
        zero_rows<T>(a, v0, ~__ballot(hit), (j % pieces) * WIDTH + lane * C::N);
        return;
    }
    const int64_t chunk = j / pieces, p0 = chunk * a.chunk, c = (j % pieces) * WIDTH + lane * C::N;
    const int count = (int)min((int64_t)a.chunk, a.n - p0);
    // lane l: token l of the chunk; the words before and after it
    const uint64_t key = lane < count ? a.sorted[p0 + lane] : ~0ull;
    const int word = (int)(key >> 32), token = (int)(uint32_t)key;
    const int prev = p0 > 0 ? __builtin_amdgcn_readfirstlane((int)(a.sorted[p0 - 1] >> 32)) : -1;
    const int next = p0 + count < a.n ? __builtin_amdgcn_readfirstlane((int)(a.sorted[p0 + count] >> 32)) : -1;
    const uint64_t held = __ballot(lane < count && word < a.vocab);     // a prefix: tokens without a word are last
    const int m = __popcll(held);     // (lanes beyond the row go along: their tokens are read by the others)
    float sum[C::N] = {};
    bool whole = m > 0 && __builtin_amdgcn_readlane(word, 0) != prev;   // the word at hand begins in this chunk
    for (int i0 = 0; i0 < m; i0 += SUM_AHEAD) {
        C x[SUM_AHEAD];
#pragma unroll
        for (int y = 0; y < SUM_AHEAD; ++y)
            if (i0 + y < m) x[y].load(static_cast<const T *>(a.dy) + (int64_t)__builtin_amdgcn_readlane(token, i0 + y) * a.lddy, c, a.d);
#pragma unroll
        for (int y = 0; y < SUM_AHEAD; ++y) {
            const int i = i0 + y;
            if (i >= m) break;
            float f[C::N];
            x[y].get(f);
#pragma unroll
            for (int e = 0; e < C::N; ++e) sum[e] += f[e];
            const int v = __builtin_amdgcn_readlane(word, i), after = i + 1 < count ? __builtin_amdgcn_readlane(word, i + 1) : next;
            const bool last = i + 1 == m;
            if (!last && after == v) continue;
            if (whole && after != v) {
                finish<T, MODE>(a, v, c, sum);
            } else {
                store_part(a.parts + (2 * chunk + (whole ? 1 : 0)) * a.d, c, a.d, sum);
            }
            whole = true;
#pragma unroll
            for (int e = 0; e < C::N; ++e) sum[e] = 0.0f;
        }
    }
}

// Words that cross chunks: a work-group takes a piece of 64 cells of the words that begin in four chunks, one to a wave.  A word of many
// chunks (one of the four at most), whose parts are a chain of loads, is shared by the work-group: every fourth part to a wave, the
// waves' sums added in order (60000 tokens of 1000 words of 512, of which one has a tenth: 52 us by one wave, 20 so; 13399 tokens of
// 970 words of 20: 32 and 13).
template <typename T, int MODE>
__global__ __launch_bounds__(256) void join_rows_kernel(EmbedArgs a) {
    using C = Cells<T>;
    constexpr int N = C::N, WIDTH = 64 * N;
    __shared__ int64_t many[4];                        // parts of a shared word; 0 where the wave's word is none
    __shared__ float sums[4][64][N + 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t chunks = (a.n + a.chunk - 1) / a.chunk, groups = (chunks + 3) / 4, first = blockIdx.x % groups * 4;
    const int64_t c = blockIdx.x / groups * WIDTH + lane * N;
    auto at = [&](int64_t p) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane((int)(a.sorted[p] >> 32)); };
    // the chunks from `chunk` on that hold the word that crosses its end, if that begins in it
    auto parts_of = [&](int64_t chunk) __attribute__((always_inline)) -> int64_t {
        if (chunk + 1 >= chunks) return 0;
        const int v = at((chunk + 1) * a.chunk);
        if (v >= a.vocab || at((chunk + 1) * a.chunk - 1) != v) return 0;                    // no word crosses
        if (chunk > 0 && at(chunk * a.chunk) == v && at(chunk * a.chunk - 1) == v) return 0;   // it began before
        int64_t end = chunk + 1;                       // chunks that begin with the word
        for (;;) {
            const int64_t k = end + lane;
            const uint64_t same = __ballot(k < chunks && (int)(a.sorted[k * a.chunk] >> 32) == v);
            end += same == ~0ull ? 64 : __builtin_ctzll(~same);
            if (same != ~0ull) return end - chunk;
        }
    };
    // parts from, from + step, .. of n, JOIN_AHEAD loads in flight
    auto add = [&](int64_t chunk, int64_t from, int64_t step, int64_t n, float (&sum)[N]) __attribute__((always_inline)) {
        for (int64_t k = from; k < n && c < a.d; k += JOIN_AHEAD * step) {
            float f[JOIN_AHEAD][N];
#pragma unroll
            for (int y = 0; y < JOIN_AHEAD; ++y) {
                const int64_t i = min(k + y * step, n - 1);
                load_part(a.parts + (2 * (chunk + i) + (i == 0 ? 1 : 0)) * a.d, c, a.d, f[y]);
            }
#pragma unroll
            for (int y = 0; y < JOIN_AHEAD; ++y)
#pragma unroll
                for (int e = 0; e < N; ++e) sum[e] = k + y * step < n ? sum[e] + f[y][e] : sum[e];
        }
    };
    const int64_t chunk = first + wave, n = parts_of(chunk);
    if (n > 0 && n <= JOIN_AHEAD) {
        float sum[N] = {};
        add(chunk, 0, 1, n, sum);
        if (c < a.d) finish<T, MODE>(a, at((chunk + 1) * a.chunk), c, sum);
    }
    if (lane == 0) many[wave] = n > JOIN_AHEAD ? n : 0;
    __syncthreads();
    for (int q = 0; q < 4; ++q) {
        const int64_t nq = many[q];
        if (nq == 0) continue;
        float sum[N] = {};
        add(first + q, wave, 4, nq, sum);
#pragma unroll
        for (int e = 0; e < N; ++e) sums[wave][lane][e] = sum[e];
        __syncthreads();
        if (wave == q && c < a.d) {
#pragma unroll
            for (int e = 0; e < N; ++e) sum[e] = ((sums[0][lane][e] + sums[1][lane][e]) + sums[2][lane][e]) + sums[3][lane][e];
            finish<T, MODE>(a, at((chunk + 1) * a.chunk), c, sum);
        }
        __syncthreads();
    }
}

// At most FEW tokens, not sorted.  Job j: token j / pieces, if it is the first of its word, with the others of that word;
// behind those, 8 words that are zeroed where no token has them.  Every wave holds all ids, 64 to a register.
template <typename T, int MODE>
__global__ __launch_bounds__(256) void few_kernel(EmbedArgs a, int64_t sum_jobs, int64_t zero_jobs) {
    using C = Cells<T>;
    constexpr int WIDTH = 64 * C::N, R = FEW / 64;
    const int lane = threadIdx.x & 63;
    int64_t j = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t pieces = (a.d + WIDTH - 1) / WIDTH;
    if (j >= sum_jobs + zero_jobs) return;
    int word[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        word[r] = -1;
        if (r * 64 + lane < a.n) word[r] = word_at(a, r * 64 + lane);
        if (word[r] == a.padding) word[r] = -1;
    }
    if (j >= sum_jobs) {
        j -= sum_jobs;
        const int v0 = (int)(j / pieces * 8);
        uint64_t none = 0;
        for (int i = 0; i < 8 && v0 + i < a.vocab; ++i) {
            bool hit = false;
#pragma unroll
            for (int r = 0; r < R; ++r) hit |= word[r] == v0 + i;
            none |= (uint64_t)(__ballot(hit) == 0) << i;
        }
        zero_rows<T>(a, v0, none, (j % pieces) * WIDTH + lane * C::N);
        return;
    }
    const int i = (int)(j / pieces);
    const int64_t c = (j % pieces) * WIDTH + lane * C::N;
    int v = -1;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (i / 64 == r) v = __builtin_amdgcn_readlane(word[r], i % 64);
    if (v < 0) return;
    uint64_t same[R];
    bool first = true;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        same[r] = __ballot(word[r] == v);
        if (r < i / 64) first = first && same[r] == 0;
        if (r == i / 64) first = first && (same[r] & ((1ull << (i % 64)) - 1)) == 0;
    }
    if (!first) return;
    float sum[C::N] = {};
#pragma unroll 1
    for (int r = i / 64; r < R; ++r) {
        uint64_t left = 0;
#pragma unroll
        for (int q = 0; q < R; ++q) left = q == r ? same[q] : left;
        while (left) {
            C x[FEW_AHEAD];
            bool on[FEW_AHEAD];
#pragma unroll
            for (int y = 0; y < FEW_AHEAD; ++y) {
                on[y] = left != 0;
                if (on[y]) x[y].load(static_cast<const T *>(a.dy) + (int64_t)(r * 64 + __builtin_ctzll(left)) * a.lddy, c, a.d);
                left &= left - 1;
            }
#pragma unroll
            for (int y = 0; y < FEW_AHEAD; ++y) {
                if (!on[y]) continue;
                float f[C::N];
                x[y].get(f);
#pragma unroll
                for (int e = 0; e < C::N; ++e) sum[e] += f[e];
            }
        }
    }
    finish<T, MODE>(a, v, c, sum);
}

// ---------------------------------------------------------------------------

struct EmbedPlan {
    int runs, merges;
    size_t sorted, parts, bytes;     // bytes of one list of sorted tokens, and of the parts
};
static EmbedPlan embed_plan(int64_t n, int64_t d) {
    EmbedPlan p{};
    p.runs = (int)((n + SORT_RUN - 1) / SORT_RUN);
    for (int64_t r = 1; r < p.runs; r *= MERGE_WAYS) ++p.merges;
    if (n <= FEW) return p;
    p.sorted = ((size_t)n * 8 + 255) & ~(size_t)255;
    p.parts = (size_t)((n + CHUNK_MIN - 1) / CHUNK_MIN) * 2 * (size_t)d * 4;
    p.bytes = p.sorted * (p.merges ? 2 : 1) + p.parts;
    return p;
}

static int embed_check(const char *name, int64_t n, int64_t vocab, int64_t d, int32_t elem) {
    if (n < 0 || n >= (1 << 28) || vocab < 1 || vocab >= (1 << 27) || d < 0 || d > (1 << 20) || (elem != MSR_BF16 && elem != MSR_F32)) {
        set_error("%s: need fewer than 2^28 tokens, 1 to 2^27 - 1 words, rows of at most 2^20 elements and bf16 or fp32 (got %lld tokens, "
                  "%lld words of %lld, type %d)", name, (long long)n, (long long)vocab, (long long)d, (int)elem);
        return MSR_ERR_ARG;
    }
    return MSR_OK;
}

template <typename T, int MODE>
static int embed_sums(EmbedArgs a, hipStream_t s) {
    constexpr int WIDTH = 64 * Cells<T>::N;
    const int64_t pieces = (a.d + WIDTH - 1) / WIDTH;
    const bool few = a.n <= FEW, zero = MODE < 0 || a.zero_init;
    a.chunk = a.vocab >= 4 * a.n ? CHUNK_MAX : CHUNK_MIN;
    const int64_t chunks = (a.n + a.chunk - 1) / a.chunk;
    const int words = few ? 8 : zero_words(a.vocab, pieces);
    const int64_t sums = (few ? a.n : chunks) * pieces, zeros = zero ? ((int64_t)a.vocab + words - 1) / words * pieces : 0;
    const dim3 grid((unsigned)((sums + zeros + 3) / 4));
    if (few) {
        if (sums + zeros > 0) hipLaunchKernelGGL((few_kernel<T, MODE>), grid, dim3(256), 0, s, a, sums, zeros);
        return check_launch("few_kernel");
    }
    if (sums + zeros > 0) {
        hipLaunchKernelGGL((sums_kernel<T, MODE>), grid, dim3(256), 0, s, a, sums, zeros, words);
        const int rc = check_launch("sums_kernel");
        if (rc || chunks < 2) return rc;
        hipLaunchKernelGGL((join_rows_kernel<T, MODE>), dim3((unsigned)((chunks + 3) / 4 * pieces)), dim3(256), 0, s, a);
    }
    return check_launch("join_rows_kernel");
}

// MODE -2: decided by the arguments
static int embed_grad(const char *name, const void *ids, int32_t ids_i64, int64_t n, const void *dy, int64_t lddy, int64_t vocab, int64_t d,
                      float scale, int64_t padding, void *out, int32_t elem, int32_t noise_mode, uint32_t seed, int32_t zero_init,
                      const uint16_t *inject, void *workspace, size_t workspace_bytes, hipStream_t s) {
    int rc = embed_check(name, n, vocab, d, elem);
    if (rc) return rc;
    if ((n > 0 && d > 0 && (!ids || !dy)) || (d > 0 && !out) || lddy < d || lddy > (int64_t(1) << 40) || noise_mode < -1 || noise_mode > 2 ||
        (noise_mode == NOISE_INJECT && !inject)) {
        set_error("%s: bad arguments", name);
        return MSR_ERR_ARG;
    }
    const size_t es = elem_bytes(elem);
    if (!aligned(ids, ids_i64 ? 8 : 4) || !aligned(dy, es) || !aligned(out, es) || !aligned(inject, 2) || !aligned(workspace, 8)) {
        set_error("%s: operands must be aligned to their types, the workspace to 8 bytes", name);
        return MSR_ERR_ALIGN;
    }
    const EmbedPlan p = embed_plan(n, d);
    if (p.bytes > 0 && d > 0 && (!workspace || workspace_bytes < p.bytes)) {
        set_error("%s: workspace of %zu bytes is smaller than the %zu required", name, workspace_bytes, p.bytes);
        return MSR_ERR_WORKSPACE;
    }
    const size_t wb = (size_t)vocab * (size_t)d * es;
    const Range r[5] = {{out, wb}, {workspace, p.bytes}, {ids, (size_t)n * (ids_i64 ? 8 : 4)}, {dy, rows_bytes(n, lddy, d, es)},
                        {inject, noise_mode == NOISE_INJECT ? wb : 0}};
    rc = ranges_apart(name, r, 5, 2);
    if (rc || d == 0) return rc;
    const int64_t pieces = (d + 64 * (16 / (int64_t)es) - 1) / (64 * (16 / (int64_t)es));
    const int64_t words = n <= FEW ? 8 : zero_words(vocab, pieces);
    const int64_t waves = ((n <= FEW ? n : (n + CHUNK_MIN - 1) / CHUNK_MIN) + (vocab + words - 1) / words) * pieces;   // at most
    if (waves >= (int64_t(1) << 26) - 4) {          // 64 threads each: fewer than 2^32 in a launch
        set_error("%s: too many rows for a launch (%lld tokens, %lld words of %lld)", name, (long long)n, (long long)vocab, (long long)d);
        return MSR_ERR_ARG;
    }
    EmbedArgs a{};
    a.ids = ids; a.i64 = ids_i64 != 0; a.n = n; a.dy = dy; a.lddy = lddy; a.vocab = (int32_t)vocab; a.d = d; a.scale = scale;
    a.padding = padding; a.out = out; a.zero_init = zero_init != 0;
    a.ns.key = seed_key(seed, 0);
    a.ns.inject = inject;
    if (n > FEW) {
        char *const ws = static_cast<char *>(workspace);
        uint64_t *list[2] = {reinterpret_cast<uint64_t *>(ws), reinterpret_cast<uint64_t *>(ws + p.sorted)};
        a.parts = reinterpret_cast<float *>(ws + p.sorted * (p.merges ? 2 : 1));
        a.sorted = list[0];
        while ((int64_t(1) << a.bits) <= vocab) ++a.bits;               // words 0 to vocab
        hipLaunchKernelGGL(sort_kernel, dim3((unsigned)p.runs), dim3(SORT_THREADS), 0, s, a);
        if ((rc = check_launch("sort_kernel"))) return rc;
        for (int m = 0; m < p.merges; ++m) {
            hipLaunchKernelGGL(merge_kernel, dim3((unsigned)((n + MERGE_KEYS - 1) / MERGE_KEYS)), dim3(MERGE_KEYS * MERGE_SHARES), 0, s,
                               list[m & 1], list[~m & 1], n, SORT_LOG + m * MERGE_LOG);
            if ((rc = check_launch("merge_kernel"))) return rc;
            a.sorted = list[~m & 1];
        }
    }
    if (noise_mode < 0) return elem == MSR_BF16 ? embed_sums<uint16_t, -1>(a, s) : embed_sums<float, -1>(a, s);
    MSR_DISPATCH_NOISE(noise_mode, MODE, return (embed_sums<uint16_t, MODE>(a, s)));
    return MSR_OK;
}

}  // namespace msr

using namespace msr;

extern "C" {

int msr_embedding(const void *ids, int32_t ids_i64, int64_t n, const void *w, int64_t vocab, int64_t d, float scale, void *y,
                  int32_t elem, msr_stream_t stream) {
    const char *const name = "msr_embedding";
    int rc = embed_check(name, n, vocab, d, elem);
    if (rc || n == 0 || d == 0) return rc;
    if (!ids || !w || !y) { set_error("%s: a pointer is NULL", name); return MSR_ERR_ARG; }
    const size_t es = elem_bytes(elem);
    if (!aligned(ids, ids_i64 ? 8 : 4) || !aligned(w, es) || !aligned(y, es)) {
        set_error("%s: operands must be aligned to their types", name);
        return MSR_ERR_ALIGN;
    }
    const Range r[3] = {{y, (size_t)n * (size_t)d * es}, {ids, (size_t)n * (ids_i64 ? 8 : 4)}, {w, (size_t)vocab * (size_t)d * es}};
    rc = ranges_apart(name, r, 3, 1);
    if (rc) return rc;
    EmbedArgs a{};
    a.ids = ids; a.i64 = ids_i64 != 0; a.n = n; a.w = w; a.vocab = (int32_t)vocab; a.d = d; a.scale = scale; a.out = y;
    const int64_t width = 64 * (16 / (int64_t)es) * LOOK_U, jobs = n * ((d + width - 1) / width);
    const dim3 grid(grid_for(jobs, 4, 256 * 64));
    if (elem == MSR_BF16) hipLaunchKernelGGL(lookup_kernel<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(lookup_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, a);
    return check_launch("lookup_kernel");
}

int msr_embedding_workspace_bytes(int64_t n, int64_t vocab, int64_t d, size_t *bytes) {
    const int rc = embed_check("msr_embedding_workspace_bytes", n, vocab, d, MSR_BF16);
    if (rc) return rc;
    if (!bytes) { set_error("msr_embedding_workspace_bytes: a pointer is NULL"); return MSR_ERR_ARG; }
    *bytes = embed_plan(n, d).bytes;
    return MSR_OK;
}

int msr_embedding_grad(const void *ids, int32_t ids_i64, int64_t n, const void *dy, int64_t lddy, int64_t vocab, int64_t d, float scale,
                       int64_t padding, void *dw, int32_t elem, void *workspace, size_t workspace_bytes, msr_stream_t stream) {
    return embed_grad("msr_embedding_grad", ids, ids_i64, n, dy, lddy, vocab, d, scale, padding, dw, elem, -1, 0, 0, nullptr, workspace,
                      workspace_bytes, (hipStream_t)stream);
}

int msr_embedding_grad_sr_accum(const void *ids, int32_t ids_i64, int64_t n, const uint16_t *dy, int64_t lddy, int64_t vocab, int64_t d,
                                float scale, int64_t padding, uint16_t *acc, uint32_t seed, int32_t zero_init, int32_t noise_mode,
                                const uint16_t *inject, void *workspace, size_t workspace_bytes, msr_stream_t stream) {
    if (noise_mode < 0) { set_error("msr_embedding_grad_sr_accum: bad noise_mode %d", (int)noise_mode); return MSR_ERR_ARG; }
    return embed_grad("msr_embedding_grad_sr_accum", ids, ids_i64, n, dy, lddy, vocab, d, scale, padding, acc, MSR_BF16, noise_mode, seed,
                      zero_init, inject, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
