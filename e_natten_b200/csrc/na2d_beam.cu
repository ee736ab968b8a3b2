// Beam search (include/na2d.h): the choice among all beams' next words, and caches that follow their beams.
//
// Choice.  Candidate (i, w) of a batch entry is worth  scores_i + logits_iw - ln sum_w e^logits_iw.
// Bound by memory: the logits are read once, by select_rows_kernel: a block takes a segment of one beam's words in chunks, the next one under
// way, every thread with a running maximum and sum of exponentials of its own, and finds the best words without sorting: with r =
// ceil(count / 8), the least of the eight warps' r-th largest thread maxima is a bound that at least `count` words reach and few more do;
// those go to shared memory, where at the end each counts the better ones.  The bound is formed anew behind 1, 2, 4 ... chunks.
// select_beams_kernel joins an entry's segments: sums in 64 bits, candidates by the same bound.  (value, lowest beam, lowest word) is a
// total order, so nothing depends on the order in which candidates arrive.  What a block keeps has room for 512: where more words reach
// the bound (equal ones, ascending ones; all of 513 to 1792 in 16 bits, 513 to 896 in 32, which leave a warp without a word and the bound at
// nothing) it looks for the best below the last one, `count` times over.
// Measured: 64 x 8 x 131072 fp32, 268 MB: 55 us, 74 % of the copy bandwidth (the rows 53, issue slots 54 %); 7 x 5 x 100003 fp16, rows on odd
// places, 15 us, of which the rows are 8 and the joining 6; 16 x 4 x 32768 bf16 10.6, the host's time of the call.
//
// Reordering.  cache[g K + i] <- cache[g K + parent_gi] for all beams of a group at once, in place: a thread has the same few bytes of
// all K beams, reads what moves and then writes it, so that no second copy of a cache exists and beams that keep their place cost
// nothing.  Bound by memory: each beam that others follow is read once, each entry that moves written once.  Blocks of all
// groups come in the order of their part of a beam, so that those behind the end of short groups, which have nothing to do, come last.
// Measured: 16 caches of 32 x 8 x 2048 x 128, bf16, groups of four at 512 to 2048 tokens, two followed: 340 us for 2.0 GB, 91 % of the copy
// bandwidth (one piece a thread under way, and a source read for each that takes it: 425).
#include <algorithm>

#include "../../include/na2d.h"
#include "na2d_host.h"
#include "na2d_launch.h"
#include "na2d_ptx.cuh"
#include "na2d_vec.cuh"

namespace {

using na2d_vec::Vec;
using na2d_vec::widen;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMostBeams = 32, kMostCount = 64;
constexpr int kKept = 512;                              // candidates of a block that are ranked by counting
constexpr float kInf = __builtin_huge_valf();

// ---- choice ---------------------------------------------------------------------------------------------------------------
// Numbers in the order of floats; 0 is below all of them.
__device__ __forceinline__ unsigned ordered(float x) {
    const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(unsigned u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ unsigned long long ordered(double x) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(x == 0.0 ? 0.0 : x);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double from_ordered(unsigned long long u) {
    return __longlong_as_double((long long)(u >> 63 ? u & 0x7fffffffffffffffull : ~u));
}

// The r-th largest of a warp's 32 numbers, equal ones counted one by one.
__device__ __forceinline__ unsigned nth_largest(unsigned x, int r) {
    unsigned top = 0;
    for (int i = 0; i < r; ++i) {
        top = __reduce_max_sync(0xffffffffu, x);
        const unsigned at = __ballot_sync(0xffffffffu, x == top);
        if ((threadIdx.x & 31) == __ffs(at) - 1) x = 0;
    }
    return top;
}

// A bound that at least `count` of the block's numbers reach (0 where there are fewer), from each thread's largest.  Every thread calls.
__device__ __forceinline__ unsigned bound_of(unsigned largest, int count, unsigned* warps) {
    const unsigned own = nth_largest(largest, (count + kWarps - 1) / kWarps);
    if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = own;
    __syncthreads();
    unsigned least = warps[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) least = min(least, warps[w]);
    return least;
}

// The same for counts of at most 32, the best of the warps' bounds.
__device__ __forceinline__ unsigned best_bound_of(unsigned largest, int count, unsigned* warps) {
    const unsigned own = nth_largest(largest, count);
    if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = own;
    __syncthreads();
    unsigned most = warps[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) most = max(most, warps[w]);
    return most;
}

struct Select {
    const void* logits;
    long long stride_b, stride_k;
    const float* scores;                // (B, K)
    const unsigned char* finished;      // (B, K), or null
    int B, K, V, count;
    long long end;
    int segments, each;                 // of a row, words of one
    float2* sums;                       // (B K, segments): maximum, sum of e^(logit - maximum)
    unsigned long long* best;           // (B K, segments, count): ordered logit, ~word; 0 where there is none
    float* out_scores;
    long long *out_parents, *out_words;
};

// e^x for x <= 0, off by 2^-22 and, x times 1 / ln 2 in one number of 32 bits being off by 2^-24 and 1.4e-8 of itself, by (2^-24 + 2^-26) x.
// With x rounded to 32 bits, too, a row's logarithm is off by 2.25 times 2^-24 of its words' mean distance from the largest (13.2 at most
// of 2^24 words), 2^-22 for each of 17 factors and 2^-24 for each of 52 roundings: 2^-16.8.  Found: 2^-20.6, one word before tails of
// equal ones 0.1 to 20 below it.
constexpr float kLog2e = 1.44269502f;
__device__ __forceinline__ float exp2_of(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float exp_of(float x) { return exp2_of(x * kLog2e); }
// The largest of three that is a number.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

constexpr int kEach = 16;                               // words that a thread has of a chunk
constexpr int kChunk = kThreads * kEach;

// N words a load, 1 where rows do not start on 16-byte boundaries.  Which thread has a word, and when, depends on the word and N
// alone, so that equal rows have equal sums.
template <typename T, int N>
struct Piece {
    Vec<T, N> part[kEach / N];
    // words at + [0, kEach) of a row's `words`, N at a time, a chunk's threads side by side
    __device__ __forceinline__ void load(const T* src, int chunk, int words) {
#pragma unroll
        for (int j = 0; j < kEach / N; ++j) {
            const int at = chunk * kChunk + (j * kThreads + (int)threadIdx.x) * N;
            if (at + N <= words) {
                part[j].load(src + at);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) part[j].at[i] = at + i < words ? src[at + i] : na2d_vec::narrow<T>(-kInf);
            }
        }
    }
};

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) select_rows_kernel(const Select x) {
    __shared__ unsigned warps[kWarps];
    __shared__ float tops[kWarps], totals[kWarps];
    __shared__ unsigned long long kept[kKept];
    __shared__ int kept_count;
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    const int row = blockIdx.x / x.segments, segment = blockIdx.x - row * x.segments, b = row / x.K, k = row - b * x.K;
    if (x.finished && x.finished[row]) return;           // (nothing of it is read)
    const int first = segment * x.each, words = min(x.each, x.V - first), tid = threadIdx.x;
    const T* src = static_cast<const T*>(x.logits) + b * x.stride_b + k * x.stride_k + first;
    const int chunks = (words + kChunk - 1) / kChunk;
    auto key_of = [&](int chunk, int j, float v) {
        const int word = first + chunk * kChunk + ((j / N) * kThreads + tid) * N + j % N;
        return ((unsigned long long)ordered(v) << 32) | (unsigned)~word;
    };
    Piece<T, N> next;
    next.load(src, 0, words);
    if (tid == 0) kept_count = 0;
    float high = -kInf, total = 0.f, least = -kInf;      // this thread's maximum and sum; what the block's best reach
    int renew = 1;                                       // the bound is formed anew behind that many chunks
    for (int c = 0; c < chunks; ++c) {
        float v[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) v[j] = widen(next.part[j / N].at[j % N]);
        if (c + 1 < chunks) next.load(src, c + 1, words);
        float most = -kInf;
#pragma unroll
        for (int j = 0; j < kEach; j += 2) most = max3(most, v[j], v[j + 1]);
        if (most > high) {
            total *= exp_of(high - most);                // (from -infinity on: a sum of nothing)
            high = most;
        }
        const float base = high == -kInf ? 0.f : high;
        // (two at a time: half the issue slots of all but the exponentials)
        const uint64_t less = na2d_ptx::pair2(-base, -base), by = na2d_ptx::pair2(kLog2e, kLog2e);
        uint64_t sum = 0;
#pragma unroll
        for (int j = 0; j < kEach; j += 2) {
            const uint64_t y = na2d_ptx::mul2(na2d_ptx::add2(na2d_ptx::pair2(v[j], v[j + 1]), less), by);
            sum = na2d_ptx::add2(sum, na2d_ptx::pair2(exp2_of(na2d_ptx::lo2(y)), exp2_of(na2d_ptx::hi2(y))));
        }
        total += na2d_ptx::lo2(sum) + na2d_ptx::hi2(sum);
        if (c + 1 == renew) {
            __syncthreads();                             // (`warps` has been read)
            const unsigned bound = bound_of(high == -kInf ? 0u : ordered(high), x.count, warps);
            least = bound ? from_ordered(bound) : -kInf;
            renew *= 2;
        }
        if (most >= least) {
#pragma unroll
            for (int j = 0; j < kEach; ++j)
                if (v[j] >= least && v[j] > -kInf) {
                    const int at = atomicAdd(&kept_count, 1);
                    if (at < kKept) kept[at] = key_of(c, j, v[j]);
                }
        }
    }
    {   // the block's maximum and sum
        float top = high;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (tid % 32 == 0) tops[tid / 32] = top;
        __syncthreads();
        top = tops[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, tops[w]);
        total *= high == -kInf ? 1.f : exp_of(high - top);       // (a NaN among words of -infinity stays one)
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
        if (tid % 32 == 0) totals[tid / 32] = total;
        high = top;
    }
    __syncthreads();
    const size_t place = (size_t)row * x.segments + segment;
    unsigned long long* best = x.best + place * x.count;
    const int n = kept_count;
    if (tid == 0) {
        total = 0.f;
        for (int w = 0; w < kWarps; ++w) total += totals[w];
        x.sums[place] = make_float2(high, total);
    }
    if (n <= kKept) {
        for (int i = tid; i < n; i += kThreads) {
            const unsigned long long own = kept[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += kept[j] > own;
            if (rank < x.count) best[rank] = own;
        }
        for (int i = n + tid; i < x.count; i += kThreads) best[i] = 0;
        return;
    }
    // many words reach the bound (equal ones, ascending ones): the best of those below the last one, `count` times
    unsigned long long below = ~0ull;
    for (int r = 0; r < x.count; ++r) {
        unsigned long long own = 0;
        for (int c = 0; c < chunks; ++c) {
            next.load(src, c, words);
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const float v = widen(next.part[j / N].at[j % N]);
                const unsigned long long key = v > -kInf ? key_of(c, j, v) : 0;
                if (key < below && key > own) own = key;
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) own = max(own, __shfl_xor_sync(0xffffffffu, own, d));
        __syncthreads();
        if (tid % 32 == 0) kept[tid / 32] = own;
        __syncthreads();
        below = kept[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) below = max(below, kept[w]);
        if (tid == 0) best[r] = below;                   // (n > count: there is one)
    }
}

// A block an entry.
__global__ void __launch_bounds__(kThreads) select_beams_kernel(const Select x) {
    // scores_i - ln sum_w e^(logits_iw - top_i), and top_i, which a logit's difference goes before all else (exact, whatever their size);
    // NaN: the beam has no candidates
    __shared__ double offset[kMostBeams];
    __shared__ float tops[kMostBeams];
    __shared__ unsigned warps[kWarps];
    __shared__ unsigned long long kept[kKept];
    __shared__ long long names[kKept];                   // beam V + word
    __shared__ int kept_count;
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid % 32;
    const int lists = x.K * x.segments, n = lists * x.count;
    const unsigned long long* best = x.best + (size_t)b * n;
    auto key_at = [&](int c) { return best[(size_t)(c % lists) * x.count + c / lists]; };
    // a thread's candidates are own_c, own_c + 256, ...; the keys of the first few are on their way meanwhile
    constexpr int kHeld = 4;
    const bool by_warp = x.count <= 32;
    const int own_c = by_warp ? tid : tid % kWarps * 32 + tid / kWarps;
    unsigned long long held[kHeld];
    long long names_held[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        held[u] = own_c + u * kThreads < n ? key_at(own_c + u * kThreads) : 0;
        names_held[u] = 0;
    }
    const double nan = __longlong_as_double(0x7ff8000000000000ll);
    for (int i = tid / 32; i < x.K; i += kWarps) {
        const int row = b * x.K + i;
        const float score = x.scores[row];
        const bool counts = score > -kInf && score < kInf;
        if (x.finished && x.finished[row]) {
            if (lane == 0) offset[i] = nan;
            continue;
        }
        const float2* sums = x.sums + (size_t)row * x.segments;
        float top = -kInf;
        for (int s = lane; s < x.segments; s += 32) top = fmaxf(top, sums[s].x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        double total = 0.0;
        for (int s = lane; s < x.segments; s += 32) {
            const float2 part = sums[s];
            total += (double)part.y * (part.x == -kInf ? 1.0 : exp((double)part.x - (double)top));       // (a sum of nothing is 0, or NaN)
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
        if (lane == 0) {
            offset[i] = counts && total > 0.0 ? (double)score - log(total) : nan;
            tops[i] = top;
        }
    }
    if (tid == 0) kept_count = 0;
    __syncthreads();
    // worth of candidate c (0: none) and its name, from its key.  Candidates lie list after list, a list a segment's best; c counts through all
    // lists' first ones, then their second ones.
    auto worth = [&](int c, unsigned long long key, long long& name) -> unsigned long long {
        const int list = c % lists, i = list / x.segments;
        const double by = offset[i];
        if (!(by == by)) {
            const int row = b * x.K + i;
            if (c != i * x.segments || !x.finished || !x.finished[row]) return 0;
            const float score = x.scores[row];           // a beam that has ended: itself
            name = (long long)i * x.V + x.end;
            return score > -kInf && score < kInf ? ordered((double)score) : 0;
        }
        if (!key) return 0;
        name = (long long)i * x.V + (unsigned)~(unsigned)key;
        return ordered(by + ((double)from_ordered((unsigned)(key >> 32)) - (double)tops[i]));
    };
    unsigned high = 0;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        held[u] = own_c + u * kThreads < n ? worth(own_c + u * kThreads, held[u], names_held[u]) : 0;
        high = max(high, (unsigned)(held[u] >> 32));
    }
    long long name = 0;
    for (int c = own_c + kHeld * kThreads; c < n; c += kThreads) high = max(high, (unsigned)(worth(c, key_at(c), name) >> 32));
    // (up to 32 candidates: a warp's `count`-th largest is a bound by itself, and the warp of the lists' first ones has a good one)
    const unsigned bound = max(by_warp ? best_bound_of(high, x.count, warps) : bound_of(high, x.count, warps), 1u);
    auto keep = [&](unsigned long long own, long long called) {
        if ((unsigned)(own >> 32) < bound) return;
        const int at = atomicAdd(&kept_count, 1);
        if (at >= kKept) return;
        kept[at] = own;
        names[at] = called;
    };
    if (high >= bound) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) keep(held[u], names_held[u]);
        for (int c = own_c + kHeld * kThreads; c < n; c += kThreads) {
            const unsigned long long own = worth(c, key_at(c), name);
            keep(own, name);
        }
    }
    __syncthreads();
    const int m = kept_count;
    auto put = [&](int r, unsigned long long own, long long called) {
        const size_t at = (size_t)b * x.count + r;
        x.out_scores[at] = own ? (float)from_ordered(own) : -kInf;
        x.out_parents[at] = own ? called / x.V : 0;
        x.out_words[at] = own ? called % x.V : 0;
    };
    if (m <= kKept) {
        for (int i = tid; i < m; i += kThreads) {
            int rank = 0;
            for (int j = 0; j < m; ++j) rank += kept[j] > kept[i] || (kept[j] == kept[i] && names[j] < names[i]);
            if (rank < x.count) put(rank, kept[i], names[i]);
        }
        for (int i = m + tid; i < x.count; i += kThreads) put(i, 0, 0);
        return;
    }
    // many of nearly equal worth: the best behind the last one, `count` times
    unsigned long long last = ~0ull;
    long long last_name = -1;
    for (int r = 0; r < x.count; ++r) {
        unsigned long long own = 0;
        long long called = 0;
        auto take = [&](unsigned long long w, long long who) {
            if (w > own || (w == own && w && who < called)) {
                own = w;
                called = who;
            }
        };
        for (int c = tid; c < n; c += kThreads) {
            const unsigned long long w = worth(c, key_at(c), name);
            if (w < last || (w == last && name > last_name)) take(w, name);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const unsigned long long w = __shfl_xor_sync(0xffffffffu, own, d);
            const long long who = __shfl_xor_sync(0xffffffffu, called, d);
            take(w, who);
        }
        __syncthreads();
        if (lane == 0) {
            kept[tid / 32] = own;
            names[tid / 32] = called;
        }
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) take(kept[w], names[w]);
        last = own;
        last_name = called;
        if (tid == 0) put(r, own, called);
    }
}

// Segments of a row: so many chunks each, up to 16, as give all SMs their four blocks.  A block that lives long has its loads under way for more of
// its time: 64 x 8 rows of 131072 words in fp32 take 55 us with 16 chunks a block (1024 blocks), 63 with 7.
struct Cut {
    int segments, each;                 // each: words of one
};
Cut cut_of(int rows, int V, int sms) {
    const long long chunks = (V + kChunk - 1) / kChunk, of_block = std::max(1LL, std::min(16LL, rows * chunks / (4LL * sms)));
    Cut c;
    c.segments = (int)((chunks + of_block - 1) / of_block);
    c.each = ((V + c.segments - 1) / c.segments + 7) / 8 * 8;
    c.segments = (V + c.each - 1) / c.each;
    return c;
}
size_t bytes_of(int rows, const Cut& c, int count) { return (size_t)rows * c.segments * (sizeof(float2) + sizeof(unsigned long long) * count); }

int check_select(const na2d_beam_select_args* a) {
    if (!a || a->struct_size < sizeof(na2d_beam_select_args)) return NA2D_ERR_BAD_ARG;
    if (a->B <= 0 || a->K <= 0 || a->V <= 0 || a->count <= 0 || a->end < 0 || a->end >= a->V) return NA2D_ERR_BAD_ARG;
    if (a->dtype != NA2D_F32 && a->dtype != NA2D_BF16 && a->dtype != NA2D_F16) return NA2D_ERR_UNSUPPORTED;
    if (a->K > kMostBeams || a->count > kMostCount) return NA2D_ERR_UNSUPPORTED;
    if (a->V > (1 << 24) || (long long)a->B * a->K > (1 << 20)) return NA2D_ERR_TOO_LARGE;
    return NA2D_OK;
}

template <typename T, int N>
int launch_rows(const Select& x, const Cut& c, cudaStream_t st) {
    const cudaError_t e = na2d_launch::launch(true, select_rows_kernel<T, N>, (unsigned)((long long)x.B * x.K * c.segments), kThreads, 0, st, x);
    return e == cudaSuccess ? NA2D_OK : na2d_host::cuda_fail(e, "beam selection launch");
}
template <typename T>
int by_alignment(const Select& x, const Cut& c, cudaStream_t st) {
    constexpr int kFull = 16 / (int)sizeof(T);
    const bool aligned = reinterpret_cast<uintptr_t>(x.logits) % 16 == 0 && x.stride_b % kFull == 0 && x.stride_k % kFull == 0;
    return aligned ? launch_rows<T, kFull>(x, c, st) : launch_rows<T, 1>(x, c, st);
}

// ---- reordering -----------------------------------------------------------------------------------------------------------
constexpr int kMostCaches = 64;                         // of a launch
struct Cache {
    char* at;
    long long e, h, t;                  // strides, bytes
    int heads, tokens, pieces;          // pieces: of a row
    int heads_first;                    // heads lie closer together than tokens
};
struct Reorder {
    Cache cache[kMostCaches];
    int B, K;
    const void* parents;                // (B, K)
    const void* lengths;                // (B K,), or null
    int parents_64, lengths_64;
    int blocks;                         // of a group
};

// V: the piece that a thread has of every beam, kPieces of them under way at once.
constexpr int kRuns = 8;                                // of 256 pieces, that a block takes
template <typename V, int MOST, int PIECES>
__global__ void __launch_bounds__(kThreads) reorder_kernel(const __grid_constant__ Reorder x) {
    __shared__ unsigned takers[kMostBeams];              // of a beam: bit i for beam i
    __shared__ int length[kMostBeams];
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    const Cache& c = x.cache[blockIdx.y];
    const int group = blockIdx.x % x.B, part = blockIdx.x / x.B;
    int longest = 0;                                     // of the beams that others follow (every warp by itself)
    {
        const int i = threadIdx.x & 31;
        int parent = i;
        if (i < x.K) {
            const size_t at = (size_t)group * x.K + i;
            const long long p = x.parents_64 ? static_cast<const long long*>(x.parents)[at] : static_cast<const int*>(x.parents)[at];
            parent = p >= 0 && p < x.K ? (int)p : i;     // (no such beam: it stays)
        }
        unsigned mine = 0;
        for (int k = 0; k < x.K; ++k) {
            const int of = __shfl_sync(0xffffffffu, parent, k);
            if (of == i && k != i) mine |= 1u << k;
        }
        int tokens = 0;
        if (mine) {
            const size_t at = (size_t)group * x.K + i;
            const long long n = !x.lengths ? c.tokens : x.lengths_64 ? static_cast<const long long*>(x.lengths)[at] : static_cast<const int*>(x.lengths)[at];
            tokens = (int)min(max(n, 0ll), (long long)c.tokens);
        }
        longest = __reduce_max_sync(0xffffffffu, tokens);
        if (threadIdx.x < 32) {
            takers[i] = mine;
            length[i] = tokens;
        }
    }
    const unsigned pieces = c.pieces, tokens = longest, heads = c.heads;
    const unsigned all = pieces * tokens * heads;        // (at most 2^30)
    const unsigned begin = part * (kRuns * kThreads), end = min(all, begin + kRuns * kThreads);
    if (begin >= all) return;
    __syncthreads();
    char* base = c.at + (long long)group * x.K * c.e;
    for (unsigned first = begin + threadIdx.x; first < end; first += PIECES * kThreads) {
        char* at[PIECES];
        int t[PIECES];
        V v[PIECES][MOST];
#pragma unroll
        for (int u = 0; u < PIECES; ++u) {
            const unsigned i = first + u * kThreads, row = i / pieces, p = i - row * pieces;
            unsigned h;
            if (c.heads_first) {
                t[u] = row / heads;
                h = row - t[u] * heads;
            } else {
                h = row / tokens;
                t[u] = row - h * tokens;
            }
            if (i >= end) t[u] = 0x7fffffff;             // no piece
            at[u] = base + h * c.h + t[u] * c.t + (long long)p * sizeof(V);
        }
#pragma unroll
        for (int k = 0; k < MOST; ++k)
            if (k < x.K && takers[k]) {
#pragma unroll
                for (int u = 0; u < PIECES; ++u)
                    if (t[u] < length[k]) v[u][k] = *reinterpret_cast<const V*>(at[u] + k * c.e);
            }
#pragma unroll
        for (int k = 0; k < MOST; ++k)
            for (unsigned left = k < x.K ? takers[k] : 0u; left; left &= left - 1) {
                const int i = __ffs(left) - 1;
#pragma unroll
                for (int u = 0; u < PIECES; ++u)
                    if (t[u] < length[k]) *reinterpret_cast<V*>(at[u] + i * c.e) = v[u][k];
            }
    }
}

// Bytes of the pieces that a cache's rows go in, and how many such pieces a beam has.
int piece_of(const na2d_cache& c) {
    const long long bits = (long long)reinterpret_cast<uintptr_t>(c.ptr) | c.stride_e | c.stride_h | c.stride_t | c.row_bytes;
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
}
long long pieces_of(const na2d_cache& c) { return c.row_bytes * c.heads * c.tokens / piece_of(c); }
long long reorder_blocks(long long pieces) { return (pieces + kRuns * kThreads - 1) / (kRuns * kThreads); }

template <typename V>
int launch_reorder(const Reorder& x, int caches, cudaStream_t st) {
    const dim3 grid((unsigned)(x.B * x.blocks), (unsigned)caches);
    auto kern = x.K <= 4 ? reorder_kernel<V, 4, 4> : x.K <= 8 ? reorder_kernel<V, 8, 2> : x.K <= 16 ? reorder_kernel<V, 16, 1> : reorder_kernel<V, 32, 1>;
    const cudaError_t e = na2d_launch::launch(true, kern, grid, kThreads, 0, st, x);
    if (e != cudaSuccess) return na2d_host::cuda_fail(e, "beam reordering launch");
    na2d_host::count_launches(1);
    return NA2D_OK;
}

}  // namespace

extern "C" {

size_t na2d_beam_select_workspace(const na2d_beam_select_args* a) {
    if (check_select(a) != NA2D_OK) return 0;
    return bytes_of(a->B * a->K, cut_of(a->B * a->K, a->V, na2d_host::sm_count(a->device)), a->count);
}

int na2d_beam_select(const na2d_beam_select_args* a) {
    if (int rc = check_select(a)) return rc;
    if (!a->logits || !a->scores || !a->out_scores || !a->out_parents || !a->out_words) return NA2D_ERR_BAD_ARG;
    Select x{};
    x.logits = a->logits;
    const bool dense = a->stride_b == 0 && a->stride_k == 0;
    x.stride_k = dense || a->K == 1 ? a->V : a->stride_k;
    x.stride_b = dense || a->B == 1 ? a->K * x.stride_k : a->stride_b;
    x.scores = a->scores;
    x.finished = a->finished;
    x.B = a->B;
    x.K = a->K;
    x.V = a->V;
    x.count = a->count;
    x.end = a->end;
    const int rows = a->B * a->K;
    const Cut c = cut_of(rows, a->V, na2d_host::sm_count(a->device));
    if (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 16 || a->workspace_bytes < bytes_of(rows, c, a->count)) return NA2D_ERR_BAD_ARG;
    if ((long long)rows * c.segments > 0x7fffffffLL || (long long)x.K * c.segments * x.count > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    x.segments = c.segments;
    x.each = c.each;
    x.best = static_cast<unsigned long long*>(a->workspace);
    x.sums = reinterpret_cast<float2*>(x.best + (size_t)rows * c.segments * a->count);
    x.out_scores = a->out_scores;
    x.out_parents = reinterpret_cast<long long*>(a->out_parents);
    x.out_words = reinterpret_cast<long long*>(a->out_words);
    return na2d_host::on_device(a->device, [&]() -> int {
        const cudaStream_t st = (cudaStream_t)a->stream;
        const int rc = a->dtype == NA2D_F32    ? by_alignment<float>(x, c, st)
                       : a->dtype == NA2D_BF16 ? by_alignment<__nv_bfloat16>(x, c, st)
                                               : by_alignment<__half>(x, c, st);
        if (rc != NA2D_OK) return rc;
        const cudaError_t e = na2d_launch::launch(true, select_beams_kernel, (unsigned)x.B, kThreads, 0, st, x);
        if (e != cudaSuccess) return na2d_host::cuda_fail(e, "beam selection launch");
        na2d_host::count_launches(2);
        return NA2D_OK;
    });
}

int na2d_beam_reorder(const na2d_beam_reorder_args* a) {
    if (!a || a->struct_size < sizeof(na2d_beam_reorder_args)) return NA2D_ERR_BAD_ARG;
    if (a->B <= 0 || a->K <= 0 || a->caches < 0 || (a->caches > 0 && !a->cache) || !a->parents) return NA2D_ERR_BAD_ARG;
    if (a->K > kMostBeams) return NA2D_ERR_UNSUPPORTED;
    if ((long long)a->B * a->K > (1 << 24)) return NA2D_ERR_TOO_LARGE;
    for (int i = 0; i < a->caches; ++i) {
        const na2d_cache& c = a->cache[i];
        if (!c.ptr || c.heads <= 0 || c.tokens <= 0 || c.row_bytes <= 0) return NA2D_ERR_BAD_ARG;
        if (c.row_bytes > (1ll << 40) / ((long long)c.heads * c.tokens)) return NA2D_ERR_TOO_LARGE;
        if (pieces_of(c) > 0x3fffffffLL || reorder_blocks(pieces_of(c)) * a->B > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    }
    if (!a->caches || a->K == 1) return NA2D_OK;
    return na2d_host::on_device(a->device, [&]() -> int {
        Reorder x{};
        x.B = a->B;
        x.K = a->K;
        x.parents = a->parents;
        x.lengths = a->lengths;
        x.parents_64 = a->parents_64 != 0;
        x.lengths_64 = a->lengths_64 != 0;
        // A launch has caches of one piece: a state of odd rows in the list leaves the others theirs.  Beside 2 GB of caches, 347 us, one of 13
        // int64 a beam: 351 us, 569 with the least piece for all; one of 13 bools: 352, 2111.
        for (const int piece : {16, 4, 1}) {
            int n = 0;
            auto launch = [&]() {
                const int caches = n;
                n = 0;
                return !caches       ? NA2D_OK
                       : piece == 16 ? launch_reorder<uint4>(x, caches, (cudaStream_t)a->stream)
                       : piece == 4  ? launch_reorder<uint32_t>(x, caches, (cudaStream_t)a->stream)
                                     : launch_reorder<uint8_t>(x, caches, (cudaStream_t)a->stream);
            };
            for (int i = 0; i < a->caches; ++i) {
                const na2d_cache& c = a->cache[i];
                if (piece_of(c) != piece) continue;
                if (n == 0) x.blocks = 0;
                x.blocks = std::max(x.blocks, (int)reorder_blocks(pieces_of(c)));
                x.cache[n++] = Cache{static_cast<char*>(c.ptr), c.stride_e, c.stride_h, c.stride_t, c.heads, c.tokens, (int)(c.row_bytes / piece),
                                     c.stride_h < c.stride_t};
                if (n == kMostCaches)
                    if (const int rc = launch()) return rc;
            }
            if (const int rc = launch()) return rc;
        }
        return NA2D_OK;
    });
}

}  // extern "C"
