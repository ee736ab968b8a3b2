// Group normalisation of channels-last maps with an activation, forward and backward (include/na2d.h).
//
//   forward    xhat = (x - mean) rstd,  z = xhat w + b,  y = act(z)
//   backward   dz = dy act'(z);  A_c = sum_p dz,  B_c = sum_p dz xhat  of a batch entry's channel;
//              s1 = sum_c w A,  s2 = sum_c w B  of a group;  dx = rstd (dz w - (s1 + xhat s2) / M),  M values a group;
//              db = sum_b A,  dw = sum_b B
//
// Bound by memory: x is read and y written, in the backward x and dy read and dx written; every value is needed for the statistics
// before the first can be written.  Two forms.
//
// On the chip: a slab of channels (whole groups, 64 bytes of a pixel where that many fit) of all pixels of a batch entry is copied to
// the shared memory of one block, or of a cluster of up to 8, each holding a share of the pixels, and read from there: global memory
// is read once.  Blocks of a cluster add their channel sums through distributed shared memory.
//
// In two passes, where a slab is too large for that, by one cooperative launch that walks sets of slabs: half of a block's threads take the
// sums of set i while the other half write set i - 1, so that neither's waits leave the memory idle.  Of what the second half reads
// again about a third is in L2 still.
//
// Measured, forward and backward (bytes at the copy bandwidth in brackets): 4 x 256^2 x 512 in 32 groups, bf16, in two passes: 149 + 221 us
// (206), memory at 4.4 TB/s; 16 x 14^2 x 1024, fp16, on the chip: 20 + 26 us with a cold L2 (5).  Forward, 2 x 97 x 131 x 384, fp16: 21 us (6).
//
// Variances are sums of squares about a mean at every step (of a slab; of four pixels, merged with those before), so that maps
// whose mean is far above their spread lose nothing.  All sums are in fp32 and in an order that the sizes alone fix; a thread of the two
// forms has some thousand values on maps of 2^20 pixels, one of the kernels for wide groups any number, which it sums with what rounding loses.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/na2d.h"
#include "na2d_host.h"
#include "na2d_launch.h"
#include "na2d_ptx.cuh"
#include "na2d_vec.cuh"

namespace {

using na2d_vec::Vec;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;

struct Map {                // a (B, P, C) operand
    const void* ptr;
    long long b, p;
};

struct Norm {
    int B, C, G, cg;        // batch, channels, groups, channels of a group
    long long P;
    float eps;
    Map x, d_y;
    void *y, *d_x;
    const void *w, *bias;   // null: ones, zeros
    int param_f32;
    float *mean, *rstd;     // (B, G)
};

template <typename T>
__device__ __forceinline__ float param(const Norm& n, const void* p, int c, float none) {
    return !p ? none : n.param_f32 ? __ldg(static_cast<const float*>(p) + c) : na2d_vec::widen(static_cast<const T*>(p)[c]);
}

// y = act(z), and its derivative
template <bool SILU>
__device__ __forceinline__ float activate(float z) {
    return SILU ? __fdividef(z, 1.f + __expf(-z)) : z;
}
template <bool SILU>
__device__ __forceinline__ float slope(float z) {
    if (!SILU) return 1.f;
    const float s = __fdividef(1.f, 1.f + __expf(-z));
    return s * fmaf(z, 1.f - s, 1.f);
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float of another block's shared memory at the place that `p` has in this one's.
__device__ __forceinline__ float peer_float(const float* p, uint32_t rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(na2d_ptx::smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(na2d_ptx::smem_u32(dst)), "l"(src) : "memory");
    else if constexpr (BYTES >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(na2d_ptx::smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
    else
        *static_cast<uint16_t*>(dst) = *static_cast<const uint16_t*>(src);
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ---- on the chip ---------------------------------------------------------------------------------------------------
// How a slab lies on a block: thread t has vector column t % cols_p2 (of `cols`) of pixels t / cols_p2, + rows, ...
struct Slab {
    int channels, slabs;            // of a slab; slabs of a batch entry
    int cols, cols_p2;
    int cluster;
    int pixels;                     // of a block at most
};

// Sums `v` of every channel over the threads of a block, then over the cluster; the result of channel c goes to total[c].
// red: kWarps * channels floats.  `part` is read by the cluster's other blocks: it may be written again after another cluster_sum.
template <int N>
__device__ __forceinline__ void cluster_sum(const Slab& s, float (&v)[N], float* red, float* part, float* total) {
    const int col = threadIdx.x % s.cols_p2, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int d = s.cols_p2; d < 32; d <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
    __syncthreads();                                 // red and total are free
    if (lane < s.cols_p2 && col < s.cols)
#pragma unroll
        for (int i = 0; i < N; ++i) red[warp * s.channels + col * N + i] = v[i];
    __syncthreads();
    float* own = s.cluster > 1 ? part : total;
    for (int c = threadIdx.x; c < s.channels; c += kThreads) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += red[w * s.channels + c];
        own[c] = sum;
    }
    if (s.cluster > 1) {
        cluster_sync();
        for (int c = threadIdx.x; c < s.channels; c += kThreads) {
            float sum = 0.f;
            for (int r = 0; r < s.cluster; ++r) sum += peer_float(part + c, r);
            total[c] = sum;
        }
    }
    __syncthreads();
}

// The sum of total[] over the group of channel c.
__device__ __forceinline__ float group_sum(const float* total, int c, int cg) {
    const float* at = total + c / cg * cg;
    float sum = 0.f;
    for (int i = 0; i < cg; ++i) sum += at[i];
    return sum;
}

template <typename T, int N, bool SILU>
__global__ void __launch_bounds__(kThreads) norm_chip_fwd_kernel(const Norm n, const Slab s) {
    extern __shared__ __align__(16) uint8_t smem_bytes[];
    uint8_t* smem = smem_bytes;
    T* data = reinterpret_cast<T*>(smem);
    float* red = reinterpret_cast<float*>(smem + ((size_t)s.pixels * s.channels * sizeof(T) + 15) / 16 * 16);
    float *part = red + kWarps * s.channels, *total = part + 2 * s.channels;        // part: one for each of the two sums
    const int rank = s.cluster > 1 ? (int)cluster_rank() : 0;
    const int at = blockIdx.x / s.cluster, b = at / s.slabs, c0 = (at - b * s.slabs) * s.channels;
    const int col = threadIdx.x % s.cols_p2, row = threadIdx.x / s.cols_p2, rows = kThreads / s.cols_p2;
    const long long p0 = (long long)rank * s.pixels;
    const int pixels = (int)max(0LL, min((long long)s.pixels, n.P - p0));
    const int c = col * N;                               // of the slab
    const bool active = col < s.cols;
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    if (active) {
        const T* src = static_cast<const T*>(n.x.ptr) + b * n.x.b + p0 * n.x.p + c0 + c;
        for (int p = row; p < pixels; p += rows) copy_async<N * sizeof(T)>(data + p * s.channels + c, src + p * n.x.p);
    }
    copies_done();                                       // (a thread reads what it copied itself)
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    if (active)
        for (int p = row; p < pixels; p += rows) {
            Vec<T, N> x;
            float f[N];
            x.load(data + p * s.channels + c);
            x.widened(f);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += f[i];
        }
    cluster_sum(s, v, red, part, total);
    const float inv_m = 1.f / ((float)n.P * n.cg);
    float mean[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        mean[i] = active ? group_sum(total, c + i, n.cg) * inv_m : 0.f;
        v[i] = 0.f;
    }
    if (active)
        for (int p = row; p < pixels; p += rows) {
            Vec<T, N> x;
            float f[N];
            x.load(data + p * s.channels + c);
            x.widened(f);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = fmaf(f[i] - mean[i], f[i] - mean[i], v[i]);
        }
    cluster_sum(s, v, red, part + s.channels, total);
    if (active) {
        float scale[N], shift[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float rstd = rsqrtf(fmaf(group_sum(total, c + i, n.cg), inv_m, n.eps));
            scale[i] = rstd * param<T>(n, n.w, c0 + c + i, 1.f);
            shift[i] = param<T>(n, n.bias, c0 + c + i, 0.f);
            if (rank == 0 && row == 0 && (c0 + c + i) % n.cg == 0) {
                n.mean[b * n.G + (c0 + c + i) / n.cg] = mean[i];
                n.rstd[b * n.G + (c0 + c + i) / n.cg] = rstd;
            }
        }
        T* dst = static_cast<T*>(n.y) + ((long long)b * n.P + p0) * n.C + c0 + c;
        for (int p = row; p < pixels; p += rows) {
            Vec<T, N> x;
            float f[N];
            x.load(data + p * s.channels + c);
            x.widened(f);
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = activate<SILU>(fmaf(f[i] - mean[i], scale[i], shift[i]));
            x.round(f);
            x.store(dst + (long long)p * n.C);
        }
    }
    if (s.cluster > 1) cluster_sync();                   // no block leaves while another reads its sums
}

// Per-channel values of the backward that a thread keeps.
template <typename T, int N>
struct Column {
    float mean[N], rstd[N], w[N], bias[N];
    __device__ __forceinline__ Column(const Norm& n, int b, int c) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int g = b * n.G + (c + i) / n.cg;
            mean[i] = n.mean[g];
            rstd[i] = n.rstd[g];
            w[i] = param<T>(n, n.w, c + i, 1.f);
            bias[i] = param<T>(n, n.bias, c + i, 0.f);
        }
    }
};

template <typename T, int N, bool SILU>
__global__ void __launch_bounds__(kThreads) norm_chip_bwd_kernel(const Norm n, const Slab s, float2* __restrict__ sums) {
    extern __shared__ __align__(16) uint8_t smem_bytes[];
    uint8_t* smem = smem_bytes;
    const size_t bytes = ((size_t)s.pixels * s.channels * sizeof(T) + 15) / 16 * 16;
    T *data = reinterpret_cast<T*>(smem), *grad = reinterpret_cast<T*>(smem + bytes);
    float* red = reinterpret_cast<float*>(smem + 2 * bytes);
    float *part = red + kWarps * s.channels, *total = part + 2 * s.channels;
    const int rank = s.cluster > 1 ? (int)cluster_rank() : 0;
    const int at = blockIdx.x / s.cluster, b = at / s.slabs, c0 = (at - b * s.slabs) * s.channels;
    const int col = threadIdx.x % s.cols_p2, row = threadIdx.x / s.cols_p2, rows = kThreads / s.cols_p2;
    const long long p0 = (long long)rank * s.pixels;
    const int pixels = (int)max(0LL, min((long long)s.pixels, n.P - p0));
    const bool active = col < s.cols;
    const int c = active ? col * N : 0;
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    if (active) {
        const T* x = static_cast<const T*>(n.x.ptr) + b * n.x.b + p0 * n.x.p + c0 + c;
        const T* g = static_cast<const T*>(n.d_y.ptr) + b * n.d_y.b + p0 * n.d_y.p + c0 + c;
        for (int p = row; p < pixels; p += rows) {
            copy_async<N * sizeof(T)>(data + p * s.channels + c, x + p * n.x.p);
            copy_async<N * sizeof(T)>(grad + p * s.channels + c, g + p * n.d_y.p);
        }
    }
    const Column<T, N> k(n, b, c0 + c);
    copies_done();
    float a[N], d[N];
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = d[i] = 0.f;
    if (active)
        for (int p = row; p < pixels; p += rows) {
            Vec<T, N> x, g;
            float f[N], e[N];
            x.load(data + p * s.channels + c);
            g.load(grad + p * s.channels + c);
            x.widened(f);
            g.widened(e);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float xhat = (f[i] - k.mean[i]) * k.rstd[i], dz = e[i] * slope<SILU>(fmaf(xhat, k.w[i], k.bias[i]));
                a[i] += dz;
                d[i] = fmaf(dz, xhat, d[i]);
            }
        }
    const float inv_m = 1.f / ((float)n.P * n.cg);
    float s1[N], s2[N];
    auto sum = [&](float (&v)[N], float* peers, float (&out)[N], int which) {
        cluster_sum(s, v, red, peers, total);
        if (sums && rank == 0)
            for (int i = threadIdx.x; i < s.channels; i += kThreads)
                reinterpret_cast<float*>(sums + (long long)b * n.C + c0 + i)[which] = total[i];
        __syncthreads();
        for (int i = threadIdx.x; i < s.channels; i += kThreads) total[i] *= param<T>(n, n.w, c0 + i, 1.f);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = group_sum(total, c + i, n.cg) * inv_m;
    };
    sum(a, part, s1, 0);
    sum(d, part + s.channels, s2, 1);
    if (active && n.d_x) {
        T* dst = static_cast<T*>(n.d_x) + ((long long)b * n.P + p0) * n.C + c0 + c;
        for (int p = row; p < pixels; p += rows) {
            Vec<T, N> x, g;
            float f[N], e[N];
            x.load(data + p * s.channels + c);
            g.load(grad + p * s.channels + c);
            x.widened(f);
            g.widened(e);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float xhat = (f[i] - k.mean[i]) * k.rstd[i], dz = e[i] * slope<SILU>(fmaf(xhat, k.w[i], k.bias[i]));
                f[i] = k.rstd[i] * (fmaf(dz, k.w[i], -s1[i]) - xhat * s2[i]);
            }
            x.round(f);
            x.store(dst + (long long)p * n.C);
        }
    }
    if (s.cluster > 1) cluster_sync();
}

// ---- in two passes -----------------------------------------------------------------------------------------------------
constexpr int kHalf = 256;                      // threads of a half

// A unit is a slab of channels (whole groups) of a batch entry; a set, `at_once` units.  A block has one run of pixels of a unit of every
// set.  All blocks are on the chip at once (a cooperative launch), and their halves wait for one another through counts in memory.
struct Pass {
    int slabs, channels;            // slabs of a batch entry; channels of a unit
    int cols, cols_p2;              // vector columns of a unit; thread t has column t % cols_p2 of pixels t / cols_p2, + rows, ...
    int groups;                     // of a unit
    long long run;                  // pixels
    int runs;
    int units, at_once, sets;
    float2* part;                   // [set % kBuffers][unit of the set][group][run]: the runs' values
    unsigned *summed, *written;     // [set]: blocks that are done with it
    unsigned* gave_up;              // a wait has: the others are short, then
    const na2d_ptx::ErrorState* errors;
};
// Sets that the sums may be ahead by: the next one's x comes in while the writing half still reads the last one's.
constexpr int kAhead = 2, kBuffers = kAhead + 1;
struct Set {
    int first, count;               // units
    float2* part;
};
// A block's run and unit of a set; its first half of threads sums, the second writes.
struct Role {
    int run, unit;
    bool writes;
    int tid, warp, lane;            // in the half
    __device__ __forceinline__ explicit Role(const Pass& s) {
        unit = blockIdx.x / s.runs;
        run = blockIdx.x - unit * s.runs;
        writes = threadIdx.x >= kHalf;
        tid = threadIdx.x % kHalf;
        warp = tid / 32;
        lane = tid % 32;
    }
    __device__ __forceinline__ void sync() const {
        __syncwarp();                   // (behind a poll that one lane ran)
        na2d_ptx::bar_sync(writes ? 2 : 1, kHalf);
    }
};
__device__ __forceinline__ Set set_of(const Pass& s, int i) {
    return Set{i * s.at_once, min(s.at_once, s.units - i * s.at_once), s.part + (long long)(i % kBuffers) * s.at_once * s.groups * s.runs};
}
// This half is done with what `count` counts.
__device__ __forceinline__ void arrive(const Role& role, unsigned* count) {
    role.sync();
    if (role.tid == 0) {
        __threadfence();
        atomicAdd(count, 1u);
    }
}
// Waits until that half of every block is; bounded, as every wait is.
__device__ __forceinline__ void wait_for(const Role& role, const Pass& s, const unsigned* count) {
    if (role.tid == 0) {
        const unsigned all = gridDim.x;
        auto value = [](const unsigned* p) {
            unsigned v;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
            return v;
        };
        const unsigned limit_us = s.errors->limit_us ? s.errors->limit_us : (unsigned)(na2d_ptx::kWaitLimitNs / 1000ull);
        bool done = false;
        for (unsigned k = 0; k < 4096 && !(done = value(count) == all); ++k) {}
        for (unsigned k = 0; k < limit_us && !done && value(s.gave_up) == 0; ++k) {
            __nanosleep(1000);
            done = value(count) == all;
        }
        if (!done) {
            atomicExch(s.gave_up, 1u);
            na2d_ptx::report_error(s.errors->error_bytes, na2d_ptx::kErrOther);
        }
    }
    role.sync();
}

// A warp's groups one after the other, `use(g, v)` with lane's values of group g's runs, lane, lane + 32, ...: the next group's come while one
// is used (each on its own was a chain of reads from L2, 8 us a set).
constexpr int kRunsLane = 8, kMostRuns = 32 * kRunsLane;
template <typename F>
__device__ __forceinline__ void each_group(const Role& role, const Pass& s, const float2* part, F&& use) {
    float2 v[kRunsLane], next[kRunsLane];
    auto fetch = [&](int g) {
#pragma unroll
        for (int j = 0; j < kRunsLane; ++j) {
            const int r = role.lane + 32 * j;
            next[j] = r < s.runs && g < s.groups ? __ldcg(part + (long long)g * s.runs + r) : make_float2(0.f, 0.f);
        }
    };
    fetch(role.warp);
    for (int g = role.warp; g < s.groups; g += kHalf / 32) {
#pragma unroll
        for (int j = 0; j < kRunsLane; ++j) v[j] = next[j];
        fetch(g + kHalf / 32);
        use(g, v);
    }
}

constexpr int kStage = 4;                       // pixels of a thread that are copied, and summed, together

// What a thread reads of a run passes through shared memory that is its own, copied there several stages ahead: enough bytes are under
// way for the memory's latency without a register for any of them, and no thread waits for another.
template <typename T, int N, int OPS, int DEPTH>
struct Stream {
    static constexpr int kVector = N * (int)sizeof(T), kPlace = kHalf * kVector, kStageBytes = kStage * OPS * kPlace;
    static constexpr int kBytes = DEPTH * kStageBytes;
    const T* src[OPS];              // the next pixel that is asked for
    long long step[OPS];            // from one of the thread's pixels to the next
    int left;                       // pixels that have not been asked for
    uint8_t *own, *at;              // [stage][pixel][operand][thread]: this thread's first, and the stage that is read next
    __device__ __forceinline__ void start(uint8_t* smem, int pixels) {
        own = at = smem + threadIdx.x % kHalf * kVector;
        left = pixels;
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) ask(own + d * kStageBytes);
    }
    __device__ __forceinline__ void ask(uint8_t* to) {
#pragma unroll
        for (int u = 0; u < kStage; ++u) {
            if (u < left)
#pragma unroll
                for (int op = 0; op < OPS; ++op) copy_async<kVector>(to + (u * OPS + op) * kPlace, src[op]);
#pragma unroll
            for (int op = 0; op < OPS; ++op) src[op] += step[op];
        }
        left -= kStage;
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // the next stage's vectors; then its place is asked for again
    __device__ __forceinline__ void take(Vec<T, N> (&v)[kStage][OPS]) {
        asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
#pragma unroll
        for (int u = 0; u < kStage; ++u)
#pragma unroll
            for (int op = 0; op < OPS; ++op) v[u][op].load(reinterpret_cast<const T*>(at + (u * OPS + op) * kPlace));
        ask(at);
        at = at + kStageBytes == own + kBytes ? own : at + kStageBytes;
    }
};
template <typename T, int N> using MapStream = Stream<T, N, 1, 5>;
template <typename T, int N> using GradStream = Stream<T, N, 2, 2>;


// N values in pairs (one value: a pair whose second is no value).
template <int N> struct Pairs {
    static constexpr int K = (N + 1) / 2;
    uint64_t at[K];
};
template <typename T>
__device__ __forceinline__ uint64_t widen_pair(uint32_t w) {
    if constexpr (sizeof(T) == 2) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return na2d_ptx::pair2(w << 16, w & 0xffff0000u);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        return na2d_ptx::pair2(f.x, f.y);
    }
    return 0;
}
template <typename T, int N>
__device__ __forceinline__ Pairs<N> widen_all(const Vec<T, N>& v) {
    Pairs<N> p;
    if constexpr (N == 1) {
        p.at[0] = na2d_ptx::pair2(na2d_vec::widen(v.at[0]), 0.f);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) p.at[i] = na2d_ptx::pair2(v.at[2 * i], v.at[2 * i + 1]);
    } else {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&v.bits);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) p.at[i] = widen_pair<T>(w[i]);
    }
    return p;
}
template <typename T, int N>
__device__ __forceinline__ void store_all(T* dst, const Pairs<N>& p) {
    Vec<T, N> v;
    if constexpr (N == 1) {
        v.at[0] = na2d_vec::narrow<T>(na2d_ptx::lo2(p.at[0]));
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float lo = na2d_ptx::lo2(p.at[i]), hi = na2d_ptx::hi2(p.at[i]);
            if constexpr (std::is_same<T, float>::value) {
                v.at[2 * i] = lo;
                v.at[2 * i + 1] = hi;
            } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                *reinterpret_cast<__nv_bfloat162*>(v.at + 2 * i) = __floats2bfloat162_rn(lo, hi);
            } else {
                *reinterpret_cast<__half2*>(v.at + 2 * i) = __floats2half2_rn(lo, hi);
            }
        }
    }
    v.store_streaming(dst);
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t both(float x) { return na2d_ptx::pair2(x, x); }
__device__ __forceinline__ uint64_t sigmoid2(uint64_t z) {
    using namespace na2d_ptx;
    const uint64_t t = mul2(z, both(-1.4426950408889634f));
    const uint64_t d = add2(pair2(exp2_approx(lo2(t)), exp2_approx(hi2(t))), both(1.f));
    return pair2(rcp_approx(lo2(d)), rcp_approx(hi2(d)));
}
template <bool SILU>
__device__ __forceinline__ uint64_t activate2(uint64_t z) {
    return SILU ? na2d_ptx::mul2(z, sigmoid2(z)) : z;
}
// g times the activation's derivative
template <bool SILU>
__device__ __forceinline__ uint64_t through2(uint64_t g, uint64_t z) {
    using namespace na2d_ptx;
    if (!SILU) return g;
    const uint64_t s = sigmoid2(z);
    return mul2(g, mul2(s, fma2(z, fma2(s, both(-1.f), both(1.f)), both(1.f))));
}

// A block's place: a run of pixels of a unit.
struct Spot {
    int unit, b, c0, col, row, rows;        // unit of the set; batch entry, first channel; this thread's column and first pixel
    long long p0, p1;
    int pixels;                             // of this thread
    __device__ __forceinline__ Spot(const Norm& n, const Pass& s, const Set& set, int unit_, long long run, int role_tid) {
        unit = unit_;
        const int u = set.first + unit;
        b = u / s.slabs;
        c0 = (u - b * s.slabs) * s.channels;
        col = role_tid % s.cols_p2;
        row = role_tid / s.cols_p2;
        rows = kHalf / s.cols_p2;
        p0 = run * s.run;
        p1 = min(n.P, p0 + s.run);
        const int all = (int)(p1 - p0) - row;
        pixels = col < s.cols && all > 0 ? (all + rows - 1) / rows : 0;
    }
    __device__ __forceinline__ long long first(const Map& m, int n) const { return b * m.b + (p0 + row) * m.p + c0 + col * n; }
};

// The merge of two sets of values: counts, means and sums of squares about them.
__device__ __forceinline__ void merge(float& count, float& mean, float& m2, float n, float mean_n, float m2_n) {
    if (n == 0.f) return;
    const float all = count + n, share = __fdividef(n, all), off = mean_n - mean;
    mean = fmaf(off, share, mean);
    m2 += fmaf(off * off, count * share, m2_n);
    count = all;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

// A thread's (count, mean, sum of squares about it) of its channels
template <typename T, int N>
__device__ __forceinline__ float take_stats(MapStream<T, N>& stream, const int pixels, Pairs<N>& mean, Pairs<N>& m2) {
    using namespace na2d_ptx;
    constexpr int K = Pairs<N>::K;
    float count = 0.f;
#pragma unroll
    for (int i = 0; i < K; ++i) mean.at[i] = m2.at[i] = 0;
    for (int k = 0; k < pixels; k += kStage) {
        Vec<T, N> x[kStage][1];
        stream.take(x);
        if (k + kStage <= pixels) {               // summed about their own mean, then merged
            const float share = __fdividef((float)kStage, count + kStage);
            const uint64_t share2 = both(share), weight2 = both(count * share);
            Pairs<N> f[kStage];
#pragma unroll
            for (int u = 0; u < kStage; ++u) f[u] = widen_all(x[u][0]);
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const uint64_t m = mul2(add2(add2(f[0].at[i], f[1].at[i]), add2(f[2].at[i], f[3].at[i])), both(1.f / kStage));
                const uint64_t minus = m ^ 0x8000000080000000ull;
                uint64_t q = m2.at[i];
#pragma unroll
                for (int u = 0; u < kStage; ++u) {
                    const uint64_t d = add2(f[u].at[i], minus);
                    q = fma2(d, d, q);
                }
                const uint64_t off = fma2(mean.at[i], both(-1.f), m);
                mean.at[i] = fma2(off, share2, mean.at[i]);
                m2.at[i] = fma2(mul2(off, off), weight2, q);
            }
            count += kStage;
        } else {
#pragma unroll
            for (int u = 0; u < kStage; ++u)
                if (k + u < pixels) {
                    const Pairs<N> f = widen_all(x[u][0]);
                    const float share = __fdividef(1.f, count + 1.f);
#pragma unroll
                    for (int i = 0; i < K; ++i) {
                        const uint64_t off = fma2(mean.at[i], both(-1.f), f.at[i]);
                        mean.at[i] = fma2(off, both(share), mean.at[i]);
                        m2.at[i] = fma2(mul2(off, off), both(count * share), m2.at[i]);
                    }
                    count += 1.f;
                }
        }
    }
    return count;
}

// Sums of a thread's channels -> red[row][channel].
template <int N>
__device__ __forceinline__ void put_rows(float2* red, const Spot& at, int channels, const Pairs<N>& u, const Pairs<N>& v) {
    using namespace na2d_ptx;
#pragma unroll
    for (int i = 0; i < N; ++i)
        red[at.row * channels + at.col * N + i] =
            make_float2(i % 2 ? hi2(u.at[i / 2]) : lo2(u.at[i / 2]), i % 2 ? hi2(v.at[i / 2]) : lo2(v.at[i / 2]));
}

// Per-channel constants of a thread: -mean, rstd w, bias.
template <int N>
struct Affine {
    Pairs<N> minus_mean, scale, shift;
    // `stats(c)`: mean and rstd of channel c of the unit
    template <typename T, typename F>
    __device__ __forceinline__ void read(const Norm& n, const Spot& at, F&& stats) {
#pragma unroll
        for (int i = 0; i < Pairs<N>::K; ++i) {
            float v[3][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = at.col * N + min(2 * i + e, N - 1);
                const float2 st = stats(c);
                v[0][e] = -st.x;
                v[1][e] = st.y * param<T>(n, n.w, at.c0 + c, 1.f);
                v[2][e] = param<T>(n, n.bias, at.c0 + c, 0.f);
            }
            minus_mean.at[i] = na2d_ptx::pair2(v[0][0], v[0][1]);
            scale.at[i] = na2d_ptx::pair2(v[1][0], v[1][1]);
            shift.at[i] = na2d_ptx::pair2(v[2][0], v[2][1]);
        }
    }
};

template <typename T, int N>
__device__ __forceinline__ void open_stream(MapStream<T, N>& stream, const Norm& n, const Spot& at, uint8_t* smem) {
    stream.src[0] = static_cast<const T*>(n.x.ptr) + at.first(n.x, N);
    stream.step[0] = at.rows * n.x.p;
    stream.start(smem, at.pixels);
}
template <typename T, int N>
__device__ __forceinline__ void open_stream(GradStream<T, N>& stream, const Norm& n, const Spot& at, uint8_t* smem) {
    stream.src[0] = static_cast<const T*>(n.x.ptr) + at.first(n.x, N);
    stream.src[1] = static_cast<const T*>(n.d_y.ptr) + at.first(n.d_y, N);
    stream.step[0] = at.rows * n.x.p;
    stream.step[1] = at.rows * n.d_y.p;
    stream.start(smem, at.pixels);
}
// This block's place in a set; one without a unit there has no pixels.
__device__ __forceinline__ Spot spot_in(const Norm& n, const Pass& s, const Role& role, int set) {
    const Set at = set_of(s, set);
    Spot spot(n, s, at, min(role.unit, at.count - 1), role.run, role.tid);
    if (role.unit >= at.count) spot.pixels = 0;
    return spot;
}

template <typename T, int N, bool SILU>
__global__ void __launch_bounds__(2 * kHalf, 1) norm_fwd_kernel(const Norm n, const Pass s) {
    using namespace na2d_ptx;
    constexpr int K = Pairs<N>::K;
    extern __shared__ __align__(16) uint8_t smem_all[];
    const Role role(s);
    uint8_t* smem = smem_all + (role.writes ? MapStream<T, N>::kBytes : 0);
    float2* red = reinterpret_cast<float2*>(smem_all + 2 * MapStream<T, N>::kBytes);     // sums: [row][channel]
    float* counts = reinterpret_cast<float*>(red + kHalf * N);                           // sums: [row]
    float2* stats = reinterpret_cast<float2*>(counts + kHalf);                           // writes: [group]
    const int warp = role.warp, lane = role.lane, channels = s.cols_p2 * N;
    MapStream<T, N> stream;
    Spot next = spot_in(n, s, role, 0);
    open_stream(stream, n, next, smem);
    for (int i = 0; i < s.sets; ++i) {
        const Set set = set_of(s, i);
        const Spot at = next;
        const bool mine = role.unit < set.count;
        if (i + 1 < s.sets) next = spot_in(n, s, role, i + 1);
        if (!role.writes) {
            Pairs<N> mean, m2;
            const float count = take_stats(stream, at.pixels, mean, m2);
            if (i >= kAhead) wait_for(role, s, s.written + i - kAhead);
            if (i + 1 < s.sets) open_stream(stream, n, next, smem);
            if (mine) {
                // rows of threads -> channels -> groups
                put_rows(red, at, channels, mean, m2);
                if (at.col == 0) counts[at.row] = count;
                role.sync();
                for (int c = role.tid; c < s.channels; c += kHalf) {
                    float all = counts[0], m = red[c].x, q = red[c].y;
                    for (int r = 1; r < at.rows; ++r) merge(all, m, q, counts[r], red[r * channels + c].x, red[r * channels + c].y);
                    red[c] = make_float2(m, q);          // (row 0's own place)
                }
                role.sync();
                const float pixels = (float)(at.p1 - at.p0);
                for (int g = warp; g < s.groups; g += kHalf / 32) {
                    float all = 0.f, m = 0.f, q = 0.f;
                    for (int c = lane; c < n.cg; c += 32) merge(all, m, q, pixels, red[g * n.cg + c].x, red[g * n.cg + c].y);
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) {
                        const float all_d = __shfl_down_sync(0xffffffffu, all, d), m_d = __shfl_down_sync(0xffffffffu, m, d),
                                    q_d = __shfl_down_sync(0xffffffffu, q, d);
                        if (lane < d) merge(all, m, q, all_d, m_d, q_d);
                    }
                    if (lane == 0) set.part[((long long)at.unit * s.groups + g) * s.runs + role.run] = make_float2(m, q);
                }
            }
            arrive(role, s.summed + i);
            continue;
        }
        wait_for(role, s, s.summed + i);
        if (mine) {
            const float inv_m = 1.f / ((float)n.P * n.cg);
            each_group(role, s, set.part + (long long)at.unit * s.groups * s.runs, [&](int g, const float2 (&part)[kRunsLane]) {
                float values[kRunsLane], sum = 0.f, square = 0.f;
#pragma unroll
                for (int j = 0; j < kRunsLane; ++j) {
                    const long long first = (lane + 32 * j) * s.run;
                    values[j] = (float)max(min(n.P, first + s.run) - first, 0ll) * n.cg;
                    sum = fmaf(values[j], part[j].x, sum);
                }
                const float mean = warp_sum(sum) * inv_m;
#pragma unroll
                for (int j = 0; j < kRunsLane; ++j) square += fmaf(values[j] * (part[j].x - mean), part[j].x - mean, part[j].y);
                const float rstd = rsqrtf(fmaf(warp_sum(square), inv_m, n.eps));
                if (lane == 0) {
                    stats[g] = make_float2(mean, rstd);
                    if (role.run == 0) {
                        n.mean[at.b * n.G + at.c0 / n.cg + g] = mean;
                        n.rstd[at.b * n.G + at.c0 / n.cg + g] = rstd;
                    }
                }
            });
            role.sync();
            if (at.pixels > 0) {
                Affine<N> k;
                k.template read<T>(n, at, [&](int c) { return stats[c / n.cg]; });
                T* dst = static_cast<T*>(n.y) + at.first(Map{nullptr, n.P * n.C, n.C}, N);
                for (int p = 0; p < at.pixels; p += kStage) {
                    Vec<T, N> x[kStage][1];
                    stream.take(x);
#pragma unroll
                    for (int u = 0; u < kStage; ++u) {
                        if (p + u >= at.pixels) break;
                        Pairs<N> f = widen_all(x[u][0]);
#pragma unroll
                        for (int j = 0; j < K; ++j)
                            f.at[j] = activate2<SILU>(fma2(add2(f.at[j], k.minus_mean.at[j]), k.scale.at[j], k.shift.at[j]));
                        store_all(dst + (long long)(p + u) * at.rows * n.C, f);
                    }
                }
            }
        }
        if (i + 1 < s.sets) open_stream(stream, n, next, smem);
        arrive(role, s.written + i);
    }
}

// Sums: A = sum dz and B = sum dz xhat of each channel, added to the block's row of `sums` (row, C), the same row for every set; and of w A
// and w B over each group.  Writes: d_x = rstd (dz w - (s1 + xhat s2) / M) = dz (rstd w) + (x - mean) c2 + c1.
template <typename T, int N, bool SILU>
__global__ void __launch_bounds__(2 * kHalf, 1) norm_bwd_kernel(const Norm n, const Pass s, float2* __restrict__ sums) {
    using namespace na2d_ptx;
    constexpr int K = Pairs<N>::K;
    extern __shared__ __align__(16) uint8_t smem_all[];
    const Role role(s);
    uint8_t* smem = smem_all + (role.writes ? GradStream<T, N>::kBytes : 0);
    float2* red = reinterpret_cast<float2*>(smem_all + 2 * GradStream<T, N>::kBytes);    // sums: [row][channel]
    float4* group = reinterpret_cast<float4*>(red + kHalf * N);                          // writes: [group]: mean, rstd, c1, c2
    const int warp = role.warp, lane = role.lane, channels = s.cols_p2 * N;
    if (role.writes && !n.d_x) return;
    GradStream<T, N> stream;
    Spot next = spot_in(n, s, role, 0);
    open_stream(stream, n, next, smem);
    for (int i = 0; i < s.sets; ++i) {
        const Set set = set_of(s, i);
        const Spot at = next;
        const bool mine = role.unit < set.count;
        if (i + 1 < s.sets) next = spot_in(n, s, role, i + 1);
        if (!role.writes) {
            Pairs<N> a, d;
#pragma unroll
            for (int j = 0; j < K; ++j) a.at[j] = d.at[j] = 0;
            if (at.pixels > 0) {
                Affine<N> k;
                k.template read<T>(n, at, [&](int c) {
                    const int g = at.b * n.G + (at.c0 + c) / n.cg;
                    return make_float2(n.mean[g], n.rstd[g]);
                });
                for (int p = 0; p < at.pixels; p += kStage) {
                    Vec<T, N> v[kStage][2];
                    stream.take(v);
#pragma unroll
                    for (int u = 0; u < kStage; ++u) {
                        if (p + u >= at.pixels) break;
                        const Pairs<N> f = widen_all(v[u][0]), e = widen_all(v[u][1]);
#pragma unroll
                        for (int j = 0; j < K; ++j) {
                            const uint64_t off = add2(f.at[j], k.minus_mean.at[j]);
                            const uint64_t dz = through2<SILU>(e.at[j], fma2(off, k.scale.at[j], k.shift.at[j]));
                            a.at[j] = add2(a.at[j], dz);
                            d.at[j] = fma2(dz, off, d.at[j]);
                        }
                    }
                }
            }
            if (i >= kAhead && n.d_x) wait_for(role, s, s.written + i - kAhead);
            if (i + 1 < s.sets) open_stream(stream, n, next, smem);
            if (mine) {
                put_rows(red, at, channels, a, d);
                role.sync();
                const long long row = (long long)role.unit * s.runs + role.run;
                for (int c = role.tid; c < s.channels; c += kHalf) {
                    float2 sum = make_float2(0.f, 0.f);
                    for (int r = 0; r < at.rows; ++r) {
                        sum.x += red[r * channels + c].x;
                        sum.y += red[r * channels + c].y;
                    }
                    sum.y *= n.rstd[at.b * n.G + (at.c0 + c) / n.cg];        // d has x - mean in the place of xhat
                    if (sums) {
                        float2* to = sums + row * n.C + at.c0 + c;
                        const float2 old = *to;
                        *to = make_float2(old.x + sum.x, old.y + sum.y);
                    }
                    const float w = param<T>(n, n.w, at.c0 + c, 1.f);
                    red[c] = make_float2(w * sum.x, w * sum.y);              // (row 0's own place)
                }
                role.sync();
                for (int g = warp; g < s.groups; g += kHalf / 32) {
                    float s1 = 0.f, s2 = 0.f;
                    for (int c = lane; c < n.cg; c += 32) {
                        s1 += red[g * n.cg + c].x;
                        s2 += red[g * n.cg + c].y;
                    }
                    s1 = warp_sum(s1);
                    s2 = warp_sum(s2);
                    if (lane == 0) set.part[((long long)at.unit * s.groups + g) * s.runs + role.run] = make_float2(s1, s2);
                }
            }
            arrive(role, s.summed + i);
            continue;
        }
        wait_for(role, s, s.summed + i);
        if (mine) {
            const float inv_m = 1.f / ((float)n.P * n.cg);
            each_group(role, s, set.part + (long long)at.unit * s.groups * s.runs, [&](int g, const float2 (&part)[kRunsLane]) {
                const int at_g = at.b * n.G + at.c0 / n.cg + g;
                const float rstd = n.rstd[at_g], mean = n.mean[at_g];
                float s1 = 0.f, s2 = 0.f;
#pragma unroll
                for (int j = 0; j < kRunsLane; ++j) {
                    s1 += part[j].x;
                    s2 += part[j].y;
                }
                s1 = warp_sum(s1) * inv_m;
                s2 = warp_sum(s2) * inv_m;
                if (lane == 0) group[g] = make_float4(mean, rstd, -rstd * s1, -rstd * rstd * s2);
            });
            role.sync();
            if (at.pixels > 0) {
                Affine<N> k;
                k.template read<T>(n, at, [&](int c) { return make_float2(group[c / n.cg].x, group[c / n.cg].y); });
                Pairs<N> c1, c2;
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    const float4 u = group[(at.col * N + 2 * j) / n.cg], v = group[(at.col * N + min(2 * j + 1, N - 1)) / n.cg];
                    c1.at[j] = pair2(u.z, v.z);
                    c2.at[j] = pair2(u.w, v.w);
                }
                T* dst = static_cast<T*>(n.d_x) + at.first(Map{nullptr, n.P * n.C, n.C}, N);
                for (int p = 0; p < at.pixels; p += kStage) {
                    Vec<T, N> v[kStage][2];
                    stream.take(v);
#pragma unroll
                    for (int u = 0; u < kStage; ++u) {
                        if (p + u >= at.pixels) break;
                        Pairs<N> f = widen_all(v[u][0]);
                        const Pairs<N> e = widen_all(v[u][1]);
#pragma unroll
                        for (int j = 0; j < K; ++j) {
                            const uint64_t off = add2(f.at[j], k.minus_mean.at[j]);
                            const uint64_t dz = through2<SILU>(e.at[j], fma2(off, k.scale.at[j], k.shift.at[j]));
                            f.at[j] = fma2(dz, k.scale.at[j], fma2(off, c2.at[j], c1.at[j]));
                        }
                        store_all(dst + (long long)(p + u) * at.rows * n.C, f);
                    }
                }
            }
        }
        if (i + 1 < s.sets) open_stream(stream, n, next, smem);
        arrive(role, s.written + i);
    }
}

// ---- groups wider than a block of vectors: a block a group, a thread a channel at a time ---------------------------------
// (Made for odd widths on small maps: 1 x 64^2 x 1542 in 3 groups, bf16, 3.1 + 3.2 ms.  4 x 64^2 x 4096 in one group takes 43 + 48 ms on 4 of
// the SMs.)
// A sum of any number of values, with what its roundings lost (a thread has all pixels of its channels, hundreds of thousands of values:
// without, the variance of 2^20 came out 5e-4 too small).
struct LongSum {
    float sum = 0.f, lost = 0.f;
    __device__ __forceinline__ void add(float x) {
        const float next = sum + x, part = next - sum;
        lost += (sum - (next - part)) + (x - part);
        sum = next;
    }
    __device__ __forceinline__ float value() const { return sum + lost; }
};
__device__ __forceinline__ float block_sum(float x, float* red) {
    x = warp_sum(x);
    __syncthreads();
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = x;
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += red[w];
    return sum;
}

template <typename T, bool SILU>
__global__ void __launch_bounds__(kThreads) norm_wide_fwd_kernel(const Norm n) {
    __shared__ float red[kWarps];
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    const int b = blockIdx.x / n.G, g = blockIdx.x - b * n.G;
    const T* x = static_cast<const T*>(n.x.ptr) + b * n.x.b + g * n.cg;
    const float inv_m = 1.f / ((float)n.P * n.cg);
    LongSum sum, square;
    for (int c = threadIdx.x; c < n.cg; c += kThreads)
        for (long long p = 0; p < n.P; ++p) sum.add(na2d_vec::widen(x[p * n.x.p + c]));
    const float mean = block_sum(sum.value(), red) * inv_m;
    for (int c = threadIdx.x; c < n.cg; c += kThreads)
        for (long long p = 0; p < n.P; ++p) {
            const float off = na2d_vec::widen(x[p * n.x.p + c]) - mean;
            square.add(off * off);
        }
    const float rstd = rsqrtf(fmaf(block_sum(square.value(), red), inv_m, n.eps));
    if (threadIdx.x == 0) {
        n.mean[blockIdx.x] = mean;
        n.rstd[blockIdx.x] = rstd;
    }
    T* y = static_cast<T*>(n.y) + (long long)b * n.P * n.C + g * n.cg;
    for (int c = threadIdx.x; c < n.cg; c += kThreads) {
        const float scale = rstd * param<T>(n, n.w, g * n.cg + c, 1.f), shift = param<T>(n, n.bias, g * n.cg + c, 0.f);
        for (long long p = 0; p < n.P; ++p)
            y[p * n.C + c] = na2d_vec::narrow<T>(activate<SILU>(fmaf(na2d_vec::widen(x[p * n.x.p + c]) - mean, scale, shift)));
    }
}

template <typename T, bool SILU>
__global__ void __launch_bounds__(kThreads) norm_wide_bwd_kernel(const Norm n, float2* __restrict__ sums) {
    __shared__ float red[kWarps];
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    const int b = blockIdx.x / n.G, g = blockIdx.x - b * n.G;
    const T* x = static_cast<const T*>(n.x.ptr) + b * n.x.b + g * n.cg;
    const T* e = static_cast<const T*>(n.d_y.ptr) + b * n.d_y.b + g * n.cg;
    const float inv_m = 1.f / ((float)n.P * n.cg), mean = n.mean[blockIdx.x], rstd = n.rstd[blockIdx.x];
    float s1 = 0.f, s2 = 0.f;
    auto dz_of = [&](long long p, int c, float w, float bias, float& xhat) {
        xhat = (na2d_vec::widen(x[p * n.x.p + c]) - mean) * rstd;
        return na2d_vec::widen(e[p * n.d_y.p + c]) * slope<SILU>(fmaf(xhat, w, bias));
    };
    for (int c = threadIdx.x; c < n.cg; c += kThreads) {
        const float w = param<T>(n, n.w, g * n.cg + c, 1.f), bias = param<T>(n, n.bias, g * n.cg + c, 0.f);
        LongSum a, d;
        float xhat;
        for (long long p = 0; p < n.P; ++p) {
            const float dz = dz_of(p, c, w, bias, xhat);
            a.add(dz);
            d.add(dz * xhat);
        }
        if (sums) sums[(long long)b * n.C + g * n.cg + c] = make_float2(a.value(), d.value());
        s1 = fmaf(w, a.value(), s1);
        s2 = fmaf(w, d.value(), s2);
    }
    s1 = block_sum(s1, red) * inv_m;
    s2 = block_sum(s2, red) * inv_m;
    if (!n.d_x) return;
    T* dst = static_cast<T*>(n.d_x) + (long long)b * n.P * n.C + g * n.cg;
    for (int c = threadIdx.x; c < n.cg; c += kThreads) {
        const float w = param<T>(n, n.w, g * n.cg + c, 1.f), bias = param<T>(n, n.bias, g * n.cg + c, 0.f);
        for (long long p = 0; p < n.P; ++p) {
            float xhat;
            const float dz = dz_of(p, c, w, bias, xhat);
            dst[p * n.C + c] = na2d_vec::narrow<T>(rstd * (fmaf(dz, w, -s1) - xhat * s2));
        }
    }
}

// d_weight and d_bias: the sums of `rows` rows of (A, B) of each channel.  32 channels a block; a warp of it has every eighth row.
template <typename W>
__global__ void __launch_bounds__(kThreads) norm_params_kernel(const float2* __restrict__ sums, W* __restrict__ d_w, W* __restrict__ d_b, int rows, int C) {
    __shared__ float2 red[kWarps][32];
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
    float u = 0.f, v = 0.f;
    if (c < C) {
#pragma unroll 8
        for (int r = warp; r < rows; r += kWarps) {
            const float2 x = sums[(long long)r * C + c];
            u += x.x;
            v += x.y;
        }
    }
    red[warp][lane] = make_float2(u, v);
    __syncthreads();
    if (warp == 0 && c < C) {
        for (int w = 1; w < kWarps; ++w) {
            u += red[w][lane].x;
            v += red[w][lane].y;
        }
        if (d_b) d_b[c] = na2d_vec::narrow<W>(u);
        if (d_w) d_w[c] = na2d_vec::narrow<W>(v);
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
constexpr int kChipBytes = 112 << 10;           // shared memory of a block on the chip: two blocks an SM
// What a set of the two passes reads.  4 x 256^2 x 512, forward and backward: 12 MB 451 us, 36 MB 415, 72 MB 385 to 407, 150 MB 380; but there
// 3 x 300^2 x 384 takes 172 us forward for 139, its sets being uneven.
constexpr long long kL2Bytes = 72ll << 20;

int power_of_two(int n) {
    int p = 1;
    while (p < n) p *= 2;
    return p;
}
int common_multiple(int a, int b) {
    int x = a, y = b;
    while (y) {
        const int r = x % y;
        x = y;
        y = r;
    }
    return a / x * b;
}

// Values of a vector: as many as 16 bytes hold where base and strides allow, else 8 bytes', else one.
int vector_of(const Norm& n, int esize, bool backward) {
    auto fits = [&](int v) {
        const int bytes = v * esize;
        bool ok = n.C % v == 0;
        auto operand = [&](const void* p, long long a, long long b) {
            ok = ok && reinterpret_cast<uintptr_t>(p) % bytes == 0 && a % v == 0 && b % v == 0;
        };
        operand(n.x.ptr, n.x.b, n.x.p);
        if (backward) operand(n.d_y.ptr, n.d_y.b, n.d_y.p);
        operand(backward ? n.d_x : n.y, 0, 0);
        return ok;
    };
    return fits(16 / esize) ? 16 / esize : fits(8 / esize) ? 8 / esize : 1;
}

size_t chip_bytes(const Slab& s, int esize, int operands) {
    return operands * (((size_t)s.pixels * s.channels * esize + 15) / 16 * 16) + (size_t)(kWarps + 3) * s.channels * sizeof(float);
}

// Whether the call runs on the chip, and how: the smallest cluster that holds a slab.
bool chip_plan(const Norm& n, int esize, int vec, bool backward, Slab* s) {
    const int unit = common_multiple(n.cg, vec);
    if (n.C % unit != 0) return false;
    s->channels = unit;
    // 64 bytes of a pixel (a sector pair): more channels a slab only where groups or vectors are larger
    while (s->channels * esize < 64 && n.C % (2 * s->channels) == 0) s->channels *= 2;
    s->cols = s->channels / vec;
    if (s->cols > 32) return false;
    s->cols_p2 = power_of_two(s->cols);
    s->slabs = n.C / s->channels;
    for (s->cluster = 1; s->cluster <= kMaxCluster; s->cluster *= 2) {
        const long long pixels = (n.P + s->cluster - 1) / s->cluster;
        if (pixels > (1 << 20)) continue;
        s->pixels = (int)pixels;
        if (chip_bytes(*s, esize, backward ? 2 : 1) <= kChipBytes) return true;
    }
    return false;
}

// The two passes with vectors of `vec` channels: units of whole groups, of at most kL2Bytes where a slab of at least 256 bytes of a pixel
// can be that small, as many of them a set as stay under it; and runs so that there is a block an SM.  False: a group is
// wider than a block.
bool pass_plan(const Norm& n, int esize, int vec, bool backward, int sms, Pass* s) {
    const int unit = common_multiple(n.cg, vec), operands = backward ? 2 : 1;
    if (n.C % unit != 0 || unit / vec > kHalf) return false;
    auto bytes = [&](int channels) { return n.P * channels * esize * operands; };
    s->channels = n.C;
    // the largest slab that divides the channels, fits a block, and stays in L2 or is as narrow as it may be
    for (int parts = 1; parts <= n.C / unit; ++parts) {
        if ((n.C / unit) % parts != 0) continue;
        s->channels = n.C / parts;
        if (s->channels / vec > kHalf) continue;
        if (bytes(s->channels) <= kL2Bytes) break;
        int next = parts + 1;
        while (next <= n.C / unit && (n.C / unit) % next != 0) ++next;
        if (next > n.C / unit || n.C / next * esize < 256) break;
    }
    if (s->channels / vec > kHalf) return false;
    s->slabs = n.C / s->channels;
    s->cols = s->channels / vec;
    s->cols_p2 = power_of_two(s->cols);
    s->groups = s->channels / n.cg;
    s->units = n.B * s->slabs;
    s->at_once = (int)std::max(1LL, std::min({(long long)s->units, kL2Bytes / std::max(1LL, (long long)bytes(s->channels)), (long long)sms}));
    s->sets = (s->units + s->at_once - 1) / s->at_once;
    const int rows = kHalf / s->cols_p2;
    const long long runs = std::max(1LL, std::min({(long long)sms / s->at_once, (long long)kMostRuns, (long long)(n.P / (kStage * rows))}));
    s->run = (n.P + runs - 1) / runs;
    s->runs = (int)((n.P + s->run - 1) / s->run);
    return true;
}

int make_norm(const na2d_norm_args* a, Norm* n) {
    if (!a || a->struct_size < sizeof(na2d_norm_args)) return NA2D_ERR_BAD_ARG;
    if (a->B <= 0 || a->C <= 0 || a->P <= 0 || a->groups <= 0 || a->C % a->groups != 0) return NA2D_ERR_BAD_ARG;
    if (a->dtype != NA2D_F32 && a->dtype != NA2D_BF16 && a->dtype != NA2D_F16) return NA2D_ERR_UNSUPPORTED;
    if (a->param_dtype != NA2D_F32 && a->param_dtype != a->dtype) return NA2D_ERR_UNSUPPORTED;
    if (a->activation != NA2D_ACT_NONE && a->activation != NA2D_ACT_SILU) return NA2D_ERR_BAD_ARG;
    if (!(a->eps >= 0.f) || !(a->eps < 3.0e38f)) return NA2D_ERR_BAD_ARG;
    if (a->workspace && reinterpret_cast<uintptr_t>(a->workspace) % 16) return NA2D_ERR_BAD_ARG;
    if (a->B > 65535 || a->C > (1 << 14) || a->P > (1ll << 31) / 4) return NA2D_ERR_TOO_LARGE;
    auto map = [&](const na2d_pixels& x) {
        const bool dense = x.stride_b == 0 && x.stride_p == 0;
        const long long p = dense || a->P == 1 ? a->C : x.stride_p;
        return Map{x.ptr, dense || a->B == 1 ? a->P * p : x.stride_b, p};
    };
    *n = Norm{a->B, a->C, a->groups, a->C / a->groups, a->P, a->eps, map(a->x), map(a->d_y), a->y, a->d_x, a->weight, a->bias,
              a->param_dtype == NA2D_F32, a->mean, a->rstd};
    return NA2D_OK;
}

// f(type, vector width): TypeTag and an integral constant
template <typename T> struct Tag { using type = T; };
template <typename F>
int by_type(int dtype, int vec, F&& f) {
    auto pick = [&](auto t, auto full, auto half) -> int {
        if (vec == decltype(full)::value) return f(t, full);
        if (vec == decltype(half)::value) return f(t, half);
        return f(t, std::integral_constant<int, 1>{});
    };
    using std::integral_constant;
    if (dtype == NA2D_F32) return pick(Tag<float>{}, integral_constant<int, 4>{}, integral_constant<int, 2>{});
    if (dtype == NA2D_BF16) return pick(Tag<__nv_bfloat16>{}, integral_constant<int, 8>{}, integral_constant<int, 4>{});
    return pick(Tag<__half>{}, integral_constant<int, 8>{}, integral_constant<int, 4>{});
}

int launched(cudaError_t e, const char* what) {
    if (e != cudaSuccess) return na2d_host::cuda_fail(e, what);
    na2d_host::count_launches(1);
    return NA2D_OK;
}

template <typename K>
int allow_smem(K kernel, size_t bytes) {
    if (bytes <= 48 * 1024) return NA2D_OK;
    const cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e == cudaSuccess ? NA2D_OK : na2d_host::cuda_fail(e, "cudaFuncSetAttribute");
}

template <typename K, typename... A>
int launch_chip(K kernel, const Slab& s, int B, size_t smem, cudaStream_t st, A... args) {
    const long long blocks = (long long)B * s.slabs * s.cluster;
    if (blocks > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    if (int rc = allow_smem(kernel, smem)) return rc;
    cudaLaunchAttribute attribute[2]{};
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    attribute[1].id = cudaLaunchAttributeClusterDimension;
    attribute[1].val.clusterDim.x = s.cluster;
    attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)blocks);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    config.attrs = attribute;
    config.numAttrs = s.cluster > 1 ? 2 : 1;
    return launched(cudaLaunchKernelEx(&config, kernel, args...), "group norm launch");
}

// Shared memory of a pass: the halves' streams, two sums a channel of each thread, a count a row and two values a group; or four values a group.
template <typename T, int N>
size_t pass_bytes(const Pass& s, bool backward) {
    const size_t sums = (size_t)kHalf * N * sizeof(float2);
    return backward ? 2 * GradStream<T, N>::kBytes + sums + s.groups * sizeof(float4)
                    : 2 * MapStream<T, N>::kBytes + sums + kHalf * sizeof(float) + s.groups * sizeof(float2);
}
// Workspace: the runs' values of kBuffers sets, the counts of blocks (cleared by each call), then (backward) the blocks' rows of channel sums
// (cleared, too); on the chip, and for wide groups, the batch entries' channel sums alone.
struct Room {
    size_t part, arrived, sums;         // bytes
    size_t all() const { return part + arrived + sums; }
};
size_t align16(size_t bytes) { return (bytes + 15) / 16 * 16; }
Room pass_room(const Norm& n, const Pass& s, bool backward) {
    return Room{align16((size_t)kBuffers * s.at_once * s.groups * s.runs * sizeof(float2)), align16((size_t)(2 * s.sets + 1) * sizeof(unsigned)),
                backward ? (size_t)s.at_once * s.runs * n.C * sizeof(float2) : 0};
}
size_t workspace_bytes(const Norm& n, int dtype, bool backward, int sms) {
    const int esize = dtype == NA2D_F32 ? 4 : 2;
    size_t bytes = 0;                   // with the vectors that need most: results need not have been allocated when this is asked
    for (int v : {16 / esize, 8 / esize, 1}) {
        Slab slab;
        Pass s;
        if (n.C % v != 0) continue;
        if (!chip_plan(n, esize, v, backward, &slab) && pass_plan(n, esize, v, backward, sms, &s)) bytes = std::max(bytes, pass_room(n, s, backward).all());
        else if (backward) bytes = std::max(bytes, (size_t)n.B * n.C * sizeof(float2));
    }
    return bytes;
}

// Sets the plan's workspace up and launches its kernel on all blocks at once.
template <typename K, typename... A>
int launch_pass(K kernel, const na2d_norm_args* a, const Norm& n, Pass& s, const Room& room, size_t smem, A... args) {
    if (!a->workspace || a->workspace_bytes < room.all()) return NA2D_ERR_BAD_ARG;
    if (int rc = allow_smem(kernel, smem)) return rc;
    if (int rc = na2d_host::error_state(a->device, &s.errors)) return rc;
    const cudaStream_t st = (cudaStream_t)a->stream;
    uint8_t* at = static_cast<uint8_t*>(a->workspace);
    s.part = reinterpret_cast<float2*>(at);
    s.summed = reinterpret_cast<unsigned*>(at + room.part);
    s.written = s.summed + s.sets;
    s.gave_up = s.written + s.sets;
    cudaError_t e = cudaMemsetAsync(s.summed, 0, room.arrived + room.sums, st);
    if (e != cudaSuccess) return na2d_host::cuda_fail(e, "cudaMemsetAsync");
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeCooperative;
    attribute.val.cooperative = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(s.runs * s.at_once);
    config.blockDim = dim3(2 * kHalf);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return launched(cudaLaunchKernelEx(&config, kernel, n, (const Pass)s, args...), "group norm launch");
}

template <typename T, int N, bool SILU>
int forward_as(const na2d_norm_args* a, const Norm& n, cudaStream_t st) {
    Slab slab;
    if (chip_plan(n, sizeof(T), N, false, &slab))
        return launch_chip(norm_chip_fwd_kernel<T, N, SILU>, slab, n.B, chip_bytes(slab, sizeof(T), 1), st, n, slab);
    Pass s;
    if (!pass_plan(n, sizeof(T), N, false, na2d_host::sm_count(a->device), &s))
        return launched(na2d_launch::launch(true, norm_wide_fwd_kernel<T, SILU>, dim3((unsigned)(n.B * n.G)), kThreads, 0, st, n), "group norm launch");
    return launch_pass(norm_fwd_kernel<T, N, SILU>, a, n, s, pass_room(n, s, false), pass_bytes<T, N>(s, false));
}

template <typename T, int N, bool SILU>
int backward_as(const na2d_norm_args* a, const Norm& n, cudaStream_t st) {
    const bool params = a->d_weight || a->d_bias;
    Slab slab;
    Pass s;
    int rows = n.B;                                      // of sums: batch entries, or blocks
    float2* sums = nullptr;
    const bool chip = chip_plan(n, sizeof(T), N, true, &slab);
    if (chip || !pass_plan(n, sizeof(T), N, true, na2d_host::sm_count(a->device), &s)) {
        if (params) {
            if (!a->workspace || a->workspace_bytes < (size_t)n.B * n.C * sizeof(float2)) return NA2D_ERR_BAD_ARG;
            sums = static_cast<float2*>(a->workspace);
        }
        int rc;
        if (chip) rc = launch_chip(norm_chip_bwd_kernel<T, N, SILU>, slab, n.B, chip_bytes(slab, sizeof(T), 2), st, n, slab, sums);
        else rc = launched(na2d_launch::launch(true, norm_wide_bwd_kernel<T, SILU>, dim3((unsigned)(n.B * n.G)), kThreads, 0, st, n, sums), "group norm launch");
        if (rc != NA2D_OK) return rc;
    } else {
        const Room room = pass_room(n, s, true);
        rows = s.at_once * s.runs;
        if (params) sums = reinterpret_cast<float2*>(static_cast<uint8_t*>(a->workspace) + room.part + room.arrived);
        if (int rc = launch_pass(norm_bwd_kernel<T, N, SILU>, a, n, s, room, pass_bytes<T, N>(s, true), sums)) return rc;
    }
    if (!params) return NA2D_OK;
    auto finish = [&](auto tag) {
        using W = typename decltype(tag)::type;
        return launched(na2d_launch::launch(true, norm_params_kernel<W>, dim3((n.C + 31) / 32), kThreads, 0, st, (const float2*)sums,
                                            (W*)a->d_weight, (W*)a->d_bias, rows, n.C), "group norm launch");
    };
    return n.param_f32 ? finish(Tag<float>{}) : finish(Tag<T>{});
}

}  // namespace

extern "C" {

int na2d_group_norm_forward(const na2d_norm_args* a) {
    if (!a || !a->x.ptr || !a->y || !a->mean || !a->rstd) return NA2D_ERR_BAD_ARG;
    Norm n;
    if (int rc = make_norm(a, &n)) return rc;
    return na2d_host::on_device(a->device, [&]() -> int {
        return by_type(a->dtype, vector_of(n, a->dtype == NA2D_F32 ? 4 : 2, false), [&](auto t, auto v) {
            using T = typename decltype(t)::type;
            constexpr int N = decltype(v)::value;
            return a->activation == NA2D_ACT_SILU ? forward_as<T, N, true>(a, n, (cudaStream_t)a->stream)
                                                  : forward_as<T, N, false>(a, n, (cudaStream_t)a->stream);
        });
    });
}

int na2d_group_norm_backward(const na2d_norm_args* a) {
    if (!a || !a->x.ptr || !a->d_y.ptr || !a->mean || !a->rstd) return NA2D_ERR_BAD_ARG;
    if (!a->d_x && !a->d_weight && !a->d_bias) return NA2D_ERR_BAD_ARG;
    Norm n;
    if (int rc = make_norm(a, &n)) return rc;
    return na2d_host::on_device(a->device, [&]() -> int {
        return by_type(a->dtype, vector_of(n, a->dtype == NA2D_F32 ? 4 : 2, true), [&](auto t, auto v) {
            using T = typename decltype(t)::type;
            constexpr int N = decltype(v)::value;
            return a->activation == NA2D_ACT_SILU ? backward_as<T, N, true>(a, n, (cudaStream_t)a->stream)
                                                  : backward_as<T, N, false>(a, n, (cudaStream_t)a->stream);
        });
    });
}

size_t na2d_group_norm_workspace(const na2d_norm_args* a, int backward) {
    Norm n;
    return make_norm(a, &n) == NA2D_OK ? workspace_bytes(n, a->dtype, backward != 0, na2d_host::sm_count(a->device)) : 0;
}

}  // extern "C"
