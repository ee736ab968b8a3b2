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
// In two passes, where a slab is too large for that: partial sums of runs of pixels, then a pass that writes.  Batch entries are taken
// as many at a time as stay in L2, and the second pass walks the pixels backwards, from what the first read last.
//
// Variances are sums of squares about a mean at every step (of a slab; of four pixels, merged with those before), so that maps
// whose mean is far above their spread lose nothing.  All sums are in fp32 and in an order that the sizes alone fix.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

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
    extern __shared__ __align__(16) uint8_t smem[];
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
    extern __shared__ __align__(16) uint8_t smem[];
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
// Runs of `run` pixels of batch entries b0, b0 + 1, ...; a block has one run of up to `cols_p2` vector columns from blockIdx.z * cols_p2 on.
struct Pass {
    int b0, batches;
    int cols, cols_p2;              // vector columns of a pixel; of a block
    long long run;
    int runs;
};

// The merge of two sets of values: counts, means and sums of squares about them.
__device__ __forceinline__ void merge(float& count, float& mean, float& m2, float n, float mean_n, float m2_n) {
    const float all = count + n;
    if (n == 0.f) return;
    const float share = n / all, off = mean_n - mean;
    mean = fmaf(off, share, mean);
    m2 += fmaf(off * off, count * share, m2_n);
    count = all;
}

// (mean, sum of squares about it) of every channel of a run -> part[(b, run, C)]
template <typename T, int N>
__global__ void __launch_bounds__(kThreads) norm_stats_kernel(const Norm n, const Pass s, float2* __restrict__ part) {
    extern __shared__ __align__(16) float red[];         // [rows][cols_p2 * N]{mean, m2}, then [rows] counts
    const int col = threadIdx.x % s.cols_p2, row = threadIdx.x / s.cols_p2, rows = kThreads / s.cols_p2;
    const int vec = blockIdx.z * s.cols_p2 + col, b = s.b0 + blockIdx.y;
    const long long p0 = blockIdx.x * s.run, p1 = min(n.P, p0 + s.run);
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    float count = 0.f, mean[N], m2[N];
#pragma unroll
    for (int i = 0; i < N; ++i) mean[i] = m2[i] = 0.f;
    if (vec < s.cols) {
        const T* src = static_cast<const T*>(n.x.ptr) + b * n.x.b + vec * N;
        constexpr int U = 4;                             // pixels whose values are summed about their own mean, then merged
        long long p = p0 + row;
        for (; p + (U - 1) * rows < p1; p += U * rows) {
            Vec<T, N> x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u].load(src + (p + u * rows) * n.x.p);
            const float share = __fdividef((float)U, count + U), weight = count * share;
            float f[U][N];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u].widened(f[u]);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float m = ((f[0][i] + f[1][i]) + (f[2][i] + f[3][i])) * (1.f / U);
                float q = 0.f;
#pragma unroll
                for (int u = 0; u < U; ++u) q = fmaf(f[u][i] - m, f[u][i] - m, q);
                const float off = m - mean[i];
                mean[i] = fmaf(off, share, mean[i]);
                m2[i] += fmaf(off * off, weight, q);
            }
            count += U;
        }
        for (; p < p1; p += rows) {
            Vec<T, N> x;
            float f[N];
            x.load(src + p * n.x.p);
            x.widened(f);
            const float share = __fdividef(1.f, count + 1.f);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float off = f[i] - mean[i];
                mean[i] = fmaf(off, share, mean[i]);
                m2[i] = fmaf(off * off, count * share, m2[i]);
            }
            count += 1.f;
        }
    }
    const int channels = s.cols_p2 * N;
    float* counts = red + rows * channels * 2;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        red[(row * channels + col * N + i) * 2] = mean[i];
        red[(row * channels + col * N + i) * 2 + 1] = m2[i];
    }
    if (col == 0) counts[row] = count;
    __syncthreads();
    for (int c = threadIdx.x; c < channels; c += kThreads) {
        const int channel = blockIdx.z * channels + c;
        if (channel >= n.C) break;
        float all = counts[0], m = red[2 * c], q = red[2 * c + 1];
        for (int r = 1; r < rows; ++r) merge(all, m, q, counts[r], red[(r * channels + c) * 2], red[(r * channels + c) * 2 + 1]);
        part[((long long)blockIdx.y * s.runs + blockIdx.x) * n.C + channel] = make_float2(m, q);
    }
}

__device__ __forceinline__ float block_sum(float x, float* red) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    __syncthreads();
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = x;
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += red[w];
    return sum;
}

// mean and rstd of group blockIdx.x of batch entry b0 + blockIdx.y from the runs' values
__global__ void __launch_bounds__(kThreads) norm_finish_stats_kernel(const Norm n, const Pass s, const float2* __restrict__ part) {
    __shared__ float red[kWarps];
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    const float2* at = part + (long long)blockIdx.y * s.runs * n.C + blockIdx.x * n.cg;
    const long long values = (long long)s.runs * n.cg;
    auto pixels = [&](long long run) { return (float)(min(n.P, (run + 1) * s.run) - run * s.run); };
    float sum = 0.f;
    for (long long i = threadIdx.x; i < values; i += kThreads) sum = fmaf(pixels(i / n.cg), at[i / n.cg * n.C + i % n.cg].x, sum);
    const float inv_m = 1.f / ((float)n.P * n.cg), mean = block_sum(sum, red) * inv_m;
    sum = 0.f;
    for (long long i = threadIdx.x; i < values; i += kThreads) {
        const float2 v = at[i / n.cg * n.C + i % n.cg];
        sum += fmaf(pixels(i / n.cg), (v.x - mean) * (v.x - mean), v.y);
    }
    const float var = block_sum(sum, red) * inv_m;
    if (threadIdx.x == 0) {
        const long long g = (long long)(s.b0 + blockIdx.y) * n.G + blockIdx.x;
        n.mean[g] = mean;
        n.rstd[g] = rsqrtf(var + n.eps);
    }
}

template <typename T, int N, bool SILU>
__global__ void __launch_bounds__(kThreads) norm_apply_kernel(const Norm n, const Pass s) {
    const int col = threadIdx.x % s.cols_p2, row = threadIdx.x / s.cols_p2, rows = kThreads / s.cols_p2;
    const int vec = blockIdx.z * s.cols_p2 + col;
    // backwards: what the pass before read last is still in L2
    const int b = s.b0 + s.batches - 1 - blockIdx.y;
    const long long run = s.runs - 1 - blockIdx.x, p0 = run * s.run, p1 = min(n.P, p0 + s.run);
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    if (vec >= s.cols) return;
    const Column<T, N> k(n, b, vec * N);
    const T* src = static_cast<const T*>(n.x.ptr) + b * n.x.b + vec * N;
    T* dst = static_cast<T*>(n.y) + (long long)b * n.P * n.C + vec * N;
    float scale[N];
#pragma unroll
    for (int i = 0; i < N; ++i) scale[i] = k.rstd[i] * k.w[i];
#pragma unroll 4
    for (long long p = p1 - 1 - row; p >= p0; p -= rows) {
        Vec<T, N> x;
        float f[N];
        x.load(src + p * n.x.p);
        x.widened(f);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = activate<SILU>(fmaf(f[i] - k.mean[i], scale[i], k.bias[i]));
        x.round(f);
        x.store(dst + p * n.C);
    }
}

// (A, B) of every channel of a run -> part[(b, run, C)]
template <typename T, int N, bool SILU>
__global__ void __launch_bounds__(kThreads) norm_grad_sums_kernel(const Norm n, const Pass s, float2* __restrict__ part) {
    extern __shared__ __align__(16) float red[];         // [rows][cols_p2 * N]{A, B}
    const int col = threadIdx.x % s.cols_p2, row = threadIdx.x / s.cols_p2, rows = kThreads / s.cols_p2;
    const int vec = blockIdx.z * s.cols_p2 + col, b = s.b0 + blockIdx.y;
    const long long p0 = blockIdx.x * s.run, p1 = min(n.P, p0 + s.run);
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    float a[N], d[N];
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = d[i] = 0.f;
    if (vec < s.cols) {
        const Column<T, N> k(n, b, vec * N);
        const T* x0 = static_cast<const T*>(n.x.ptr) + b * n.x.b + vec * N;
        const T* g0 = static_cast<const T*>(n.d_y.ptr) + b * n.d_y.b + vec * N;
#pragma unroll 4
        for (long long p = p0 + row; p < p1; p += rows) {
            Vec<T, N> x, g;
            float f[N], e[N];
            x.load(x0 + p * n.x.p);
            g.load(g0 + p * n.d_y.p);
            x.widened(f);
            g.widened(e);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float xhat = (f[i] - k.mean[i]) * k.rstd[i], dz = e[i] * slope<SILU>(fmaf(xhat, k.w[i], k.bias[i]));
                a[i] += dz;
                d[i] = fmaf(dz, xhat, d[i]);
            }
        }
    }
    const int channels = s.cols_p2 * N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        red[(row * channels + col * N + i) * 2] = a[i];
        red[(row * channels + col * N + i) * 2 + 1] = d[i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < channels; c += kThreads) {
        const int channel = blockIdx.z * channels + c;
        if (channel >= n.C) break;
        float u = 0.f, v = 0.f;
        for (int r = 0; r < rows; ++r) {
            u += red[(r * channels + c) * 2];
            v += red[(r * channels + c) * 2 + 1];
        }
        part[((long long)blockIdx.y * s.runs + blockIdx.x) * n.C + channel] = make_float2(u, v);
    }
}

// Sums of the runs: (A, B) of each channel of the batch entry -> sums[(b, C)], and of group blockIdx.x (s1, s2) / M -> group[(b, G)]
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_finish_sums_kernel(const Norm n, const Pass s, const float2* __restrict__ part,
                                                                    float2* __restrict__ sums, float2* __restrict__ group) {
    __shared__ float red[kWarps];
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    const int b = s.b0 + blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    float s1 = 0.f, s2 = 0.f;
    // a warp a channel: its lanes share the runs
    for (int i = warp; i < n.cg; i += kWarps) {
        const int c = blockIdx.x * n.cg + i;
        float u = 0.f, v = 0.f;
        for (int r = lane; r < s.runs; r += 32) {
            const float2 x = part[((long long)blockIdx.y * s.runs + r) * n.C + c];
            u += x.x;
            v += x.y;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            u += __shfl_xor_sync(0xffffffffu, u, d);
            v += __shfl_xor_sync(0xffffffffu, v, d);
        }
        if (lane == 0) {
            sums[(long long)b * n.C + c] = make_float2(u, v);
            const float w = param<T>(n, n.w, c, 1.f);
            s1 = fmaf(w, u, s1);
            s2 = fmaf(w, v, s2);
        }
    }
    const float inv_m = 1.f / ((float)n.P * n.cg);
    s1 = block_sum(s1, red);
    s2 = block_sum(s2, red);
    if (threadIdx.x == 0) group[(long long)b * n.G + blockIdx.x] = make_float2(s1 * inv_m, s2 * inv_m);
}

template <typename T, int N, bool SILU>
__global__ void __launch_bounds__(kThreads) norm_grad_kernel(const Norm n, const Pass s, const float2* __restrict__ group) {
    const int col = threadIdx.x % s.cols_p2, row = threadIdx.x / s.cols_p2, rows = kThreads / s.cols_p2;
    const int vec = blockIdx.z * s.cols_p2 + col;
    const int b = s.b0 + s.batches - 1 - blockIdx.y;
    const long long run = s.runs - 1 - blockIdx.x, p0 = run * s.run, p1 = min(n.P, p0 + s.run);
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    if (vec >= s.cols) return;
    const Column<T, N> k(n, b, vec * N);
    float s1[N], s2[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float2 g = group[(long long)b * n.G + (vec * N + i) / n.cg];
        s1[i] = g.x;
        s2[i] = g.y;
    }
    const T* x0 = static_cast<const T*>(n.x.ptr) + b * n.x.b + vec * N;
    const T* g0 = static_cast<const T*>(n.d_y.ptr) + b * n.d_y.b + vec * N;
    T* dst = static_cast<T*>(n.d_x) + (long long)b * n.P * n.C + vec * N;
#pragma unroll 4
    for (long long p = p1 - 1 - row; p >= p0; p -= rows) {
        Vec<T, N> x, g;
        float f[N], e[N];
        x.load(x0 + p * n.x.p);
        g.load(g0 + p * n.d_y.p);
        x.widened(f);
        g.widened(e);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float xhat = (f[i] - k.mean[i]) * k.rstd[i], dz = e[i] * slope<SILU>(fmaf(xhat, k.w[i], k.bias[i]));
            f[i] = k.rstd[i] * (fmaf(dz, k.w[i], -s1[i]) - xhat * s2[i]);
        }
        x.round(f);
        x.store(dst + p * n.C);
    }
}

// d_weight and d_bias: the batch entries' sums, in their order.
template <typename W>
__global__ void __launch_bounds__(kThreads) norm_params_kernel(const float2* __restrict__ sums, W* __restrict__ d_w, W* __restrict__ d_b, int B, int C) {
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= C) return;
    float u = 0.f, v = 0.f;
#pragma unroll 4
    for (int b = 0; b < B; ++b) {
        const float2 x = sums[(long long)b * C + c];
        u += x.x;
        v += x.y;
    }
    if (d_b) d_b[c] = na2d_vec::narrow<W>(u);
    if (d_w) d_w[c] = na2d_vec::narrow<W>(v);
}

// ---- host ---------------------------------------------------------------------------------------------------------------
constexpr int kChipBytes = 100 << 10;           // shared memory of a block on the chip: two blocks an SM
constexpr long long kL2Bytes = 48ll << 20;      // what the two passes take of batch entries at a time: under half of L2

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

// The two passes: batch entries at a time, and runs so that a pass has about four blocks an SM.
Pass pass_plan(const Norm& n, int esize, int vec, bool backward) {
    Pass s{};
    s.cols = n.C / vec;
    s.cols_p2 = std::min(power_of_two(s.cols), 64);
    const long long bytes = n.P * n.C * esize * (backward ? 2 : 1);
    s.batches = (int)std::max(1LL, std::min<long long>(n.B, kL2Bytes / std::max(1LL, bytes)));
    const long long blocks = (long long)s.batches * ((s.cols + s.cols_p2 - 1) / s.cols_p2);
    const long long runs = std::max(1LL, std::min((4LL * 148 + blocks - 1) / blocks, (n.P + 31) / 32));
    s.run = (n.P + runs - 1) / runs;
    s.runs = (int)((n.P + s.run - 1) / s.run);
    return s;
}

int make_norm(const na2d_norm_args* a, Norm* n) {
    if (!a || a->struct_size < sizeof(na2d_norm_args)) return NA2D_ERR_BAD_ARG;
    if (a->B <= 0 || a->C <= 0 || a->P <= 0 || a->groups <= 0 || a->C % a->groups != 0) return NA2D_ERR_BAD_ARG;
    if (a->dtype != NA2D_F32 && a->dtype != NA2D_BF16 && a->dtype != NA2D_F16) return NA2D_ERR_UNSUPPORTED;
    if (a->param_dtype != NA2D_F32 && a->param_dtype != a->dtype) return NA2D_ERR_UNSUPPORTED;
    if (a->activation != NA2D_ACT_NONE && a->activation != NA2D_ACT_SILU) return NA2D_ERR_BAD_ARG;
    if (!(a->eps >= 0.f) || !(a->eps < 3.0e38f)) return NA2D_ERR_BAD_ARG;
    if (a->workspace && reinterpret_cast<uintptr_t>(a->workspace) % 16) return NA2D_ERR_BAD_ARG;
    if (a->B > 65535 || a->C > (1 << 20) || a->P > (1ll << 40)) return NA2D_ERR_TOO_LARGE;
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

template <typename K, typename... A>
int launch_chip(K kernel, const Slab& s, int B, size_t smem, cudaStream_t st, A... args) {
    const long long blocks = (long long)B * s.slabs * s.cluster;
    if (blocks > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kChipBytes);
        if (e != cudaSuccess) return na2d_host::cuda_fail(e, "cudaFuncSetAttribute");
    }
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

template <typename K, typename... A>
int launch_pass(K kernel, const Pass& s, int vec, int smem_floats, cudaStream_t st, A... args) {
    (void)vec;
    const dim3 grid(s.runs, s.batches, (s.cols + s.cols_p2 - 1) / s.cols_p2);
    return launched(na2d_launch::launch(true, kernel, grid, kThreads, (size_t)smem_floats * sizeof(float), st, args...), "group norm launch");
}

// Floats that a block of a pass keeps: two for each channel and row, and a count a row.
int pass_floats(const Pass& s, int vec) { return kThreads * vec * 2 + kThreads / s.cols_p2; }

// Workspace: the runs' float2 values, then (backward) the channels' and the groups'.
size_t run_values(const Norm& n, const Pass& s) { return (size_t)s.batches * s.runs * n.C; }
size_t workspace_bytes(const Norm& n, int dtype, bool backward) {
    const int esize = dtype == NA2D_F32 ? 4 : 2;
    Slab slab;
    const size_t own = backward ? (size_t)n.B * (n.C + n.G) : 0;
    size_t runs = 0;                    // with the vectors that need most: results need not have been allocated when this is asked
    for (int v : {16 / esize, 8 / esize, 1})
        if (n.C % v == 0 && !chip_plan(n, esize, v, backward, &slab)) runs = std::max(runs, run_values(n, pass_plan(n, esize, v, backward)));
    return (runs + own) * sizeof(float2);
}

template <typename T, int N, bool SILU>
int forward_as(const na2d_norm_args* a, const Norm& n, cudaStream_t st) {
    Slab slab;
    if (chip_plan(n, sizeof(T), N, false, &slab))
        return launch_chip(norm_chip_fwd_kernel<T, N, SILU>, slab, n.B, chip_bytes(slab, sizeof(T), 1), st, n, slab);
    Pass s = pass_plan(n, sizeof(T), N, false);
    if (!a->workspace || a->workspace_bytes < run_values(n, s) * sizeof(float2)) return NA2D_ERR_BAD_ARG;
    float2* part = static_cast<float2*>(a->workspace);
    const int batches = s.batches;
    for (s.b0 = 0; s.b0 < n.B; s.b0 += batches) {
        s.batches = std::min(batches, n.B - s.b0);
        if (int rc = launch_pass(norm_stats_kernel<T, N>, s, N, pass_floats(s, N), st, n, s, part)) return rc;
        if (int rc = launched(na2d_launch::launch(true, norm_finish_stats_kernel, dim3(n.G, s.batches), kThreads, 0, st, n, s, (const float2*)part),
                              "group norm launch"))
            return rc;
        if (int rc = launch_pass(norm_apply_kernel<T, N, SILU>, s, N, 0, st, n, s)) return rc;
    }
    return NA2D_OK;
}

template <typename T, int N, bool SILU>
int backward_as(const na2d_norm_args* a, const Norm& n, cudaStream_t st) {
    Slab slab;
    const bool chip = chip_plan(n, sizeof(T), N, true, &slab), params = a->d_weight || a->d_bias;
    Pass s = pass_plan(n, sizeof(T), N, true);
    const size_t runs = chip ? 0 : run_values(n, s);
    if (!a->workspace || a->workspace_bytes < (runs + (size_t)n.B * (n.C + n.G)) * sizeof(float2)) return NA2D_ERR_BAD_ARG;
    float2 *part = static_cast<float2*>(a->workspace), *sums = part + runs, *group = sums + (size_t)n.B * n.C;
    if (chip) {
        if (int rc = launch_chip(norm_chip_bwd_kernel<T, N, SILU>, slab, n.B, chip_bytes(slab, sizeof(T), 2), st, n, slab, params ? sums : nullptr))
            return rc;
    } else {
        const int batches = s.batches;
        for (s.b0 = 0; s.b0 < n.B; s.b0 += batches) {
            s.batches = std::min(batches, n.B - s.b0);
            if (int rc = launch_pass(norm_grad_sums_kernel<T, N, SILU>, s, N, pass_floats(s, N), st, n, s, part)) return rc;
            if (int rc = launched(na2d_launch::launch(true, norm_finish_sums_kernel<T>, dim3(n.G, s.batches), kThreads, 0, st, n, s,
                                                      (const float2*)part, sums, group), "group norm launch"))
                return rc;
            if (!n.d_x) continue;
            if (int rc = launch_pass(norm_grad_kernel<T, N, SILU>, s, N, 0, st, n, s, (const float2*)group)) return rc;
        }
    }
    if (!params) return NA2D_OK;
    auto finish = [&](auto tag) {
        using W = typename decltype(tag)::type;
        return launched(na2d_launch::launch(true, norm_params_kernel<W>, dim3((n.C + kThreads - 1) / kThreads), kThreads, 0, st,
                                            (const float2*)sums, (W*)a->d_weight, (W*)a->d_bias, n.B, n.C), "group norm launch");
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
    return make_norm(a, &n) == NA2D_OK ? workspace_bytes(n, a->dtype, backward != 0) : 0;
}

}  // extern "C"
