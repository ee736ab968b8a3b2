// Attention over all keys on CUDA cores: fp32, head dims that are no multiple of 8 or beyond 128, and any strides.
//
// A block has BT query rows (or keys) and walks the other side in tiles of BT, in fp32.  256 threads as 16 x 16; a thread has a
// (BT / 16)^2 piece of a score tile and (BT / 16) x (CP / 16) sums of an output tile, all in registers.  Tiles lie in shared memory as
// rows of CP + 4 floats, so that the 16-byte loads of a column of threads fall into different banks.
// What bounds it: the multiply-adds, and beside them shared memory (12 wavefronts for 64 multiply-adds a thread).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "na2d_attn_entry.h"

namespace na2d_attn {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ float narrow<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }

template <int CP>
struct SimtCfg {
    static constexpr int BT = CP <= 128 ? 64 : 32;       // rows of a tile
    static constexpr int R = BT / 16;                    // rows and columns of a thread's piece of a score tile
    static constexpr int NC = CP / 16;                   // columns of a thread's output row: 4 at 4 tx + 64 j (2 at 2 tx for CP 32)
    static constexpr int LD = CP + 4, LS = BT + 4;
    static constexpr int TILE = BT * LD, SCORES = BT * LS;       // floats
};

// Rows [row0, row0 + BT) of a (T, C) operand as a tile; zeros beyond `rows` and beyond C.
template <typename DT, int CP>
__device__ __forceinline__ void load_tile(float* dst, const DT* src, long long stride, int row0, int rows, int C, bool vec) {
    using S = SimtCfg<CP>;
    if (vec) {                                           // fp32 on 16-byte boundaries, C a multiple of 4
        for (int i = threadIdx.x; i < S::BT * (CP / 4); i += kThreads) {
            const int r = i / (CP / 4), c = 4 * (i % (CP / 4));
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row0 + r < rows && c < C) v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + (row0 + r) * stride + c);
            *reinterpret_cast<float4*>(dst + r * S::LD + c) = v;
        }
    } else {
        for (int i = threadIdx.x; i < S::BT * CP; i += kThreads) {
            const int r = i / CP, c = i % CP;
            dst[r * S::LD + c] = row0 + r < rows && c < C ? widen(src[(row0 + r) * stride + c]) : 0.f;
        }
    }
}

// s[i][j] = a row (ty + 16 i) . b row (tx + 16 j)
template <int CP>
__device__ __forceinline__ void dot_tile(const float* a, const float* b, float (&s)[SimtCfg<CP>::R][SimtCfg<CP>::R], int tx, int ty) {
    using S = SimtCfg<CP>;
#pragma unroll
    for (int i = 0; i < S::R; ++i)
#pragma unroll
        for (int j = 0; j < S::R; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int c = 0; c < CP; c += 4) {
        float4 x[S::R], y[S::R];
#pragma unroll
        for (int i = 0; i < S::R; ++i) x[i] = *reinterpret_cast<const float4*>(a + (ty + 16 * i) * S::LD + c);
#pragma unroll
        for (int j = 0; j < S::R; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * S::LD + c);
#pragma unroll
        for (int i = 0; i < S::R; ++i)
#pragma unroll
            for (int j = 0; j < S::R; ++j)
                s[i][j] = fmaf(x[i].w, y[j].w, fmaf(x[i].z, y[j].z, fmaf(x[i].y, y[j].y, fmaf(x[i].x, y[j].x, s[i][j]))));
    }
}

// First channel of the k-th pair of a thread's output columns.
template <int CP>
__device__ __forceinline__ int out_col(int tx, int k) {
    return CP == 32 ? 2 * tx + 32 * k : 4 * tx + 64 * (k / 2) + 2 * (k % 2);
}

// acc[i][] += sum_k w[row ty + 16 i][k] b[k][], w in rows of LS floats
template <int CP>
__device__ __forceinline__ void apply_tile(const float* w, const float* b, float (&acc)[SimtCfg<CP>::R][SimtCfg<CP>::NC], int tx, int ty) {
    using S = SimtCfg<CP>;
#pragma unroll 2
    for (int k = 0; k < S::BT; k += 4) {
        float4 x[S::R];
#pragma unroll
        for (int i = 0; i < S::R; ++i) x[i] = *reinterpret_cast<const float4*>(w + (ty + 16 * i) * S::LS + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            float y[S::NC];
            if constexpr (CP == 32) {
                const float2 v = *reinterpret_cast<const float2*>(b + (k + kk) * S::LD + 2 * tx);
                y[0] = v.x;
                y[1] = v.y;
            } else {
#pragma unroll
                for (int j = 0; j < S::NC / 4; ++j)
                    *reinterpret_cast<float4*>(y + 4 * j) = *reinterpret_cast<const float4*>(b + (k + kk) * S::LD + 4 * tx + 64 * j);
            }
#pragma unroll
            for (int i = 0; i < S::R; ++i) {
                const float xi = kk == 0 ? x[i].x : kk == 1 ? x[i].y : kk == 2 ? x[i].z : x[i].w;
#pragma unroll
                for (int c = 0; c < S::NC; ++c) acc[i][c] = fmaf(xi, y[c], acc[i][c]);
            }
        }
    }
}

template <typename DT, int CP>
__device__ __forceinline__ void store_rows(DT* dst, long long stride, int row0, int rows, int C,
                                           const float (&acc)[SimtCfg<CP>::R][SimtCfg<CP>::NC], const float (&scale)[SimtCfg<CP>::R], int tx, int ty) {
    using S = SimtCfg<CP>;
#pragma unroll
    for (int i = 0; i < S::R; ++i) {
        const int r = row0 + ty + 16 * i;
        if (r >= rows) continue;
#pragma unroll
        for (int k = 0; k < S::NC / 2; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = out_col<CP>(tx, k) + e;
                if (c < C) dst[r * stride + c] = narrow<DT>(acc[i][2 * k + e] * scale[i]);
            }
    }
}

// Sum (or maximum) over the 16 threads of a row: half a warp.
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
__device__ __forceinline__ float row_max(float x) {
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}

template <typename DT>
__device__ __forceinline__ DT* rows_of(const Operand& x, int b, int n) { return static_cast<DT*>(x.ptr) + b * x.b + n * x.n; }

// ---- forward: a block has BT queries of one head ------------------------------------------------------------------
template <typename DT, int CP>
__global__ void __launch_bounds__(kThreads)
simt_fwd_kernel(const Operand q, const Operand k, const Operand v, const Operand o, float* __restrict__ lse, const Geom g, const int tiles, const int vec) {
    using S = SimtCfg<CP>;
    extern __shared__ __align__(16) float smem[];
    float *sQ = smem, *sKV = sQ + S::TILE, *sP = sKV + S::TILE;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int bn = blockIdx.x / tiles, b = bn / g.N, n = bn - b * g.N, m = n / g.G;
    const int t0 = (g.causal ? tiles - 1 - (int)(blockIdx.x % tiles) : (int)(blockIdx.x % tiles)) * S::BT;
    const int count = key_count(g, b), keys = keys_seen(g, count, min(t0 + S::BT, g.Tq) - 1);
    load_tile<DT, CP>(sQ, rows_of<DT>(q, b, n), q.t, t0, g.Tq, g.C, vec);
    float acc[S::R][S::NC], top[S::R], total[S::R];
#pragma unroll
    for (int i = 0; i < S::R; ++i) {
        top[i] = -CUDART_INF_F;
        total[i] = 0.f;
#pragma unroll
        for (int c = 0; c < S::NC; ++c) acc[i][c] = 0.f;
    }
    for (int k0 = 0; k0 < keys; k0 += S::BT) {
        __syncthreads();
        load_tile<DT, CP>(sKV, rows_of<DT>(k, b, m), k.t, k0, count, g.C, vec);
        __syncthreads();
        float s[S::R][S::R];
        dot_tile<CP>(sQ, sKV, s, tx, ty);
#pragma unroll
        for (int i = 0; i < S::R; ++i) {
            const int t = t0 + ty + 16 * i, seen = t < g.Tq ? keys_seen(g, count, t) : 0;
            float high = top[i];
#pragma unroll
            for (int j = 0; j < S::R; ++j) {
                s[i][j] = k0 + tx + 16 * j < seen ? s[i][j] * g.sl2 : -CUDART_INF_F;
                high = fmaxf(high, s[i][j]);
            }
            high = row_max(high);
            const float base = high == -CUDART_INF_F ? 0.f : high, old = exp2f(top[i] - base);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < S::R; ++j) {
                s[i][j] = exp2f(s[i][j] - base);
                sum += s[i][j];
                sP[(ty + 16 * i) * S::LS + tx + 16 * j] = s[i][j];
            }
            total[i] = fmaf(total[i], old, sum);
            top[i] = high;
#pragma unroll
            for (int c = 0; c < S::NC; ++c) acc[i][c] *= old;
        }
        __syncthreads();
        load_tile<DT, CP>(sKV, rows_of<DT>(v, b, m), v.t, k0, count, g.C, vec);
        __syncthreads();
        apply_tile<CP>(sP, sKV, acc, tx, ty);
    }
    float inv[S::R];
#pragma unroll
    for (int i = 0; i < S::R; ++i) {
        const float sum = row_sum(total[i]);
        inv[i] = sum == 0.f ? 0.f : 1.f / sum;
        const int t = t0 + ty + 16 * i;
        if (tx == 0 && t < g.Tq)
            lse[row_index(g, b, n, t)] = sum == 0.f ? -CUDART_INF_F : (top[i] + log2f(sum)) * na2d_tc::kLn2;
    }
    store_rows<DT, CP>(rows_of<DT>(o, b, n), o.t, t0, g.Tq, g.C, acc, inv, tx, ty);
}

// ---- delta = dO . o, a warp a row -------------------------------------------------------------------------------------
template <typename DT>
__global__ void __launch_bounds__(kThreads) simt_delta_kernel(const Operand d_o, const Operand o, float* __restrict__ delta, const Geom g) {
    const long long rows = (long long)g.B * g.N * g.Tq, row = (long long)blockIdx.x * 8 + threadIdx.x / 32;
    if (row >= rows) return;
    const long long bn = row / g.Tq;
    const int t = (int)(row % g.Tq), b = (int)(bn / g.N), n = (int)(bn % g.N);
    const DT *x = rows_of<DT>(d_o, b, n) + t * d_o.t, *y = rows_of<DT>(o, b, n) + t * o.t;
    float acc = 0.f;
    for (int c = threadIdx.x % 32; c < g.C; c += 32) acc = fmaf(widen(x[c]), widen(y[c]), acc);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, d);
    if (threadIdx.x % 32 == 0) delta[row] = acc;
}

// ---- query half of the backward -----------------------------------------------------------------------------------------
template <typename DT, int CP>
__global__ void __launch_bounds__(kThreads)
simt_dq_kernel(const Operand q, const Operand k, const Operand v, const Operand d_o, const Operand d_q, const float* __restrict__ lse,
               const float* __restrict__ delta, const Geom g, const int tiles, const int vec) {
    using S = SimtCfg<CP>;
    extern __shared__ __align__(16) float smem[];
    float *sQ = smem, *sG = sQ + S::TILE, *sKV = sG + S::TILE, *sP = sKV + S::TILE;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int bn = blockIdx.x / tiles, b = bn / g.N, n = bn - b * g.N, m = n / g.G;
    const int t0 = (g.causal ? tiles - 1 - (int)(blockIdx.x % tiles) : (int)(blockIdx.x % tiles)) * S::BT;
    const int count = key_count(g, b), keys = keys_seen(g, count, min(t0 + S::BT, g.Tq) - 1);
    load_tile<DT, CP>(sQ, rows_of<DT>(q, b, n), q.t, t0, g.Tq, g.C, vec);
    load_tile<DT, CP>(sG, rows_of<DT>(d_o, b, n), d_o.t, t0, g.Tq, g.C, vec);
    float acc[S::R][S::NC], neg[S::R], del[S::R], scale[S::R];
    int seen[S::R];
#pragma unroll
    for (int i = 0; i < S::R; ++i) {
        const int t = t0 + ty + 16 * i;
        seen[i] = t < g.Tq ? keys_seen(g, count, t) : 0;
        neg[i] = seen[i] ? -lse[row_index(g, b, n, t)] * na2d_tc::kLog2e : 0.f;
        del[i] = seen[i] ? delta[row_index(g, b, n, t)] : 0.f;
        scale[i] = g.scale;
#pragma unroll
        for (int c = 0; c < S::NC; ++c) acc[i][c] = 0.f;
    }
    for (int k0 = 0; k0 < keys; k0 += S::BT) {
        __syncthreads();
        load_tile<DT, CP>(sKV, rows_of<DT>(v, b, m), v.t, k0, count, g.C, vec);
        __syncthreads();
        float dp[S::R][S::R], s[S::R][S::R];
        dot_tile<CP>(sG, sKV, dp, tx, ty);
        __syncthreads();
        load_tile<DT, CP>(sKV, rows_of<DT>(k, b, m), k.t, k0, count, g.C, vec);
        __syncthreads();
        dot_tile<CP>(sQ, sKV, s, tx, ty);
#pragma unroll
        for (int i = 0; i < S::R; ++i)
#pragma unroll
            for (int j = 0; j < S::R; ++j)
                sP[(ty + 16 * i) * S::LS + tx + 16 * j] =
                    k0 + tx + 16 * j < seen[i] ? exp2f(fmaf(s[i][j], g.sl2, neg[i])) * (dp[i][j] - del[i]) : 0.f;
        __syncthreads();
        apply_tile<CP>(sP, sKV, acc, tx, ty);
    }
    store_rows<DT, CP>(rows_of<DT>(d_q, b, n), d_q.t, t0, g.Tq, g.C, acc, scale, tx, ty);
}

// ---- key half: a block has BT keys of one key head and walks the queries of every head that shares it ------------------------
template <typename DT, int CP>
__global__ void __launch_bounds__(kThreads)
simt_dkdv_kernel(const Operand q, const Operand k, const Operand v, const Operand d_o, const Operand d_k, const Operand d_v,
                 const float* __restrict__ lse, const float* __restrict__ delta, const Geom g, const int tiles, const int vec) {
    using S = SimtCfg<CP>;
    extern __shared__ __align__(16) float smem[];
    float *sK = smem, *sV = sK + S::TILE, *sX = sV + S::TILE, *sP = sX + S::TILE;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int unit = blockIdx.x / tiles, b = unit / g.Nk, m = unit - b * g.Nk;
    const int k0 = (blockIdx.x % tiles) * S::BT;
    const int count = key_count(g, b);
    const int t_min = g.causal ? max(k0 + g.Tq - count, 0) : 0;      // the first token that sees the tile
    load_tile<DT, CP>(sK, rows_of<DT>(k, b, m), k.t, k0, count, g.C, vec);
    load_tile<DT, CP>(sV, rows_of<DT>(v, b, m), v.t, k0, count, g.C, vec);
    float acc_k[S::R][S::NC], acc_v[S::R][S::NC], scale_k[S::R], scale_v[S::R];
#pragma unroll
    for (int i = 0; i < S::R; ++i) {
        scale_k[i] = g.scale;
        scale_v[i] = 1.f;
#pragma unroll
        for (int c = 0; c < S::NC; ++c) acc_k[i][c] = acc_v[i][c] = 0.f;
    }
    for (int n = m * g.G; k0 < count && n < (m + 1) * g.G; ++n) {
        for (int t0 = t_min / S::BT * S::BT; t0 < g.Tq; t0 += S::BT) {
            // rows of a piece are keys (ty), columns queries (tx)
            __syncthreads();
            load_tile<DT, CP>(sX, rows_of<DT>(q, b, n), q.t, t0, g.Tq, g.C, vec);
            __syncthreads();
            float p[S::R][S::R], dp[S::R][S::R];
            dot_tile<CP>(sK, sX, p, tx, ty);
            float del[S::R];
#pragma unroll
            for (int j = 0; j < S::R; ++j) {
                const int t = t0 + tx + 16 * j, seen = t < g.Tq ? keys_seen(g, count, t) : 0;
                const float neg = seen ? -lse[row_index(g, b, n, t)] * na2d_tc::kLog2e : 0.f;
                del[j] = seen ? delta[row_index(g, b, n, t)] : 0.f;
#pragma unroll
                for (int i = 0; i < S::R; ++i) p[i][j] = k0 + ty + 16 * i < seen ? exp2f(fmaf(p[i][j], g.sl2, neg)) : 0.f;
            }
            __syncthreads();
            load_tile<DT, CP>(sX, rows_of<DT>(d_o, b, n), d_o.t, t0, g.Tq, g.C, vec);
#pragma unroll
            for (int i = 0; i < S::R; ++i)
#pragma unroll
                for (int j = 0; j < S::R; ++j) sP[(ty + 16 * i) * S::LS + tx + 16 * j] = p[i][j];
            __syncthreads();
            dot_tile<CP>(sV, sX, dp, tx, ty);
            apply_tile<CP>(sP, sX, acc_v, tx, ty);
            __syncthreads();
            load_tile<DT, CP>(sX, rows_of<DT>(q, b, n), q.t, t0, g.Tq, g.C, vec);
#pragma unroll
            for (int i = 0; i < S::R; ++i)
#pragma unroll
                for (int j = 0; j < S::R; ++j)       // (by selection: what is not seen may hold anything)
                    sP[(ty + 16 * i) * S::LS + tx + 16 * j] = p[i][j] == 0.f ? 0.f : p[i][j] * (dp[i][j] - del[j]);
            __syncthreads();
            apply_tile<CP>(sP, sX, acc_k, tx, ty);
        }
    }
    store_rows<DT, CP>(rows_of<DT>(d_k, b, m), d_k.t, k0, g.Tk, g.C, acc_k, scale_k, tx, ty);
    store_rows<DT, CP>(rows_of<DT>(d_v, b, m), d_v.t, k0, g.Tk, g.C, acc_v, scale_v, tx, ty);
}

// ---- launchers ---------------------------------------------------------------------------------------------------------
template <typename DT, typename F>
int by_channels(int C, F&& f) {
    if (C <= 32) return f(std::integral_constant<int, 32>{});
    if (C <= 64) return f(std::integral_constant<int, 64>{});
    if (C <= 128) return f(std::integral_constant<int, 128>{});
    return f(std::integral_constant<int, 256>{});
}

bool vectors(const Operand& x, int dtype, int C) {
    return dtype == NA2D_F32 && C % 4 == 0 && reinterpret_cast<uintptr_t>(x.ptr) % 16 == 0 && x.b % 4 == 0 && x.n % 4 == 0 && x.t % 4 == 0;
}

// Blocks of `rows` in tiles, for each of `units`.
int blocks_of(long long units, int rows, int tile, int* tiles, unsigned* blocks) {
    *tiles = (rows + tile - 1) / tile;
    if (units * *tiles > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    *blocks = (unsigned)(units * *tiles);
    return NA2D_OK;
}

template <typename K, typename... A>
int start(const Place& at, K kernel, unsigned blocks, int floats, std::atomic<unsigned long long>& opted, A... args) {
    if (na2d_tc::opt_in_smem(kernel, floats * 4, at.device, opted) != cudaSuccess) return NA2D_ERR_CUDA;
    kernel<<<blocks, kThreads, floats * 4, at.st>>>(args...);
    *at.launched += 1;
    return cudaGetLastError() == cudaSuccess ? NA2D_OK : NA2D_ERR_CUDA;
}

template <typename DT, int CP>
int forward_as(const Place& at, const Geom& g, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse) {
    using S = SimtCfg<CP>;
    static std::atomic<unsigned long long> opted{0};
    const int vec = vectors(q, at.dtype, g.C) && vectors(k, at.dtype, g.C) && vectors(v, at.dtype, g.C);
    int tiles = 0;
    unsigned blocks = 0;
    if (int rc = blocks_of((long long)g.B * g.N, g.Tq, S::BT, &tiles, &blocks)) return rc;
    return start(at, simt_fwd_kernel<DT, CP>, blocks, 2 * S::TILE + S::SCORES, opted, q, k, v, o, lse, g, tiles, vec);
}

template <typename DT, int CP>
int backward_as(const Place& at, const Geom& g, const Backward& x) {
    using S = SimtCfg<CP>;
    static std::atomic<unsigned long long> opted_q{0}, opted_k{0};
    int vec = 1, tiles = 0;
    for (const Operand* t : {&x.q, &x.k, &x.v, &x.d_o}) vec = vec && vectors(*t, at.dtype, g.C);
    const long long rows = (long long)g.B * g.N * g.Tq;
    if ((rows + 7) / 8 > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    simt_delta_kernel<DT><<<(unsigned)((rows + 7) / 8), kThreads, 0, at.st>>>(x.d_o, x.o, x.delta, g);
    *at.launched += 1;
    if (cudaGetLastError() != cudaSuccess) return NA2D_ERR_CUDA;
    unsigned blocks = 0;
    if (x.d_q.ptr) {
        if (int rc = blocks_of((long long)g.B * g.N, g.Tq, S::BT, &tiles, &blocks)) return rc;
        if (int rc = start(at, simt_dq_kernel<DT, CP>, blocks, 3 * S::TILE + S::SCORES, opted_q, x.q, x.k, x.v, x.d_o, x.d_q, x.lse,
                           (const float*)x.delta, g, tiles, vec))
            return rc;
    }
    if (!x.d_k.ptr) return NA2D_OK;
    if (int rc = blocks_of(g.units, g.Tk, S::BT, &tiles, &blocks)) return rc;
    return start(at, simt_dkdv_kernel<DT, CP>, blocks, 3 * S::TILE + S::SCORES, opted_k, x.q, x.k, x.v, x.d_o, x.d_k, x.d_v, x.lse,
                 (const float*)x.delta, g, tiles, vec);
}

}  // namespace

int simt_forward(const Place& at, const Geom& g, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse) {
    auto run = [&](auto type) {
        using DT = decltype(type);
        return by_channels<DT>(g.C, [&](auto cp) { return forward_as<DT, decltype(cp)::value>(at, g, q, k, v, o, lse); });
    };
    return at.dtype == NA2D_F32 ? run(float{}) : at.dtype == NA2D_BF16 ? run(__nv_bfloat16{}) : run(__half{});
}

int simt_backward(const Place& at, const Geom& g, const Backward& x) {
    auto run = [&](auto type) {
        using DT = decltype(type);
        return by_channels<DT>(g.C, [&](auto cp) { return backward_as<DT, decltype(cp)::value>(at, g, x); });
    };
    return at.dtype == NA2D_F32 ? run(float{}) : at.dtype == NA2D_BF16 ? run(__nv_bfloat16{}) : run(__half{});
}

}  // namespace na2d_attn
