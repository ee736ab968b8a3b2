// Attention over all keys on CUDA cores: fp32, head dims that are no multiple of 8 or beyond 128, and any strides.
//
// A block has 128 or 64 query rows (or 64 keys) and walks the other side in tiles, in fp32; the next tile is on its way to registers
// meanwhile.  256 threads as 16 x 16; a thread has 8 x 4 (4 x 4) of a score tile and its rows' part of an output tile, all in registers, and
// multiplies and adds two channels at a time.  Tiles lie in shared memory as rows of CP + 4 floats, so that the 16-byte loads of a column
// of threads fall into different banks; neighbouring lanes are two rows of one column, because a warp's 16-byte loads are shared between
// neighbours only (with 16 columns side by side each load took its full four turns: 1305 us against 1209).
// What bounds it: the multiply-adds, and beside them the loads from shared memory.  Batch 4, 4 heads of 128, 1024 tokens, fp32, forward and
// backward: 1130 us, 34 TFLOP/s over the nine products that are done (the seven that have to be: 406 us at the 74 TFLOP/s that 148 SMs of 128
// multiply-adds come to at 1965 MHz).
#include "na2d_attn_entry.h"
#include "na2d_vec.cuh"

namespace na2d_attn {

namespace {

constexpr int kThreads = 256;

using na2d_vec::narrow;
using na2d_vec::widen;

// BM rows of one side stay, tiles of BT of the other pass by.
template <int CP, int BM>
struct SimtCfg {
    static constexpr int BT = CP <= 128 ? 64 : 32;
    static constexpr int RM = BM / 16, R = BT / 16;      // rows and columns of a thread's piece of a score tile
    static constexpr int NC = CP / 16;                   // columns of a thread's output row: 4 at 4 tx + 64 j (2 at 2 tx for CP 32)
    static constexpr int LD = CP + 4, LS = BT + 4;
    static constexpr int HELD = BM * LD, TILE = BT * LD, SCORES = BM * LS;       // floats
};

// Rows [row0, row0 + BT) of a (T, C) operand on their way to a tile, in registers (`fetch`, well ahead) and then in shared memory (`put`);
// zeros beyond `rows` and beyond C.
template <typename DT, int CP, int ROWS>
struct Tile {
    static constexpr int LD = CP + 4, K = ROWS * CP / 4 / kThreads;              // pieces of 4 channels a thread
    float4 piece[K];
    __device__ __forceinline__ void fetch(const DT* src, long long stride, int row0, int rows, int C, bool vec) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = threadIdx.x + k * kThreads, r = i / (CP / 4), c = 4 * (i % (CP / 4));
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row0 + r < rows) {
                const DT* at = src + (row0 + r) * stride + c;
                if (vec) {                                           // fp32 on 16-byte boundaries, C a multiple of 4
                    if (c < C) v = __ldg(reinterpret_cast<const float4*>(at));
                } else {
                    if (c < C) v.x = widen(at[0]);
                    if (c + 1 < C) v.y = widen(at[1]);
                    if (c + 2 < C) v.z = widen(at[2]);
                    if (c + 3 < C) v.w = widen(at[3]);
                }
            }
            piece[k] = v;
        }
    }
    // One after the other, for rows that stay.
    static __device__ __forceinline__ void bring(float* dst, const DT* src, long long stride, int row0, int rows, int C, bool vec) {
        Tile<DT, CP, ROWS / 2> half;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
            half.fetch(src, stride, row0 + h * (ROWS / 2), rows, C, vec);
            half.put(dst + h * (ROWS / 2) * LD);
        }
    }
    __device__ __forceinline__ void put(float* dst) const {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = threadIdx.x + k * kThreads;
            *reinterpret_cast<float4*>(dst + (i / (CP / 4)) * LD + 4 * (i % (CP / 4))) = piece[k];
        }
    }
};

// s[i][j] = a row (ty + 16 i) . b row (tx + 16 j).  Two channels' sums side by side: a packed multiply-add leaves every other issue slot to
// the loads.
template <int CP, int BM>
__device__ __forceinline__ void dot_tile(const float* a, const float* b, float (&s)[BM / 16][SimtCfg<CP, BM>::R], int tx, int ty) {
    using S = SimtCfg<CP, BM>;
    uint64_t sum[S::RM][S::R];
#pragma unroll
    for (int i = 0; i < S::RM; ++i)
#pragma unroll
        for (int j = 0; j < S::R; ++j) sum[i][j] = 0;
#pragma unroll 4
    for (int c = 0; c < CP; c += 4) {
        ulonglong2 x[S::RM], y[S::R];
#pragma unroll
        for (int i = 0; i < S::RM; ++i) x[i] = *reinterpret_cast<const ulonglong2*>(a + (ty + 16 * i) * S::LD + c);
#pragma unroll
        for (int j = 0; j < S::R; ++j) y[j] = *reinterpret_cast<const ulonglong2*>(b + (tx + 16 * j) * S::LD + c);
#pragma unroll
        for (int i = 0; i < S::RM; ++i)
#pragma unroll
            for (int j = 0; j < S::R; ++j) sum[i][j] = na2d_ptx::fma2(x[i].x, y[j].x, sum[i][j]);
#pragma unroll
        for (int i = 0; i < S::RM; ++i)
#pragma unroll
            for (int j = 0; j < S::R; ++j) sum[i][j] = na2d_ptx::fma2(x[i].y, y[j].y, sum[i][j]);
    }
#pragma unroll
    for (int i = 0; i < S::RM; ++i)
#pragma unroll
        for (int j = 0; j < S::R; ++j) s[i][j] = na2d_ptx::lo2(sum[i][j]) + na2d_ptx::hi2(sum[i][j]);
}

// First channel of the k-th pair of a thread's output columns.
template <int CP>
__device__ __forceinline__ int out_col(int tx, int k) {
    return CP == 32 ? 2 * tx + 32 * k : 4 * tx + 64 * (k / 2) + 2 * (k % 2);
}

// A thread's part of an output tile, in pairs of columns.
template <int CP, int BM>
struct Sums {
    using S = SimtCfg<CP, BM>;
    uint64_t at[S::RM][S::NC / 2];
    __device__ __forceinline__ Sums() {
#pragma unroll
        for (int i = 0; i < S::RM; ++i)
#pragma unroll
            for (int c = 0; c < S::NC / 2; ++c) at[i][c] = 0;
    }
    // += sum_k w[row ty + 16 i][k] b[k][], w in rows of LS floats
    __device__ __forceinline__ void add(const float* w, const float* b, int tx, int ty) {
#pragma unroll 2
        for (int k = 0; k < S::BT; k += 4) {
            float4 x[S::RM];
#pragma unroll
            for (int i = 0; i < S::RM; ++i) x[i] = *reinterpret_cast<const float4*>(w + (ty + 16 * i) * S::LS + k);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                uint64_t y[S::NC / 2];
                if constexpr (CP == 32) {
                    y[0] = *reinterpret_cast<const uint64_t*>(b + (k + kk) * S::LD + 2 * tx);
                } else {
#pragma unroll
                    for (int j = 0; j < S::NC / 4; ++j) {
                        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(b + (k + kk) * S::LD + 4 * tx + 64 * j);
                        y[2 * j] = v.x;
                        y[2 * j + 1] = v.y;
                    }
                }
#pragma unroll
                for (int i = 0; i < S::RM; ++i) {
                    const float xi = kk == 0 ? x[i].x : kk == 1 ? x[i].y : kk == 2 ? x[i].z : x[i].w;
                    const uint64_t xx = na2d_ptx::pair2(xi, xi);
#pragma unroll
                    for (int c = 0; c < S::NC / 2; ++c) at[i][c] = na2d_ptx::fma2(xx, y[c], at[i][c]);
                }
            }
        }
    }
};

// (a scale of 0: a row that sees nothing, or a key that is none, whose products may be 0 times infinity)
template <typename DT, int CP, int BM>
__device__ __forceinline__ void store_rows(DT* dst, long long stride, int row0, int rows, int C,
                                           const Sums<CP, BM>& acc, const float (&scale)[BM / 16], int tx, int ty) {
    using S = SimtCfg<CP, BM>;
#pragma unroll
    for (int i = 0; i < S::RM; ++i) {
        const int r = row0 + ty + 16 * i;
        if (r >= rows) continue;
#pragma unroll
        for (int k = 0; k < S::NC / 2; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = out_col<CP>(tx, k) + e;
                const float x = (e ? na2d_ptx::hi2(acc.at[i][k]) : na2d_ptx::lo2(acc.at[i][k])) * scale[i];
                if (c < C) dst[r * stride + c] = narrow<DT>(scale[i] == 0.f ? 0.f : x);
            }
    }
}

// Sum (or maximum) over the 16 threads of a row: every other lane of a warp.
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int d = 16; d > 1; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
__device__ __forceinline__ float row_max(float x) {
#pragma unroll
    for (int d = 16; d > 1; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}

template <typename DT>
__device__ __forceinline__ DT* rows_of(const Operand& x, int b, int n) { return static_cast<DT*>(x.ptr) + b * x.b + n * x.n; }

// ---- forward: a block has BT queries of one head ------------------------------------------------------------------
template <typename DT, int CP, int BM>
__global__ void __launch_bounds__(kThreads)
simt_fwd_kernel(const Operand q, const Operand k, const Operand v, const Operand o, float* __restrict__ lse, const Geom g, const int tiles, const int vec) {
    using S = SimtCfg<CP, BM>;
    extern __shared__ __align__(16) float smem[];
    float *sQ = smem, *sKV = sQ + S::HELD, *sP = sKV + S::TILE;
    const int tx = threadIdx.x % 32 / 2, ty = threadIdx.x / 32 * 2 + threadIdx.x % 2;
    const int bn = blockIdx.x / tiles, b = bn / g.N, n = bn - b * g.N, m = n / g.G;
    const int t0 = (g.causal ? tiles - 1 - (int)(blockIdx.x % tiles) : (int)(blockIdx.x % tiles)) * BM;
    const int count = key_count(g, b), keys = keys_seen(g, count, min(t0 + BM, g.Tq) - 1);
    Tile<DT, CP, BM>::bring(sQ, rows_of<DT>(q, b, n), q.t, t0, g.Tq, g.C, vec);
    Tile<DT, CP, S::BT> tile;
    if (keys > 0) tile.fetch(rows_of<DT>(k, b, m), k.t, 0, count, g.C, vec);
    Sums<CP, BM> acc;
    float top[S::RM], total[S::RM];
#pragma unroll
    for (int i = 0; i < S::RM; ++i) {
        top[i] = -CUDART_INF_F;
        total[i] = 0.f;
    }
    for (int k0 = 0; k0 < keys; k0 += S::BT) {
        __syncthreads();
        tile.put(sKV);
        tile.fetch(rows_of<DT>(v, b, m), v.t, k0, count, g.C, vec);
        __syncthreads();
        float s[S::RM][S::R];
        dot_tile<CP, BM>(sQ, sKV, s, tx, ty);
#pragma unroll
        for (int i = 0; i < S::RM; ++i) {
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
            const uint64_t old2 = na2d_ptx::pair2(old, old);
#pragma unroll
            for (int c = 0; c < S::NC / 2; ++c) acc.at[i][c] = na2d_ptx::mul2(acc.at[i][c], old2);
        }
        __syncthreads();
        tile.put(sKV);
        if (k0 + S::BT < keys) tile.fetch(rows_of<DT>(k, b, m), k.t, k0 + S::BT, count, g.C, vec);
        __syncthreads();
        acc.add(sP, sKV, tx, ty);
    }
    float inv[S::RM];
#pragma unroll
    for (int i = 0; i < S::RM; ++i) {
        const float sum = row_sum(total[i]);
        inv[i] = sum == 0.f ? 0.f : 1.f / sum;
        const int t = t0 + ty + 16 * i;
        if (tx == 0 && t < g.Tq)
            lse[row_index(g, b, n, t)] = sum == 0.f ? -CUDART_INF_F : (top[i] + log2f(sum)) * na2d_tc::kLn2;
    }
    store_rows<DT, CP, BM>(rows_of<DT>(o, b, n), o.t, t0, g.Tq, g.C, acc, inv, tx, ty);
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
template <typename DT, int CP, int BM>
__global__ void __launch_bounds__(kThreads)
simt_dq_kernel(const Operand q, const Operand k, const Operand v, const Operand d_o, const Operand d_q, const float* __restrict__ lse,
               const float* __restrict__ delta, const Geom g, const int tiles, const int vec) {
    using S = SimtCfg<CP, BM>;
    extern __shared__ __align__(16) float smem[];
    float *sQ = smem, *sG = sQ + S::HELD, *sKV = sG + S::HELD, *sP = sKV + S::TILE;
    const int tx = threadIdx.x % 32 / 2, ty = threadIdx.x / 32 * 2 + threadIdx.x % 2;
    const int bn = blockIdx.x / tiles, b = bn / g.N, n = bn - b * g.N, m = n / g.G;
    const int t0 = (g.causal ? tiles - 1 - (int)(blockIdx.x % tiles) : (int)(blockIdx.x % tiles)) * BM;
    const int count = key_count(g, b), keys = keys_seen(g, count, min(t0 + BM, g.Tq) - 1);
    Tile<DT, CP, BM>::bring(sQ, rows_of<DT>(q, b, n), q.t, t0, g.Tq, g.C, vec);
    Tile<DT, CP, BM>::bring(sG, rows_of<DT>(d_o, b, n), d_o.t, t0, g.Tq, g.C, vec);
    Tile<DT, CP, S::BT> tile;
    if (keys > 0) tile.fetch(rows_of<DT>(v, b, m), v.t, 0, count, g.C, vec);
    Sums<CP, BM> acc;
    float neg[S::RM], del[S::RM], scale[S::RM];
#pragma unroll
    for (int i = 0; i < S::RM; ++i) {
        const int t = t0 + ty + 16 * i;
        const bool row = t < g.Tq && keys_seen(g, count, t) > 0;
        neg[i] = row ? -lse[row_index(g, b, n, t)] * na2d_tc::kLog2e : 0.f;
        del[i] = row ? delta[row_index(g, b, n, t)] : 0.f;
        scale[i] = row ? g.scale : 0.f;
    }
    for (int k0 = 0; k0 < keys; k0 += S::BT) {
        __syncthreads();
        tile.put(sKV);
        tile.fetch(rows_of<DT>(k, b, m), k.t, k0, count, g.C, vec);
        __syncthreads();
        float s[S::RM][S::R];
        dot_tile<CP, BM>(sG, sKV, s, tx, ty);
#pragma unroll
        for (int i = 0; i < S::RM; ++i)
#pragma unroll
            for (int j = 0; j < S::R; ++j) sP[(ty + 16 * i) * S::LS + tx + 16 * j] = s[i][j] - del[i];
        __syncthreads();
        tile.put(sKV);
        if (k0 + S::BT < keys) tile.fetch(rows_of<DT>(v, b, m), v.t, k0 + S::BT, count, g.C, vec);
        __syncthreads();
        dot_tile<CP, BM>(sQ, sKV, s, tx, ty);
#pragma unroll
        for (int i = 0; i < S::RM; ++i) {
            const int t = t0 + ty + 16 * i, seen = t < g.Tq ? keys_seen(g, count, t) : 0;
#pragma unroll
            for (int j = 0; j < S::R; ++j) {
                float* at = sP + (ty + 16 * i) * S::LS + tx + 16 * j;        // holds dP - delta, of this very thread
                *at = k0 + tx + 16 * j < seen ? exp2f(fmaf(s[i][j], g.sl2, neg[i])) * *at : 0.f;
            }
        }
        __syncwarp();
        acc.add(sP, sKV, tx, ty);
    }
    store_rows<DT, CP, BM>(rows_of<DT>(d_q, b, n), d_q.t, t0, g.Tq, g.C, acc, scale, tx, ty);
}

// ---- key half: a block has BT keys of one key head and walks the queries of every head that shares it ------------------------
template <typename DT, int CP>
__global__ void __launch_bounds__(kThreads)
simt_dkdv_kernel(const Operand q, const Operand k, const Operand v, const Operand d_o, const Operand d_k, const Operand d_v,
                 const float* __restrict__ lse, const float* __restrict__ delta, const Geom g, const int tiles, const int vec) {
    constexpr int BM = CP <= 128 ? 64 : 32;
    using S = SimtCfg<CP, BM>;
    extern __shared__ __align__(16) float smem[];
    float *sK = smem, *sV = sK + S::TILE, *sX = sV + S::TILE, *sY = sX + S::TILE, *sP = sY + S::TILE;
    const int tx = threadIdx.x % 32 / 2, ty = threadIdx.x / 32 * 2 + threadIdx.x % 2;
    const int unit = blockIdx.x / tiles, b = unit / g.Nk, m = unit - b * g.Nk;
    const int k0 = (blockIdx.x % tiles) * S::BT;
    const int count = key_count(g, b);
    const int t_min = g.causal ? max(k0 + g.Tq - count, 0) : 0;      // the first token that sees the tile
    Tile<DT, CP, BM> tile;
    tile.fetch(rows_of<DT>(k, b, m), k.t, k0, count, g.C, vec);
    tile.put(sK);
    tile.fetch(rows_of<DT>(v, b, m), v.t, k0, count, g.C, vec);
    tile.put(sV);
    Sums<CP, BM> acc_k, acc_v;
    float scale_k[S::R], scale_v[S::R];
#pragma unroll
    for (int i = 0; i < S::R; ++i) {
        const bool there = k0 + ty + 16 * i < count;
        scale_k[i] = there ? g.scale : 0.f;
        scale_v[i] = there ? 1.f : 0.f;
    }
    const int first = t_min / S::BT * S::BT;
    const bool any = k0 < count && first < g.Tq;
    if (any) tile.fetch(rows_of<DT>(q, b, m * g.G), q.t, first, g.Tq, g.C, vec);
    for (int n = m * g.G; any && n < (m + 1) * g.G; ++n) {
        for (int t0 = first; t0 < g.Tq; t0 += S::BT) {
            // rows of a piece are keys (ty), columns queries (tx).  Q stays in sX, dO goes to sY.
            __syncthreads();
            tile.put(sX);
            tile.fetch(rows_of<DT>(d_o, b, n), d_o.t, t0, g.Tq, g.C, vec);
            __syncthreads();
            float p[S::R][S::R], dp[S::R][S::R];
            dot_tile<CP, BM>(sK, sX, p, tx, ty);
            float del[S::R];
#pragma unroll
            for (int j = 0; j < S::R; ++j) {
                const int t = t0 + tx + 16 * j, seen = t < g.Tq ? keys_seen(g, count, t) : 0;
                const float neg = seen ? -lse[row_index(g, b, n, t)] * na2d_tc::kLog2e : 0.f;
                del[j] = seen ? delta[row_index(g, b, n, t)] : 0.f;
#pragma unroll
                for (int i = 0; i < S::R; ++i) p[i][j] = k0 + ty + 16 * i < seen ? exp2f(fmaf(p[i][j], g.sl2, neg)) : 0.f;
            }
            tile.put(sY);                                // (last read before the first barrier of this round)
            const bool more = t0 + S::BT < g.Tq;
            if (more || n + 1 < (m + 1) * g.G)
                tile.fetch(rows_of<DT>(q, b, more ? n : n + 1), q.t, more ? t0 + S::BT : first, g.Tq, g.C, vec);
#pragma unroll
            for (int i = 0; i < S::R; ++i)
#pragma unroll
                for (int j = 0; j < S::R; ++j) sP[(ty + 16 * i) * S::LS + tx + 16 * j] = p[i][j];
            __syncthreads();
            dot_tile<CP, BM>(sV, sY, dp, tx, ty);
            acc_v.add(sP, sY, tx, ty);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < S::R; ++i)
#pragma unroll
                for (int j = 0; j < S::R; ++j)       // (by selection: what is not seen may hold anything)
                    sP[(ty + 16 * i) * S::LS + tx + 16 * j] = p[i][j] == 0.f ? 0.f : p[i][j] * (dp[i][j] - del[j]);
            __syncthreads();
            acc_k.add(sP, sX, tx, ty);
        }
    }
    store_rows<DT, CP, BM>(rows_of<DT>(d_k, b, m), d_k.t, k0, g.Tk, g.C, acc_k, scale_k, tx, ty);
    store_rows<DT, CP, BM>(rows_of<DT>(d_v, b, m), d_v.t, k0, g.Tk, g.C, acc_v, scale_v, tx, ty);
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

// 128 query rows a block where blocks of 64 would take the SMs more than one round: a piece of 8 x 4 scores reads 12 operands from shared
// memory for its 32 products, one of 4 x 4 reads 8 for 16.  Forward and query half with 256 blocks of 64: 277 and 417 us; with 128 of 128:
// 244 and 365 us.
template <int CP, typename F>
int by_rows(const Place& at, const Geom& g, F&& f) {
    if constexpr (CP <= 128) {
        if ((long long)g.B * g.N * ((g.Tq + 63) / 64) > na2d_tc::sm_count(at.device)) return f(std::integral_constant<int, 128>{});
        return f(std::integral_constant<int, 64>{});
    } else {
        return f(std::integral_constant<int, 32>{});
    }
}

template <typename DT, int CP, int BM>
int forward_as(const Place& at, const Geom& g, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse) {
    using S = SimtCfg<CP, BM>;
    static std::atomic<unsigned long long> opted{0};
    const int vec = vectors(q, at.dtype, g.C) && vectors(k, at.dtype, g.C) && vectors(v, at.dtype, g.C);
    int tiles = 0;
    unsigned blocks = 0;
    if (int rc = blocks_of((long long)g.B * g.N, g.Tq, BM, &tiles, &blocks)) return rc;
    return start(at, simt_fwd_kernel<DT, CP, BM>, blocks, S::HELD + S::TILE + S::SCORES, opted, q, k, v, o, lse, g, tiles, vec);
}

template <typename DT, int CP, int BM>
int queries_as(const Place& at, const Geom& g, const Backward& x, int vec) {
    using S = SimtCfg<CP, BM>;
    static std::atomic<unsigned long long> opted{0};
    int tiles = 0;
    unsigned blocks = 0;
    if (int rc = blocks_of((long long)g.B * g.N, g.Tq, BM, &tiles, &blocks)) return rc;
    return start(at, simt_dq_kernel<DT, CP, BM>, blocks, 2 * S::HELD + S::TILE + S::SCORES, opted, x.q, x.k, x.v, x.d_o, x.d_q, x.lse,
                 (const float*)x.delta, g, tiles, vec);
}

template <typename DT, int CP>
int backward_as(const Place& at, const Geom& g, const Backward& x) {
    constexpr int BM = CP <= 128 ? 64 : 32;
    using S = SimtCfg<CP, BM>;
    static std::atomic<unsigned long long> opted{0};
    int vec = 1, tiles = 0;
    for (const Operand* t : {&x.q, &x.k, &x.v, &x.d_o}) vec = vec && vectors(*t, at.dtype, g.C);
    const long long rows = (long long)g.B * g.N * g.Tq;
    if ((rows + 7) / 8 > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    simt_delta_kernel<DT><<<(unsigned)((rows + 7) / 8), kThreads, 0, at.st>>>(x.d_o, x.o, x.delta, g);
    *at.launched += 1;
    if (cudaGetLastError() != cudaSuccess) return NA2D_ERR_CUDA;
    if (x.d_q.ptr) {
        if (int rc = by_rows<CP>(at, g, [&](auto bm) { return queries_as<DT, CP, decltype(bm)::value>(at, g, x, vec); })) return rc;
    }
    if (!x.d_k.ptr) return NA2D_OK;
    unsigned blocks = 0;
    if (int rc = blocks_of(g.units, g.Tk, BM, &tiles, &blocks)) return rc;
    return start(at, simt_dkdv_kernel<DT, CP>, blocks, 4 * S::TILE + S::SCORES, opted, x.q, x.k, x.v, x.d_o, x.d_k, x.d_v, x.lse,
                 (const float*)x.delta, g, tiles, vec);
}

}  // namespace

int simt_forward(const Place& at, const Geom& g, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse) {
    auto run = [&](auto type) {
        using DT = decltype(type);
        return by_channels<DT>(g.C, [&](auto cp) {
            constexpr int CP = decltype(cp)::value;
            return by_rows<CP>(at, g, [&](auto bm) { return forward_as<DT, CP, decltype(bm)::value>(at, g, q, k, v, o, lse); });
        });
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
