// Attention over all keys on CUDA cores: fp32, head dims that are no multiple of 8 or beyond 128, and any strides.
//
// A block has 128 or 64 query rows (or 64 keys) and walks the other side in tiles, in fp32; the next tile is on its way to registers
// meanwhile.  256 threads as 16 x 16; a thread has 8 x 4 (4 x 4) of a score tile and its rows' part of an output tile, all in registers, and
// multiplies and adds two channels at a time.  Tiles lie in shared memory as rows of CP + 4 floats, so that the 16-byte loads of a column
// of threads fall into different banks; neighbouring lanes are two rows of one column, because a warp's 16-byte loads are shared between
// neighbours only (with 16 columns side by side each load took its full four turns: 1305 us against 1209).
// What bounds it: the multiply-adds, and beside them the loads from shared memory.  Batch 4, 4 heads of 128, 1024 tokens, fp32, forward and
// backward: 1077 us, 36 TFLOP/s over the nine products that are done (the seven that have to be: 406 us at the 74 TFLOP/s that 148 SMs of 128
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
template <typename OT, int CP, int BM>
__device__ __forceinline__ void store_rows(OT* dst, long long stride, int row0, int rows, int C,
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
                if (c < C) dst[r * stride + c] = narrow<OT>(scale[i] == 0.f ? 0.f : x);
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

// What a launch works on: one problem, or two whose blocks share it (a prefix's keys and the entries' own: small ones take as long alone as
// together).  `out`: o, dQ or dK; out2: dV.  WIDE kernels take the other side (keys; rows in the key half) in `splits` parts of `each` tiles,
// whose fp32 results lie `part` values apart, and lse B N Tq; sums and sums2 are those of the key half.
struct SimtWork {
    Operand q, k, v, d_o, out, out2;
    float *lse, *delta, *sums, *sums2;
    Geom g;
    int tiles, vec, splits, each;
    size_t part;
    unsigned blocks;                    // of all parts
};
struct SimtPair {
    SimtWork at[2];
};
// The problem of this block, its block of a part, and which part.  ONE: there is no second problem.
template <bool WIDE, bool ONE = false>
__device__ __forceinline__ const SimtWork& work_of(const SimtPair& p, unsigned& block, int& split) {
    if constexpr (ONE) {
        block = blockIdx.x;
        split = 0;
        return p.at[0];
    }
    const bool second = blockIdx.x >= p.at[0].blocks;
    block = blockIdx.x - (second ? p.at[0].blocks : 0u);
    split = 0;
    if constexpr (WIDE) {
        const unsigned each = p.at[second].blocks / p.at[second].splits;
        split = block / each;
        block -= split * each;
    }
    return p.at[second];
}

// ---- forward: a block has BT queries of one head ------------------------------------------------------------------
template <typename DT, bool WIDE, int CP, int BM>
__global__ void __launch_bounds__(kThreads)
simt_fwd_kernel(const __grid_constant__ SimtPair pair) {
    using S = SimtCfg<CP, BM>;
    using OT = std::conditional_t<WIDE, float, DT>;
    unsigned block;
    int split;
    const SimtWork& work = work_of<WIDE>(pair, block, split);
    const Operand q = work.q, k = work.k, v = work.v, o = work.out;
    const Geom g = work.g;
    float* __restrict__ lse = work.lse + (WIDE ? split * ((size_t)g.B * g.N * g.Tq) : 0);
    const int tiles = work.tiles, vec = work.vec;
    extern __shared__ __align__(16) float smem[];
    float *sQ = smem, *sKV = sQ + S::HELD, *sP = sKV + S::TILE;
    const int tx = threadIdx.x % 32 / 2, ty = threadIdx.x / 32 * 2 + threadIdx.x % 2;
    const int bn = block / tiles, b = bn / g.N, n = bn - b * g.N, m = n / g.G;
    const int t0 = (g.causal ? tiles - 1 - (int)(block % tiles) : (int)(block % tiles)) * BM;
    const int count = key_count(g, b), all_keys = keys_seen(g, count, min(t0 + BM, g.Tq) - 1);
    const int from = WIDE ? split * work.each * S::BT : 0, keys = WIDE ? min(all_keys, from + work.each * S::BT) : all_keys;
    Tile<DT, CP, BM>::bring(sQ, rows_of<DT>(q, b, n), q.t, t0, g.Tq, g.C, vec);
    Tile<DT, CP, S::BT> tile;
    if (keys > from) tile.fetch(rows_of<DT>(k, b, m), k.t, from, count, g.C, vec);
    Sums<CP, BM> acc;
    float top[S::RM], total[S::RM];
#pragma unroll
    for (int i = 0; i < S::RM; ++i) {
        top[i] = -CUDART_INF_F;
        total[i] = 0.f;
    }
    for (int k0 = from; k0 < keys; k0 += S::BT) {
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
    store_rows<OT, CP, BM>(rows_of<OT>(o, b, n) + (WIDE ? split * work.part : 0), o.t, t0, g.Tq, g.C, acc, inv, tx, ty);
}

// ---- delta = dO . o, a warp a row -------------------------------------------------------------------------------------
template <typename DT>
__global__ void __launch_bounds__(kThreads) simt_delta_kernel(const __grid_constant__ SimtPair pair) {
    unsigned block;
    int split;
    const SimtWork& work = work_of<false>(pair, block, split);
    const Operand d_o = work.d_o, o = work.out;
    float* __restrict__ delta = work.delta;
    const Geom& g = work.g;
    const long long rows = (long long)g.B * g.N * g.Tq, row = (long long)block * 8 + threadIdx.x / 32;
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
// Head dims above 128: 128 registers, with which an SM has two blocks.  2 x 8 heads x 1024 x 256, fp32: 953 us; 136 registers, one block, 1068.
// (0: as many as the compiler takes.)
template <typename DT, bool WIDE, int CP, int BM>
__global__ void __launch_bounds__(kThreads, CP > 128 ? 2 : 0)
simt_dq_kernel(const __grid_constant__ SimtPair pair) {
    using S = SimtCfg<CP, BM>;
    using OT = std::conditional_t<WIDE, float, DT>;
    unsigned block;
    int split;
    const SimtWork& work = work_of<WIDE>(pair, block, split);
    const Operand q = work.q, k = work.k, v = work.v, d_o = work.d_o, d_q = work.out;
    const float *__restrict__ lse = work.lse, *__restrict__ delta = work.delta;
    const Geom g = work.g;
    const int tiles = work.tiles, vec = work.vec;
    extern __shared__ __align__(16) float smem[];
    float *sQ = smem, *sG = sQ + S::HELD, *sKV = sG + S::HELD, *sP = sKV + S::TILE;
    const int tx = threadIdx.x % 32 / 2, ty = threadIdx.x / 32 * 2 + threadIdx.x % 2;
    const int bn = block / tiles, b = bn / g.N, n = bn - b * g.N, m = n / g.G;
    const int t0 = (g.causal ? tiles - 1 - (int)(block % tiles) : (int)(block % tiles)) * BM;
    const int count = key_count(g, b), all_keys = keys_seen(g, count, min(t0 + BM, g.Tq) - 1);
    const int from = WIDE ? split * work.each * S::BT : 0, keys = WIDE ? min(all_keys, from + work.each * S::BT) : all_keys;
    Tile<DT, CP, BM>::bring(sQ, rows_of<DT>(q, b, n), q.t, t0, g.Tq, g.C, vec);
    Tile<DT, CP, BM>::bring(sG, rows_of<DT>(d_o, b, n), d_o.t, t0, g.Tq, g.C, vec);
    Tile<DT, CP, S::BT> tile;
    if (keys > from) tile.fetch(rows_of<DT>(v, b, m), v.t, from, count, g.C, vec);
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
    for (int k0 = from; k0 < keys; k0 += S::BT) {
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
    store_rows<OT, CP, BM>(rows_of<OT>(d_q, b, n) + (WIDE ? split * work.part : 0), d_q.t, t0, g.Tq, g.C, acc, scale, tx, ty);
}

// ---- key half: a block has BT keys of one key head and walks the queries of every head that shares it ------------------------
// Head dims above 128: calls of one problem that is not taken in parts have instances without the choice between two, whose operands then
// stay in constant memory.  2 x 8 heads x 1024 x 256, fp32: 1422 us for 1510, fp16 causal 1032 for 1091.  (Below it is the other way round: 128
// channels 1063 us for 1028.  Forward and query half are faster with the choice throughout.)
template <int CP, bool WIDE> constexpr bool kOneProblem = CP > 128 && !WIDE;
template <typename DT, bool WIDE, int CP>
__global__ void __launch_bounds__(kThreads)
simt_dkdv_kernel(const __grid_constant__ SimtPair pair) {
    constexpr int BM = CP <= 128 ? 64 : 32;
    using S = SimtCfg<CP, BM>;
    unsigned block;
    int split;
    const SimtWork& work = work_of<WIDE, kOneProblem<CP, WIDE>>(pair, block, split);
    const Operand q = work.q, k = work.k, v = work.v, d_o = work.d_o, d_k = work.out, d_v = work.out2;
    const float *__restrict__ lse = work.lse, *__restrict__ delta = work.delta;
    const Geom g = work.g;
    const int tiles = work.tiles, vec = work.vec;
    extern __shared__ __align__(16) float smem[];
    float *sK = smem, *sV = sK + S::TILE, *sX = sV + S::TILE, *sY = sX + S::TILE, *sP = sY + S::TILE;
    const int tx = threadIdx.x % 32 / 2, ty = threadIdx.x / 32 * 2 + threadIdx.x % 2;
    const int unit = block / tiles, b = unit / g.Nk, m = unit - b * g.Nk;
    const int k0 = (block % tiles) * S::BT;
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
    // tiles of rows, of one head after the other: the part's first one and how many it has
    int n = m * g.G, t0 = first, left = any ? g.G * ((g.Tq - first + S::BT - 1) / S::BT) : 0;
    if constexpr (WIDE) {
        const int per_head = (g.Tq - first + S::BT - 1) / S::BT, at = min(split * work.each, left);
        left = min(left - at, work.each);
        if (left > 0) {
            n += at / per_head;
            t0 += at % per_head * S::BT;
        }
    }
    if (left > 0) tile.fetch(rows_of<DT>(q, b, n), q.t, t0, g.Tq, g.C, vec);
    for (; left > 0; --left) {
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
        t0 += S::BT;
        if (t0 >= g.Tq) {
            t0 = first;
            ++n;
        }
        if (left > 1) tile.fetch(rows_of<DT>(q, b, n), q.t, t0, g.Tq, g.C, vec);
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
    if (WIDE && work.splits > 1) {                       // summed by simt_sum_kernel
        const size_t at = split * work.part + ((size_t)b * g.Nk + m) * g.Tk * g.C;
        store_rows<float, CP, BM>(work.sums + at, g.C, k0, g.Tk, g.C, acc_k, scale_k, tx, ty);
        store_rows<float, CP, BM>(work.sums2 + at, g.C, k0, g.Tk, g.C, acc_v, scale_v, tx, ty);
        return;
    }
    store_rows<DT, CP, BM>(rows_of<DT>(d_k, b, m), d_k.t, k0, g.Tk, g.C, acc_k, scale_k, tx, ty);
    store_rows<DT, CP, BM>(rows_of<DT>(d_v, b, m), d_v.t, k0, g.Tk, g.C, acc_v, scale_v, tx, ty);
}

// dK and dV (the second row of blocks) from their parts, in the parts' order.
template <typename DT>
__global__ void __launch_bounds__(kThreads)
simt_sum_kernel(const float* __restrict__ sums, const float* __restrict__ sums2, DT* __restrict__ d_k, DT* __restrict__ d_v, const size_t part, const int splits) {
    const size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= part) return;
    const float* from = blockIdx.y ? sums2 : sums;
    float acc = 0.f;
    for (int s = 0; s < splits; ++s) acc += from[s * part + i];
    (blockIdx.y ? d_v : d_k)[i] = narrow<DT>(acc);
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
int cut_work(SimtWork* w, long long units, int rows, int tile) {
    w->tiles = (rows + tile - 1) / tile;
    if (units * w->tiles > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    w->blocks = (unsigned)(units * w->tiles);
    return NA2D_OK;
}

// floats: of dynamic shared memory, 0: none.
template <typename K>
int start(const Place& at, K kernel, const SimtPair& pair, int floats, std::atomic<unsigned long long>& opted) {
    const unsigned long long blocks = (unsigned long long)pair.at[0].blocks + pair.at[1].blocks;
    if (blocks == 0) return NA2D_OK;
    if (blocks > 0x7fffffffULL) return NA2D_ERR_TOO_LARGE;
    if (floats > 0 && na2d_tc::opt_in_smem(kernel, floats * 4, at.device, opted) != cudaSuccess) return NA2D_ERR_CUDA;
    kernel<<<(unsigned)blocks, kThreads, floats * 4, at.st>>>(pair);
    *at.launched += 1;
    return cudaGetLastError() == cudaSuccess ? NA2D_OK : NA2D_ERR_CUDA;
}

// 128 query rows a block where blocks of 64 would take the SMs more than one round, and where that adds no more than an eighth of rows that are
// none: a piece of 8 x 4 scores reads 12 operands from shared memory for its 32 products, one of 4 x 4 reads 8 for 16.  Forward and query
// half (with delta), fp32: 16 heads x 1024 x 128, 256 blocks of 64: 258 and 384 us, 128 of 128: 233 and 349.  18 x 16 x 36 rows x 64, of which blocks of
// 128 do twice the work, 18 and 32 with 64, 29 and 40 with 128; 16 x 16 x 129 x 128 160 and 237 for 191 and 283.  (Where blocks of 128 are just half as
// many the rule can lose: 64 x 8 x 65 x 32 57 and 79 us, 45 and 67 with blocks of 64.)
template <int CP, typename F>
int by_rows(const Place& at, const SimtPair& pair, F&& f) {
    if constexpr (CP <= 128) {
        long long small = 0, large = 0;
        for (const SimtWork& w : pair.at) {
            small += (long long)w.g.B * w.g.N * ((w.g.Tq + 63) / 64);
            large += (long long)w.g.B * w.g.N * ((w.g.Tq + 127) / 128);
        }
        if (small > na2d_tc::sm_count(at.device) && 16 * large <= 9 * small) return f(std::integral_constant<int, 128>{});
        return f(std::integral_constant<int, 64>{});
    } else {
        return f(std::integral_constant<int, 32>{});
    }
}

// Parts of a WIDE kernel's other side.
void cut_parts(SimtWork* w, int tiles, int splits) {
    w->splits = splits;
    w->each = (tiles + splits - 1) / splits;
    w->blocks *= splits;
}
int tile_of(int C) { return C <= 128 ? 64 : 32; }
size_t dense_rows(const Geom& g) { return (size_t)g.B * g.N * g.Tq * g.C; }

template <typename DT, bool WIDE, int CP, int BM>
int forward_as(const Place& at, SimtPair pair) {
    using S = SimtCfg<CP, BM>;
    static std::atomic<unsigned long long> opted{0};
    for (SimtWork& w : pair.at) {
        if (!w.q.ptr) continue;
        w.vec = vectors(w.q, at.dtype, w.g.C) && vectors(w.k, at.dtype, w.g.C) && vectors(w.v, at.dtype, w.g.C);
        if (int rc = cut_work(&w, (long long)w.g.B * w.g.N, w.g.Tq, BM)) return rc;
        if (WIDE) cut_parts(&w, (w.g.Tk + S::BT - 1) / S::BT, simt_key_parts(w.g, na2d_tc::sm_count(at.device)));
        w.part = dense_rows(w.g);
    }
    return start(at, simt_fwd_kernel<DT, WIDE, CP, BM>, pair, S::HELD + S::TILE + S::SCORES, opted);
}

template <typename DT, bool WIDE, int CP, int BM>
int queries_as(const Place& at, SimtPair pair) {
    using S = SimtCfg<CP, BM>;
    static std::atomic<unsigned long long> opted{0};
    for (SimtWork& w : pair.at) {
        if (!w.q.ptr) continue;
        if (int rc = cut_work(&w, (long long)w.g.B * w.g.N, w.g.Tq, BM)) return rc;
        if (WIDE) cut_parts(&w, (w.g.Tk + S::BT - 1) / S::BT, simt_key_parts(w.g, na2d_tc::sm_count(at.device)));
        w.part = dense_rows(w.g);
    }
    return start(at, simt_dq_kernel<DT, WIDE, CP, BM>, pair, 2 * S::HELD + S::TILE + S::SCORES, opted);
}

template <typename DT, int CP>
int backward_as(const Place& at, const Backward* x, int count) {
    constexpr int BM = CP <= 128 ? 64 : 32;
    using S = SimtCfg<CP, BM>;
    static std::atomic<unsigned long long> opted[2]{};
    SimtPair delta{}, queries{}, keys{};
    bool wide = false, parts = false;
    for (int i = 0; i < count; ++i) {
        SimtWork w{};
        w.q = x[i].q;
        w.k = x[i].k;
        w.v = x[i].v;
        w.d_o = x[i].d_o;
        w.lse = const_cast<float*>(x[i].lse);
        w.delta = x[i].delta;
        w.g = *x[i].g;
        w.splits = 1;
        w.vec = 1;
        for (const Operand* t : {&w.q, &w.k, &w.v, &w.d_o}) w.vec = w.vec && vectors(*t, at.dtype, w.g.C);
        delta.at[i] = w;
        delta.at[i].out = x[i].o;
        const long long blocks = ((long long)w.g.B * w.g.N * w.g.Tq + 7) / 8;        // a warp a row
        if (blocks > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
        delta.at[i].blocks = (unsigned)blocks;
        if (x[i].d_q.ptr) {
            queries.at[i] = w;
            queries.at[i].out = x[i].d_q;
            wide = x[i].d_q.wide;
        }
        if (x[i].d_k.ptr) {
            SimtWork& y = keys.at[i];
            y = w;
            y.out = x[i].d_k;
            y.out2 = x[i].d_v;
            if (int rc = cut_work(&y, w.g.units, w.g.Tk, BM)) return rc;
            const int splits = x[i].key_sums ? simt_row_parts(w.g, na2d_tc::sm_count(at.device)) : 1;
            cut_parts(&y, w.g.G * ((w.g.Tq + S::BT - 1) / S::BT), splits);
            y.part = (size_t)w.g.units * w.g.Tk * w.g.C;
            y.sums = x[i].key_sums;
            y.sums2 = x[i].key_sums + splits * y.part;
            parts = parts || splits > 1;
        }
    }
    if (int rc = start(at, simt_delta_kernel<DT>, delta, 0, opted[0])) return rc;
    if (int rc = by_rows<CP>(at, queries, [&](auto bm) {
            constexpr int kRowsOf = decltype(bm)::value;
            return wide ? queries_as<DT, true, CP, kRowsOf>(at, queries) : queries_as<DT, false, CP, kRowsOf>(at, queries);
        }))
        return rc;
    if (!keys.at[0].blocks) std::swap(keys.at[0], keys.at[1]);
    for (SimtWork& y : keys.at)
        if (!y.splits) y.splits = 1;                     // (no blocks)
    if (!parts && !(kOneProblem<CP, false> && keys.at[1].blocks))
        return start(at, simt_dkdv_kernel<DT, false, CP>, keys, 4 * S::TILE + S::SCORES, opted[0]);
    if (int rc = start(at, simt_dkdv_kernel<DT, true, CP>, keys, 4 * S::TILE + S::SCORES, opted[1])) return rc;
    for (const SimtWork& y : keys.at) {
        if (y.splits == 1) continue;
        const size_t blocks = (y.part + kThreads - 1) / kThreads;
        if (blocks > 0x7fffffffULL) return NA2D_ERR_TOO_LARGE;
        simt_sum_kernel<DT><<<dim3((unsigned)blocks, 2), kThreads, 0, at.st>>>(y.sums, y.sums2, static_cast<DT*>(y.out.ptr), static_cast<DT*>(y.out2.ptr),
                                                                              y.part, y.splits);
        *at.launched += 1;
        if (cudaGetLastError() != cudaSuccess) return NA2D_ERR_CUDA;
    }
    return NA2D_OK;
}

// As many parts as give each SM two blocks where there are fewer blocks than SMs, of at least four tiles each.  The key half of 12 key heads of 119
// keys, 4 x 648 rows each, fp32, 64 channels: 24 blocks of 41 tiles took 396 us, in parts they take 152.
int parts_for(long long blocks, long long tiles, int sms) {
    if (blocks >= sms) return 1;
    return (int)std::max(1LL, std::min(2 * sms / std::max(1LL, blocks), tiles / 4));
}

}  // namespace

int simt_key_parts(const Geom& g, int sms) {
    return parts_for((long long)g.B * g.N * ((g.Tq + 63) / 64), (g.Tk + tile_of(g.C) - 1) / tile_of(g.C), sms);
}
int simt_row_parts(const Geom& g, int sms) {
    if (g.causal) return 1;
    const int tile = tile_of(g.C);
    return parts_for((long long)g.units * ((g.Tk + tile - 1) / tile), (long long)g.G * ((g.Tq + tile - 1) / tile), sms);
}

int simt_forward(const Place& at, const Forward* x, int count) {
    SimtPair pair{};
    for (int i = 0; i < count; ++i) {
        SimtWork& w = pair.at[i];
        w.q = x[i].q;
        w.k = x[i].k;
        w.v = x[i].v;
        w.out = x[i].o;
        w.lse = x[i].lse;
        w.g = *x[i].g;
    }
    for (SimtWork& w : pair.at) w.splits = 1;
    auto run = [&](auto type) {
        using DT = decltype(type);
        return by_channels<DT>(x[0].g->C, [&](auto cp) {
            constexpr int CP = decltype(cp)::value;
            return by_rows<CP>(at, pair, [&](auto bm) {
                constexpr int kRowsOf = decltype(bm)::value;
                return x[0].o.wide ? forward_as<DT, true, CP, kRowsOf>(at, pair) : forward_as<DT, false, CP, kRowsOf>(at, pair);
            });
        });
    };
    return at.dtype == NA2D_F32 ? run(float{}) : at.dtype == NA2D_BF16 ? run(__nv_bfloat16{}) : run(__half{});
}

int simt_backward(const Place& at, const Backward* x, int count) {
    auto run = [&](auto type) {
        using DT = decltype(type);
        return by_channels<DT>(x[0].g->C, [&](auto cp) { return backward_as<DT, decltype(cp)::value>(at, x, count); });
    };
    return at.dtype == NA2D_F32 ? run(float{}) : at.dtype == NA2D_BF16 ? run(__nv_bfloat16{}) : run(__half{});
}

}  // namespace na2d_attn
