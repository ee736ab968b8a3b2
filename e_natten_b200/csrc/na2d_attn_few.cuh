// Attention over all keys, forward, for units of at most 16 query rows: single tokens on caches.
//
// Bound by memory (every key and value is read once, for 2 x 16 x D multiply-adds a key), so what counts is how many bytes are under way
// and how short the chain from a key to its weight is.  On tcgen05 a tile has 128 rows and its scores go through tensor memory: 5000
// cycles a chunk for a group, two groups an SM, 60 % of the bandwidth (16 x 4 caches of up to 32768 keys of 128, 16 heads: 137 us).  Here
// a warp takes 16 keys at a time by itself: mma.sync of 16 x 8 x 16 on registers, the scores' own registers being the next product's
// operand (rounded once to 16 bits, as in na2d_attn_fwd.cuh), its keys and values in stages of shared memory that no other warp touches.
//
// Measured: 16 x 16 heads on 4 key heads, caches of up to 32768 keys of 128, bf16: 95 us with the joining of the parts, 87 % of the copy
// bandwidth over the caches' bytes.
//
// The keys of all units lie on one line (na2d_attn_fwd.cuh); a CTA has a stretch of it, its eight warps 16 keys each of every 128.  At
// the end of a unit the warps' sums are joined in shared memory and go to the workspace.
#pragma once

#include "na2d_attn_fwd.cuh"

namespace na2d_attn {

constexpr int kFewRows = 16, kFewWarps = 8;

template <typename DT>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (IsBf16<DT>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes, or (not `there`) zeros.
__device__ __forceinline__ void copy_16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

template <int D, int NST>
struct FewCfg {
    static constexpr int PIECES = D / 8;                                 // 16-byte pieces of a row
    static constexpr int TILE = 16 * D * 2;                              // 16 keys, or their values
    static constexpr int SMEM = 1024 /*alignment*/ + (kLineEntries + 1 + 2 * kFewWarps * kFewRows + 15) / 4 * 16 + kFewWarps * NST * 2 * TILE;
    static int bytes(int rows) { return SMEM + kFewWarps * rows * D * 4; }
    // Piece p of row r: eight rows' pieces lie in different banks.
    static __device__ __forceinline__ uint32_t at(int r, int p) {
        return (uint32_t)(r * PIECES + (p ^ (PIECES >= 8 ? r & 7 : (r >> 1) & 3))) * 16u;
    }
};

template <typename DT, int D, int NST>
__global__ void __launch_bounds__(kFewWarps * 32, 1)
attn_few_kernel(const Operand q, const Operand k, const Operand v, const Geom g, const FwdCut cut, const int rows) {
    using C = FewCfg<D, NST>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* stages = smem;                                              // [warp][stage]{K, V}
    float* sums = reinterpret_cast<float*>(stages + kFewWarps * NST * 2 * C::TILE);      // [warp][row][D]
    float* tops = sums + kFewWarps * rows * D;                           // [warp][16]{maximum * log2(e), sum}
    int* before = reinterpret_cast<int*>(tops + 2 * kFewWarps * kFewRows);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    after_previous_grid();
    if (warp == 0) line_table(g, before, lane);
    __syncthreads();
    next_grid_may_start();

    const uint32_t own = smem_u32(stages) + warp * NST * 2 * C::TILE;
    Stretch ahead, here;
    here.start(g, before, blockIdx.x, gridDim.x);
    ahead = here;
    int unit_end = ahead.any() ? ahead.first(g, before) + ahead.length(before) : 0, slot_ahead = 0, slot = 0;
    auto ask = [&]() {                                                   // this warp's keys of the next chunk on the line
        if (ahead.any()) {
            const int key0 = (ahead.at - ahead.first(g, before)) * kRows + 16 * warp, count = key_count(g, ahead.b);
            const DT* kp = static_cast<const DT*>(k.ptr) + ahead.b * k.b + ahead.m * k.n;
            const DT* vp = static_cast<const DT*>(v.ptr) + ahead.b * v.b + ahead.m * v.n;
            const uint32_t to = own + slot_ahead * 2 * C::TILE;
#pragma unroll
            for (int i = 0; i < 16 * C::PIECES / 32; ++i) {
                const int piece = lane + 32 * i, r = piece / C::PIECES, p = piece % C::PIECES, key = key0 + r;
                const bool there = key < count && 8 * p < g.C;           // beyond: zeros, whatever memory holds
                const long long row = there ? key : 0;
                copy_16(to + C::at(r, p), kp + row * k.t + (there ? 8 * p : 0), there);
                copy_16(to + C::TILE + C::at(r, p), vp + row * v.t + (there ? 8 * p : 0), there);
            }
            if (++ahead.at == unit_end && ahead.any()) {
                --ahead.at;
                ahead.next(g, before);
                unit_end = ahead.first(g, before) + ahead.length(before);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (++slot_ahead == NST) slot_ahead = 0;
    };
#pragma unroll
    for (int i = 0; i < NST - 1; ++i) ask();

    const int r_lo = lane / 4, c_lo = 2 * (lane % 4);                    // of a fragment: rows r_lo and r_lo + 8, columns c_lo, + 1
    while (here.any()) {
        const int b = here.b, m = here.m, count = key_count(g, b), unit = b * g.Nk + m;
        const int first = here.first(g, before), n = min(here.end, first + here.length(before)) - here.at, c0 = here.at - first;
        // Q as the first product's operand, and the keys that the thread's two rows see
        uint32_t qf[D / 16][4];
        int seen[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = r_lo + 8 * half, h = r / g.Tq, t = r - h * g.Tq;
            const bool ok = r < rows;
            seen[half] = ok ? keys_seen(g, count, t) : 0;
            const DT* src = static_cast<const DT*>(q.ptr) + b * q.b + (m * g.G + (ok ? h : 0)) * q.n + (ok ? t : 0) * q.t;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int c = 16 * kk + 8 * e + c_lo;
                    qf[kk][half + 2 * e] = ok && c < g.C ? __ldg(reinterpret_cast<const unsigned*>(src + c)) : 0u;
                }
        }
        float acc[D / 8][4], top[2] = {-CUDART_INF_F, -CUDART_INF_F}, total[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;

        for (int i = 0; i < n; ++i) {
            ask();
            asm volatile("cp.async.wait_group %0;" ::"n"(NST - 1) : "memory");
            __syncwarp();
            const uint32_t tk = own + slot * 2 * C::TILE, tv = tk + C::TILE;
            if (++slot == NST) slot = 0;
            // scores of 16 rows and 16 keys
            float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                uint32_t kb[4];                                          // keys 0-7: channels 0-7, 8-15; keys 8-15: the same
                load_matrices(kb, tk + C::at((lane & 7) + 8 * (lane >> 4), 2 * kk + ((lane >> 3) & 1)));
                mma_16816<DT>(s[0], qf[kk], kb[0], kb[1]);
                mma_16816<DT>(s[1], qf[kk], kb[2], kb[3]);
            }
            const int key0 = (c0 + i) * kRows + 16 * warp;
            float high[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                high[half] = -CUDART_INF_F;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = s[j][2 * half + e];
                        x = key0 + 8 * j + c_lo + e < seen[half] ? x * g.sl2 : -CUDART_INF_F;
                        high[half] = fmaxf(high[half], x);
                    }
                high[half] = fmaxf(high[half], __shfl_xor_sync(0xffffffffu, high[half], 1));
                high[half] = fmaxf(high[half], __shfl_xor_sync(0xffffffffu, high[half], 2));
            }
            if (__any_sync(0xffffffffu, high[0] > top[0] + kGrow || high[1] > top[1] + kGrow ||
                                            (top[0] == -CUDART_INF_F && high[0] > top[0]) || (top[1] == -CUDART_INF_F && high[1] > top[1]))) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float to = fmaxf(top[half], high[half]), base = to == -CUDART_INF_F ? 0.f : to;
                    const float alpha = fast_exp2(top[half] - base);
                    top[half] = to;
                    total[half] *= alpha;
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        acc[j][2 * half] *= alpha;
                        acc[j][2 * half + 1] *= alpha;
                    }
                }
            }
            uint32_t p[4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float base = (top[half] == -CUDART_INF_F ? 0.f : top[half]) - kLift<DT>;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float p0 = fast_exp2(s[j][2 * half] - base), p1 = fast_exp2(s[j][2 * half + 1] - base);
                    total[half] += p0 + p1;
                    p[half + 2 * j] = pack2<DT>(p0, p1);
                }
            }
#pragma unroll
            for (int jj = 0; jj < D / 16; ++jj) {
                uint32_t vb[4];                                          // channels 0-7: keys 0-7, 8-15; channels 8-15: the same
                load_matrices_transposed(vb, tv + C::at(lane & 15, 2 * jj + (lane >> 4)));
                mma_16816<DT>(acc[2 * jj], p, vb[0], vb[1]);
                mma_16816<DT>(acc[2 * jj + 1], p, vb[2], vb[3]);
            }
            __syncwarp();                                                // the stage has been read
        }
        // the warps' sums -> the unit's part
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            total[half] += __shfl_xor_sync(0xffffffffu, total[half], 1);
            total[half] += __shfl_xor_sync(0xffffffffu, total[half], 2);
            const int r = r_lo + 8 * half;
            if (lane % 4 == 0) {
                tops[(warp * kFewRows + r) * 2] = top[half];
                tops[(warp * kFewRows + r) * 2 + 1] = total[half];
            }
            if (r < rows)
#pragma unroll
                for (int j = 0; j < D / 8; ++j)
                    *reinterpret_cast<float2*>(sums + (warp * rows + r) * D + 8 * j + c_lo) = make_float2(acc[j][2 * half], acc[j][2 * half + 1]);
        }
        __syncthreads();
        const size_t part = static_cast<size_t>(blockIdx.x + unit) * rows;
        for (int i = threadIdx.x; i < rows * (D / 4); i += kFewWarps * 32) {
            const int r = i / (D / 4), c = 4 * (i % (D / 4));
            float high = -CUDART_INF_F, all = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) high = fmaxf(high, tops[(w * kFewRows + r) * 2]);
            const float base = high == -CUDART_INF_F ? 0.f : high;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) {
                const float by = fast_exp2(tops[(w * kFewRows + r) * 2] - base);
                const float4 x = *reinterpret_cast<const float4*>(sums + (w * rows + r) * D + c);
                all = fmaf(by, tops[(w * kFewRows + r) * 2 + 1], all);
                o.x = fmaf(by, x.x, o.x);
                o.y = fmaf(by, x.y, o.y);
                o.z = fmaf(by, x.z, o.z);
                o.w = fmaf(by, x.w, o.w);
            }
            const float inv = all == 0.f ? 0.f : 1.f / all;
            if (c < g.C) *reinterpret_cast<float4*>(cut.part_o + (part + r) * g.C + c) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
            if (c == 0) cut.part_lse[part + r] = all == 0.f ? -CUDART_INF_F : (base - kLift<DT> + log2f(all)) * kLn2;
        }
        __syncthreads();
        here.next(g, before);
    }
}

template <typename DT, int D, int NST>
int launch_few_as(const Place& at, const Geom& g, const FwdCut& cut, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse) {
    auto kern = attn_few_kernel<DT, D, NST>;
    static std::atomic<unsigned long long> opted{0};
    const int rows = g.G * g.Tq, smem = FewCfg<D, NST>::bytes(rows);
    if (na2d_tc::opt_in_smem(kern, kSmemLimit, at.device, opted) != cudaSuccess) return NA2D_ERR_CUDA;
    *at.launched += 1;
    if (na2d_launch::launch(false, kern, cut.line, kFewWarps * 32, smem, at.st, q, k, v, g, cut, rows) != cudaSuccess) return NA2D_ERR_CUDA;
    return launch_combine<DT>(at, g, cut, o, lse);
}

// (three stages of 16 keys a warp at head dim 128, two where the rows' sums take their room, from 8 rows on; twice, and four times as many
// of the narrower ones)
template <typename DT, int D>
int launch_few(const Place& at, const Geom& g, const FwdCut& cut, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse) {
    constexpr int kFull = 3 * 128 / D, kLess = 2 * 128 / D;
    static_assert(FewCfg<D, kLess>::SMEM + kFewWarps * kFewRows * D * 4 <= kSmemLimit, "stages");
    return FewCfg<D, kFull>::bytes(g.G * g.Tq) <= kSmemLimit ? launch_few_as<DT, D, kFull>(at, g, cut, q, k, v, o, lse)
                                                              : launch_few_as<DT, D, kLess>(at, g, cut, q, k, v, o, lse);
}

}  // namespace na2d_attn
