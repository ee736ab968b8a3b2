// Attention over a prefix that entries share and their own keys, forward, for units of few query rows: single tokens, or a few, on caches.
//
// A unit is a key head of a prefix with the rows of all its entries, or a key head of one entry's own keys; either has up to 16 MT rows,
// which stay in registers as operands of mma.sync of 16 x 8 x 16.  Bound by memory, like the kernel for few rows of
// na2d_attn_few.cuh, whose inner step this is; there the eight warps of a block share a unit and join their sums at its end, which caches
// of a few hundred keys pay for at every unit.  Here the keys of all units, 16 a step, lie on one line of which every warp takes a
// stretch by itself: no barrier in the loop, loads that run ahead into the next unit, its queries among them, and at a unit's end the sums
// go from registers to the workspace.  A unit counts kUnitSteps steps more than it has keys for, since warps that met many short ones
// were the last by far.  prefix_join_kernel joins a row's parts, of its prefix and its own keys at once.
//
// Measured, bf16, 128 channels: 16 prompts x 4 key heads of 32768 keys, 16 rows each: 175 us, 94 % of the copy bandwidth; of 8192 to 2730 keys, with 64 caches
// of up to 256, 196 MB: 40 us, 75 %, about 8 of them before the first keys arrive and behind the last; the joins 8 more.
#pragma once

#include "na2d_attn_few.cuh"
#include "na2d_prefix_entry.h"

namespace na2d_prefix {

using namespace na2d_attn;

constexpr int kStep = 16, kTokenWarps = 8, kTokenThreads = kTokenWarps * 32;

// Stages of a warp's keys and values that fit beside the table.
template <int D> constexpr int kTokenStages = 3 * 128 / D;
template <int D> constexpr int kTokenSmem = kTokenWarps * kTokenStages<D> * 2 * kStep * D * 2 + (kTokenEntries + 1 + kTokenWarps) * 4 + 1024;
static_assert(kTokenSmem<128> <= kSmemLimit && kTokenSmem<64> <= kSmemLimit && kTokenSmem<32> <= kSmemLimit, "stages");

// Keys of entry e of the line: prefixes, then the batch's.
__device__ __forceinline__ int token_keys(const Tokens& x, int e) {
    const TokenSide& s = x.side[e >= x.side[0].entries];
    const int i = e >= x.side[0].entries ? e - x.side[0].entries : e;
    return s.lengths ? min(max(__ldg(s.lengths + i), 0), s.T) : s.T;
}

// A warp's stretch [at, end) of the line, and the unit that `at` lies in.  (Lengths count a unit's kUnitSteps, which come first.)
struct TokenStretch {
    int at, end, e, m;
    // the steps of the unit that the stretch has: [from, to)
    __device__ __forceinline__ void steps(const int* before, int Nk, int& from, int& to) const {
        const int unit = first(before, Nk);
        from = max(at - unit - kUnitSteps, 0);
        to = max(min(end - unit, length(before)) - kUnitSteps, 0);
    }
    __device__ __forceinline__ void start(const int* before, int entries, int Nk, int each, int warp) {
        const int all = before[entries] * Nk;
        at = (int)min((long long)warp * each, (long long)all);
        end = min(at + each, all);
        if (at >= end) return;
        int lo = 0, hi = entries;                        // before[lo] <= at's < before[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (before[mid] * Nk <= at) lo = mid;
            else hi = mid;
        }
        e = lo;
        m = (at - before[e] * Nk) / (before[e + 1] - before[e]);
    }
    __device__ __forceinline__ bool any() const { return at < end; }
    __device__ __forceinline__ int length(const int* before) const { return before[e + 1] - before[e]; }
    __device__ __forceinline__ int first(const int* before, int Nk) const { return before[e] * Nk + m * length(before); }
    __device__ __forceinline__ void next(const int* before, int Nk) {
        at = min(end, first(before, Nk) + length(before));
        if (at < end && ++m == Nk) {
            m = 0;
            do ++e;
            while (length(before) == 0);                 // (at < end: there is one)
        }
    }
};

template <typename DT, int D, int MT>
__global__ void __launch_bounds__(kTokenThreads, 1) prefix_tokens_kernel(const __grid_constant__ Tokens x) {
    constexpr int NST = kTokenStages<D>, PIECES = D / 8, TILE = kStep * D * 2;
    static_assert(MT <= 2, "a stage holds the rows of Q");
    using At = FewCfg<D, 1>;                             // places of a tile's pieces
    extern __shared__ uint8_t smem_raw[];
    uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));     // [warp][stage]{K, V}
    int* before = reinterpret_cast<int*>(stages + kTokenWarps * NST * 2 * TILE);     // steps of one key head of the entries before
    int* warp_sums = before + kTokenEntries + 1;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int E0 = x.side[0].entries, E = E0 + x.side[1].entries;

    // (behind another kernel of this call nothing here reads what that one wrote; the join that follows does, and the wait at the end is
    // for it)
    if (!x.behind) after_previous_grid();
    {   // the table
        for (int e = threadIdx.x; e < E; e += kTokenThreads) {
            const int steps = (token_keys(x, e) + kStep - 1) / kStep;
            before[e] = steps ? steps + kUnitSteps : 0;
        }
        __syncthreads();
        const int run = (E + kTokenThreads - 1) / kTokenThreads, e0 = threadIdx.x * run, e1 = min(e0 + run, E);
        int sum = 0;
        for (int e = e0; e < e1; ++e) sum += before[e];
        int up_to = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, up_to, d);
            if (lane >= d) up_to += up;
        }
        if (lane == 31) warp_sums[warp] = up_to;
        __syncthreads();
        int at = up_to - sum;
        for (int w = 0; w < warp; ++w) at += warp_sums[w];
        for (int e = e0; e < e1; ++e) {
            const int n = before[e];
            before[e] = at;
            at += n;
        }
        if (threadIdx.x == kTokenThreads - 1) before[E] = at;
        __syncthreads();
    }
    next_grid_may_start();
    const int warps = gridDim.x * kTokenWarps, all = before[E] * x.Nk, each = max(x.least, (all + warps - 1) / warps);
    if (blockIdx.x == 0) {                               // for the joins
        for (int e = threadIdx.x; e <= E; e += kTokenThreads) x.table[e] = before[e];
        if (threadIdx.x == 0) x.table[E + 1] = each;
    }

    const int own_warp = blockIdx.x * kTokenWarps + warp;
    const uint32_t own = smem_u32(stages) + warp * NST * 2 * TILE;
    TokenStretch ahead, here;
    here.start(before, E, x.Nk, each, own_warp);
    ahead = here;
    // of the unit that is loaded: its keys, their place, and the warp's steps of it that are left
    const DT *kp = nullptr, *vp = nullptr;
    long long k_t = 0, v_t = 0;
    int step = 0, stop = 0, unit_keys = 0, slot_ahead = 0, slot = 0;
    bool rows_due = false;
    auto enter = [&]() {
        for (; ahead.any(); ahead.next(before, x.Nk)) {
            ahead.steps(before, x.Nk, step, stop);
            if (step < stop) break;
        }
        if (!ahead.any()) return;
        const bool second = ahead.e >= E0;
        const TokenSide& s = x.side[second];
        const int i = second ? ahead.e - E0 : ahead.e;
        kp = static_cast<const DT*>(s.k.ptr) + i * s.k.b + ahead.m * s.k.n;
        vp = static_cast<const DT*>(s.v.ptr) + i * s.v.b + ahead.m * s.v.n;
        k_t = s.k.t;
        v_t = s.v.t;
        unit_keys = token_keys(x, ahead.e);
        rows_due = true;
    };
    enter();
    auto ask = [&]() {                                   // the next stage: a unit's rows, or 16 keys and their values
        if (ahead.any() && rows_due) {
            const bool second = ahead.e >= E0;
            const TokenSide& s = x.side[second];
            const int i0 = (second ? ahead.e - E0 : ahead.e) * s.share, tokens = s.share * x.Tq;         // tokens: of one head
            const uint32_t to = own + slot_ahead * 2 * TILE;
#pragma unroll
            for (int i = 0; i < 16 * MT * PIECES / 32; ++i) {
                const int piece = lane + 32 * i, r = piece / PIECES, p = piece % PIECES;
                const int h = r / tokens, rest = r - h * tokens, a = rest / x.Tq, token = rest - a * x.Tq;
                const bool there = r < s.rows && 8 * p < x.C;
                const DT* src = static_cast<const DT*>(x.q.ptr) +
                                (there ? (long long)(i0 + a) * x.q.b + (ahead.m * x.G + h) * x.q.n + token * x.q.t + 8 * p : 0);
                copy_16(to + At::at(r, p), src, there);
            }
            rows_due = false;
        } else if (ahead.any()) {
            const int key0 = step * kStep;
            const uint32_t to = own + slot_ahead * 2 * TILE;
#pragma unroll
            for (int i = 0; i < kStep * PIECES / 32; ++i) {
                const int piece = lane + 32 * i, r = piece / PIECES, p = piece % PIECES, key = key0 + r;
                const bool there = key < unit_keys && 8 * p < x.C;       // beyond: zeros, whatever memory holds
                const long long row = there ? key : 0;
                copy_16(to + At::at(r, p), kp + row * k_t + (there ? 8 * p : 0), there);
                copy_16(to + TILE + At::at(r, p), vp + row * v_t + (there ? 8 * p : 0), there);
            }
            if (++step == stop) {
                ahead.next(before, x.Nk);
                enter();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (++slot_ahead == NST) slot_ahead = 0;
    };
#pragma unroll 1
    for (int i = 0; i < NST - 1; ++i) ask();

    const int r_lo = lane / 4, c_lo = 2 * (lane % 4);    // of a fragment: rows r_lo and r_lo + 8, columns c_lo, + 1
    int c0 = 0, c1 = 0;
    auto settle = [&]() {                                // on to a unit of which the stretch has steps
        for (; here.any(); here.next(before, x.Nk)) {
            here.steps(before, x.Nk, c0, c1);
            if (c0 < c1) return true;
        }
        return false;
    };
    while (settle()) {
        const bool second = here.e >= E0;
        const TokenSide& side = x.side[second];
        const int i0 = second ? here.e - E0 : here.e, m = here.m, count = token_keys(x, here.e), unit = i0 * x.Nk + m;
        const int tokens = side.share * x.Tq;            // of one head
        // Q as the first product's operand, and the keys that the thread's rows see
        uint32_t qf[MT][D / 16][4];
        int seen[MT][2];
        auto arrive = [&]() {                            // the next stage is there, one more is asked for
            ask();
            asm volatile("cp.async.wait_group %0;" ::"n"(NST - 1) : "memory");
            __syncwarp();
            const uint32_t at = own + slot * 2 * TILE;
            if (++slot == NST) slot = 0;
            return at;
        };
        {
            const uint32_t tq = arrive();
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    load_matrices(qf[t][kk], tq + At::at(16 * t + (lane & 15), 2 * kk + (lane >> 4)));
            __syncwarp();
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = 16 * t + r_lo + 8 * half, token = r % tokens % x.Tq;
                seen[t][half] = r >= side.rows ? 0 : second && x.causal ? max(count - x.Tq + 1 + token, 0) : count;
            }
        float acc[MT][D / 8][4], top[MT][2], total[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            top[t][0] = top[t][1] = -CUDART_INF_F;
            total[t][0] = total[t][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][i][e] = 0.f;
        }
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
            const uint32_t tk = arrive(), tv = tk + TILE;
            // scores of the rows and 16 keys
            float s[MT][2][4];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][j][e] = 0.f;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                uint32_t kb[4];                          // keys 0-7: channels 0-7, 8-15; keys 8-15: the same
                load_matrices(kb, tk + At::at((lane & 7) + 8 * (lane >> 4), 2 * kk + ((lane >> 3) & 1)));
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    mma_16816<DT>(s[t][0], qf[t][kk], kb[0], kb[1]);
                    mma_16816<DT>(s[t][1], qf[t][kk], kb[2], kb[3]);
                }
            }
            const int key0 = c * kStep;
            float high[MT][2];
            bool grows = false;
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float& h = high[t][half];
                    h = -CUDART_INF_F;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float& y = s[t][j][2 * half + e];
                            y = key0 + 8 * j + c_lo + e < seen[t][half] ? y * x.sl2 : -CUDART_INF_F;
                            h = fmaxf(h, y);
                        }
                    h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, 1));
                    h = fmaxf(h, __shfl_xor_sync(0xffffffffu, h, 2));
                    grows = grows || h > top[t][half] + kGrow || (top[t][half] == -CUDART_INF_F && h > top[t][half]);
                }
            if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float to = fmaxf(top[t][half], high[t][half]), base = to == -CUDART_INF_F ? 0.f : to;
                        const float alpha = fast_exp2(top[t][half] - base);
                        top[t][half] = to;
                        total[t][half] *= alpha;
#pragma unroll
                        for (int j = 0; j < D / 8; ++j) {
                            acc[t][j][2 * half] *= alpha;
                            acc[t][j][2 * half + 1] *= alpha;
                        }
                    }
            }
            uint32_t p[MT][4];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float base = (top[t][half] == -CUDART_INF_F ? 0.f : top[t][half]) - kLift<DT>;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float p0 = fast_exp2(s[t][j][2 * half] - base), p1 = fast_exp2(s[t][j][2 * half + 1] - base);
                        total[t][half] += p0 + p1;
                        p[t][half + 2 * j] = pack2<DT>(p0, p1);          // (rounded once for the product, as everywhere in attention's forward)
                    }
                }
#pragma unroll
            for (int jj = 0; jj < D / 16; ++jj) {
                uint32_t vb[4];                          // channels 0-7: keys 0-7, 8-15; channels 8-15: the same
                load_matrices_transposed(vb, tv + At::at(lane & 15, 2 * jj + (lane >> 4)));
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    mma_16816<DT>(acc[t][2 * jj], p[t], vb[0], vb[1]);
                    mma_16816<DT>(acc[t][2 * jj + 1], p[t], vb[2], vb[3]);
                }
            }
            __syncwarp();                                // the stage has been read
        }
        // the sums -> the unit's part
        const size_t part = side.first_row + static_cast<size_t>(own_warp + unit) * side.rows;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float all_of = total[t][half];
                all_of += __shfl_xor_sync(0xffffffffu, all_of, 1);
                all_of += __shfl_xor_sync(0xffffffffu, all_of, 2);
                const int r = 16 * t + r_lo + 8 * half;
                if (r >= side.rows) continue;
                const bool none = all_of == 0.f;
                const float inv = none ? 0.f : 1.f / all_of, base = top[t][half] == -CUDART_INF_F ? 0.f : top[t][half];
                float* to = x.part_o + (part + r) * x.C + c_lo;
#pragma unroll
                for (int j = 0; j < D / 8; ++j)
                    if (8 * j < x.C)
                        *reinterpret_cast<float2*>(to + 8 * j) = none ? make_float2(0.f, 0.f)
                                                                      : make_float2(acc[t][j][2 * half] * inv, acc[t][j][2 * half + 1] * inv);
                if (lane % 4 == 0) x.part_lse[part + r] = none ? -CUDART_INF_F : (base - kLift<DT> + log2f(all_of)) * kLn2;
            }
        here.next(before, x.Nk);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (x.behind) after_previous_grid();
}

// A row's parts of one side: rows first, first + stride, ... of o and lse.
struct PartList {
    const float *o, *lse;
    size_t first, stride;
    int count;
};
template <bool OWN>
__device__ __forceinline__ PartList parts_of(const Tokens& x, const JoinPrefix& j, int b, int n, int t) {
    PartList l{};
    const TokenSide& s = x.side[OWN];
    const int share = OWN ? 1 : j.share;
    int entry = b, a = 0;
    if (share > 1) entry = j.by_share.split(b, a);
    const size_t row = static_cast<size_t>(a) * x.Tq + t;
    if (!OWN && j.count > 0) {                           // of another kernel: rows of (entries, N, share Tq)
        l.o = j.o;
        l.lse = j.lse;
        l.first = (static_cast<size_t>(entry) * x.N + n) * share * x.Tq + row;
        l.stride = j.stride;
        l.count = j.count;
        return l;
    }
    if (s.entries == 0) return l;
    int h;
    const int e = (OWN ? x.side[0].entries : 0) + entry, m = x.by_g.split(n, h), unit = entry * x.Nk + m;
    const int E = x.side[0].entries + x.side[1].entries, each = x.table[E + 1], before = x.table[e], length = x.table[e + 1] - before;
    if (length == 0) return l;
    const int at = before * x.Nk + m * length, lo = (at + kUnitSteps) / each, hi = (at + length - 1) / each;       // warps with steps of it
    l.o = x.part_o;
    l.lse = x.part_lse;
    l.stride = s.rows;
    l.first = s.first_row + static_cast<size_t>(lo + unit) * s.rows + static_cast<size_t>(h) * share * x.Tq + row;
    l.count = hi - lo + 1;
    return l;
}

// lse = ln sum_s e^lse_s, o = sum_s e^(lse_s - lse) o_s over a row's parts of both sides.  A block a row: its warps share the parts, 4
// channels a lane; where they lie and what they weigh, each lane of a warp works out for one of 32.
template <typename DT>
__global__ void __launch_bounds__(128) prefix_join_kernel(const __grid_constant__ Tokens x, const __grid_constant__ JoinPrefix prefix,
                                                          DT* __restrict__ o, float* __restrict__ lse) {
    constexpr int W = 4;
    __shared__ float4 sums[W][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x, c = 4 * lane;
    int t, n;
    const int b = x.by_n.split(x.by_tq.split(row, t), n);
    after_previous_grid();
    next_grid_may_start();
    const PartList first = parts_of<false>(x, prefix, b, n, t), second = parts_of<true>(x, prefix, b, n, t);
    const int parts = first.count + second.count;
    auto part = [&](int i, const float*& at) {           // lse of part i, and its o
        const PartList& l = i < first.count ? first : second;
        const size_t r = l.first + (i < first.count ? i : i - first.count) * l.stride;
        at = l.o + r * x.C;
        return l.lse[r];
    };
    const float* at = nullptr;
    float of = lane < parts ? part(lane, at) : -CUDART_INF_F, top = of;
    for (int i = lane + 32; i < parts; i += 32) {
        const float* ignored;
        top = fmaxf(top, part(i, ignored));
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    // (a NaN of a part stays one: the maximum skips it, its weight does not)
    const float base = top == -CUDART_INF_F ? 0.f : top;
    float total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < parts; i0 += 32) {
        if (i0 > 0) of = i0 + lane < parts ? part(i0 + lane, at) : -CUDART_INF_F;
        const float w = of == -CUDART_INF_F ? 0.f : expf(of - base);
        total += w;
        const unsigned there = __ballot_sync(0xffffffffu, of != -CUDART_INF_F);      // of the others nothing was written
        const unsigned long long place = reinterpret_cast<unsigned long long>(at);
#pragma unroll
        for (int k = 0; k < 32 / W; ++k) {
            const int j = W * k + warp;
            if (i0 + W * k >= parts) break;
            const float by = __shfl_sync(0xffffffffu, w, j);
            const float* from = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, place, j));
            if ((there >> j & 1) && c < x.C) {
                const float4 v = *reinterpret_cast<const float4*>(from + c);
                acc.x = fmaf(by, v.x, acc.x);
                acc.y = fmaf(by, v.y, acc.y);
                acc.z = fmaf(by, v.z, acc.z);
                acc.w = fmaf(by, v.w, acc.w);
            }
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    if (warp > 0) sums[warp][lane] = acc;
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
        acc.x += sums[w][lane].x;
        acc.y += sums[w][lane].y;
        acc.z += sums[w][lane].z;
        acc.w += sums[w][lane].w;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    if (c < x.C) store_4(o + static_cast<size_t>(row) * x.C + c, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    if (lane == 0) lse[row] = total == 0.f ? -CUDART_INF_F : base + logf(total);
}

}  // namespace na2d_prefix
