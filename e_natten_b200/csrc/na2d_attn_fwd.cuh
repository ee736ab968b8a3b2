// Attention over all keys, forward, on tcgen05 (bf16 / fp16, head dims up to 128).
//
// Persistent, one CTA per SM, two tiles of 128 query rows in flight: softmax group a (warps 0-3) has one, group b (warps 4-7) the
// other, each with an S / P buffer and an output accumulator of its own in tensor memory.  Keys are walked in chunks of 128; on the
// tensor pipe
//     S_a(0) S_b(0) | PV_a(0) S_a(1) | PV_b(0) S_b(1) | ...
// so that one group's MMAs run under the other group's exponentials.  PAIR: the two tiles are neighbours of one unit and share every
// chunk of K and V in shared memory; else (units of a single tile) each has its own.
//
// Few rows and many keys: the keys of a tile are cut into `splits` parts, each an item of its own, whose o (fp32) and lse go to a
// workspace and are joined by combine_kernel.
//
//   warps 0-7   softmax: a thread owns a row, reads its 128 scores, writes P over S as packed 16-bit pairs;
//   warps 8, 10 producers of Q and K, and of V;    warp 9  MMA issue;
//   warp 11     clears the rows of V beyond a batch entry's keys;
//   warps 12-15 epilogue: o and lse of either group while its next tile is under way.
#pragma once

#include "na2d_attn.cuh"

namespace na2d_attn {

using namespace na2d_ptx;
using na2d_tc::fast_exp2;
using na2d_tc::IsBf16;
using na2d_tc::kDkvRegsCtl;
using na2d_tc::kDkvRegsEpi;
using na2d_tc::kDkvRegsSoftmax;
using na2d_tc::kLn2;
using na2d_tc::kLog2e;
using na2d_tc::kSmemLimit;
using na2d_tc::max3;
using na2d_tc::OutStage;
using na2d_tc::pack2;
using na2d_tc::Ring;

// How the work is cut: items of two tiles (or two parts of tiles).
struct FwdCut {
    int splits;
    int pairs;              // PAIR: items of a unit and split
    int items;
    float* part_o;          // (splits, B, N, Tq, C), where splits > 1
    float* part_lse;        // (splits, B, N, Tq)
};

// One group's half of an item: chunks [c0, c0 + n) of a tile.
struct FwdPart {
    RowTile tile;
    bool any;               // there is a tile
    int split, c0, n;
};

template <bool PAIR>
__device__ __forceinline__ void fwd_parts(const Geom& g, const FwdCut& cut, int item, FwdPart (&p)[2]) {
    if constexpr (PAIR) {
        const int split = item % cut.splits, rest = item / cut.splits;
        // with a causal mask the later tiles are the longer ones: they go first, so that no CTA is left with one at the end
        const int pair = g.causal ? cut.pairs - 1 - rest / g.units : rest % cut.pairs;
        const int unit = g.causal ? rest % g.units : rest / cut.pairs;
        int chunks[2], most = 0;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            p[x].any = 2 * pair + x < g.tiles;
            p[x].tile = RowTile(g, unit, p[x].any ? 2 * pair + x : 2 * pair);
            chunks[x] = p[x].any ? (p[x].tile.keys(g) + kRows - 1) / kRows : 0;
            most = max(most, chunks[x]);
        }
        const int c0 = (int)((long long)most * split / cut.splits), c1 = (int)((long long)most * (split + 1) / cut.splits);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            p[x].split = split;
            p[x].c0 = c0;
            p[x].n = max(min(chunks[x], c1) - c0, 0);
        }
    } else {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int f = 2 * item + x;
            p[x].any = f < g.units * cut.splits;
            p[x].split = p[x].any ? f / g.units : 0;
            p[x].tile = RowTile(g, p[x].any ? f - p[x].split * g.units : 0, 0);
            const int chunks = (p[x].tile.keys(g) + kRows - 1) / kRows;
            p[x].c0 = (int)((long long)chunks * p[x].split / cut.splits);
            p[x].n = p[x].any ? (int)((long long)chunks * (p[x].split + 1) / cut.splits) - p[x].c0 : 0;
        }
    }
}

// The part's chunk that holds keys beyond its batch entry's (and not beyond Tk, where TMA fills with zeros), or -1.
__device__ __forceinline__ int fwd_ragged_chunk(const Geom& g, int count, int c0, int n) {
    const int at = count / kRows - c0;
    return count % kRows != 0 && count < g.Tk && at >= 0 && at < n ? at : -1;
}

template <int D>
struct FwdCfg : TileCfg<D> {
    using T = TileCfg<D>;
    static constexpr int NST = D == 128 ? 2 : 4;                         // chunks of K, and of V
    static constexpr int OUT_BYTES = 4 * 2 * OutStage<32>::BYTES;        // two staging buffers for each epilogue warp
    static constexpr int X_BYTES = 2 * 2 * 2 * kRows * 4;                // row sum, final maximum [group][tile parity][row]
    static constexpr int SMEM = 2 * T::BYTES + 2 * NST * T::BYTES + OUT_BYTES + X_BYTES + 512 /*barriers*/ + 1024 /*alignment*/;
    static constexpr int TMEM_S = 0, TMEM_O = 256;                       // of group x: S + 128 x, O + D x
    static_assert(SMEM <= kSmemLimit, "forward kernel shared memory");
};

// Logarithm (base 2) by which a row's maximum may grow before its sums are rescaled: the weights stay below 2^8, within fp16 by far,
// and most chunks after the first rescale nothing.
constexpr float kGrow = 8.f;

template <typename DT, int D, bool PAIR>
__global__ void __launch_bounds__(512, 1)
attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o, DT* __restrict__ o_rows,
                const Operand o_st, float* __restrict__ lse, const ErrorState* __restrict__ errors, const Geom g, const FwdCut cut) {
    using C = FwdCfg<D>;
    constexpr int NST = C::NST;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;                                   // Q tile of each group
    uint8_t* sK = sQ + 2 * C::BYTES;                      // NST x K chunk
    uint8_t* sV = sK + NST * C::BYTES;                    // NST x V chunk
    uint8_t* sOut = sV + NST * C::BYTES;                  // output staging
    float* x_sum = reinterpret_cast<float*>(sOut + C::OUT_BYTES);     // [group][tile parity][row]
    float* x_fin = x_sum + 4 * kRows;
    uint64_t* bars = reinterpret_cast<uint64_t*>(x_fin + 4 * kRows);
    uint64_t* q_full = bars;                 // [2] TMA -> MMA, per group
    uint64_t* q_empty = bars + 2;            // [2] MMA (commit) -> TMA
    uint64_t* o_full = bars + 4;             // [2] MMA (commit) -> epilogue
    uint64_t* o_free = bars + 6;             // [2] epilogue -> MMA
    uint64_t* s_full = bars + 8;             // [2] MMA (commit) -> softmax
    uint64_t* p_full = bars + 10;            // [2] softmax -> MMA
    uint64_t* k_full = bars + 12;            // [4] TMA -> MMA
    uint64_t* k_empty = bars + 16;           // [4] MMA (commit) -> TMA
    uint64_t* v_full = bars + 20;            // [4] TMA -> MMA
    uint64_t* v_empty = bars + 24;           // [4] MMA (commit) -> TMA
    uint64_t* v_clear = bars + 28;           // [4] warp 11 -> MMA: rows beyond the keys are zeros
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 32);
    const WaitCtx wctx{reinterpret_cast<WaitState*>(bars + 33)};

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        wait_state_init(wctx.st, errors, kWaitLimitNs);
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + i, 1);
            mbar_init(q_empty + i, 1);
            mbar_init(o_full + i, 1);
            mbar_init(o_free + i, 4);
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 4);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(k_full + i, 1);
            mbar_init(k_empty + i, 1);
            mbar_init(v_full + i, 1);
            mbar_init(v_empty + i, 1);
            mbar_init(v_clear + i, 1);
        }
        mbar_fence_init();
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        tma_prefetch_desc(&tm_o);
    }
    after_previous_grid();
    if (warp == 0) {
        __syncwarp();
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    next_grid_may_start();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 8 || warp == 10) {
        // ------------------------------------------------------------------ producers
        // (warp 8: Q and K, whose buffers the score MMAs release early; warp 10: V)
        reg_dec<kDkvRegsCtl>();
        if (lane == 0) {
            LoadTracker lt(bars);
            Ring ring;
            uint32_t it[2] = {0, 0};
            for (int item = blockIdx.x; item < cut.items && lt.ok; item += gridDim.x) {
                FwdPart p[2];
                fwd_parts<PAIR>(g, cut, item, p);
                if (warp == 8) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (p[x].n == 0) continue;
                        if (!lt.acquire(q_empty + x, (it[x] & 1) ^ 1, wctx)) break;
                        lt.arm(q_full + x, it[x] & 1, C::load_bytes(g.hp * g.tt));
#pragma unroll
                        for (int s = 0; s < C::NS; ++s)
                            tma_load_5d(sQ + x * C::BYTES + s * C::SLAB, &tm_q, q_full + x, s * 64, p[x].tile.t0, p[x].tile.h0,
                                        p[x].tile.b, 0);
                        ++it[x];
                    }
                }
                const int most = max(p[0].n, p[1].n);
                for (int c = 0; c < most && lt.ok; ++c) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (PAIR ? x == 1 : c >= p[x].n) continue;       // (a pair's tiles have their unit and first chunk in common)
                        // (the tensor map is named in each call: a map chosen through a run-time pointer may be
                        // copied to local memory, where TMA cannot read it)
                        if (warp == 8) {
                            if (!lt.acquire(k_empty + ring.at, ring.phase ^ 1, wctx)) break;
                            lt.arm(k_full + ring.at, ring.phase, C::BYTES);
#pragma unroll
                            for (int s = 0; s < C::NS; ++s)
                                tma_load_5d(sK + ring.at * C::BYTES + s * C::SLAB, &tm_k, k_full + ring.at, s * 64,
                                            (p[x].c0 + c) * kRows, p[x].tile.m, p[x].tile.b, 0);
                        } else {
                            if (!lt.acquire(v_empty + ring.at, ring.phase ^ 1, wctx)) break;
                            lt.arm(v_full + ring.at, ring.phase, C::BYTES);
#pragma unroll
                            for (int s = 0; s < C::NS; ++s)
                                tma_load_5d(sV + ring.at * C::BYTES + s * C::SLAB, &tm_v, v_full + ring.at, s * 64,
                                            (p[x].c0 + c) * kRows, p[x].tile.m, p[x].tile.b, 0);
                        }
                        ring.next(NST);
                    }
                }
            }
            lt.drain(wctx);
        }
    } else if (warp == 11) {
        // ------------------------------------------------------------------ zeros beyond the keys
        reg_dec<kDkvRegsCtl>();
        if (g.lengths) {
            Ring ring;
            for (int item = blockIdx.x; item < cut.items; item += gridDim.x) {
                FwdPart p[2];
                fwd_parts<PAIR>(g, cut, item, p);
                const int most = max(p[0].n, p[1].n);
                const int at[2] = {fwd_ragged_chunk(g, p[0].tile.count, p[0].c0, PAIR ? most : p[0].n),
                                   PAIR ? -1 : fwd_ragged_chunk(g, p[1].tile.count, p[1].c0, p[1].n)};
                for (int c = 0; c < most; ++c) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (PAIR ? x == 1 : c >= p[x].n) continue;
                        if (c == at[x]) {
                            mbar_wait(v_full + ring.at, ring.phase, wctx, kErrLoadWait);
                            __syncwarp();
                            clear_rows<D>(sV + ring.at * C::BYTES, p[x].tile.count % kRows, lane);
                            if (lane == 0) mbar_arrive(v_clear + ring.at);
                        } else if (lane == 0) {
                            mbar_wait(v_full + ring.at, ring.phase, wctx, kErrLoadWait);
                            mbar_arrive(v_clear + ring.at);
                        }
                        ring.next(NST);
                    }
                }
            }
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------------ MMA issue
        // (the whole warp walks the loop so that addresses stay warp-uniform; one lane issues)
        reg_dec<kDkvRegsCtl>();
        constexpr uint32_t idesc_s = umma_idesc(kRows, kRows, IsBf16<DT>::value, IsBf16<DT>::value, false, false);
        constexpr uint32_t idesc_o = umma_idesc(kRows, D, IsBf16<DT>::value, IsBf16<DT>::value, false, true);
        constexpr uint32_t hi = smem_desc_hi(C::ATOM, C::SWZ);
        // The steps in their order: chunk c of group x of an item; a group that has fewer chunks than the other leaves steps out.
        struct Place {
            int item, n[2], c = 0, x = 0;
            uint32_t tile[2] = {0, 0}, chunk[2] = {0, 0};        // of the group so far
            __device__ __forceinline__ void read(const Geom& g, const FwdCut& cut) {
                while (item < cut.items) {                       // items without chunks have no steps
                    FwdPart p[2];
                    fwd_parts<PAIR>(g, cut, item, p);
                    n[0] = p[0].n;
                    n[1] = p[1].n;
                    if (max(n[0], n[1]) > 0) return;
                    item += gridDim.x;
                }
            }
            __device__ __forceinline__ void next(const Geom& g, const FwdCut& cut) {
#pragma unroll
                for (int y = 0; y < 2; ++y)
                    if (x == y && c < n[y]) {
                        ++chunk[y];
                        if (c + 1 == n[y]) ++tile[y];
                    }
                x ^= 1;
                if (x == 0 && ++c == max(n[0], n[1])) {
                    c = 0;
                    item += gridDim.x;
                    read(g, cut);
                }
            }
            __device__ __forceinline__ int mine() const { return x ? n[1] : n[0]; }
            __device__ __forceinline__ uint32_t tiles() const { return x ? tile[1] : tile[0]; }
            __device__ __forceinline__ uint32_t chunks() const { return x ? chunk[1] : chunk[0]; }
            // the last step that reads this chunk's buffer
            __device__ __forceinline__ bool last() const { return !PAIR || x == 1 || c >= n[1]; }
        };
        const uint32_t q_lo0 = smem_desc_lo(smem_u32(sQ), 16), k_lo0 = smem_desc_lo(smem_u32(sK), 16);
        const uint32_t v_lo0 = smem_desc_lo(smem_u32(sV), C::SLAB);
        Ring rk, rv;
        Place ps, po;
        ps.item = po.item = blockIdx.x;
        ps.read(g, cut);
        po.read(g, cut);
        auto scores = [&]() {
            const int x = ps.x;
            if (ps.c < ps.mine()) {
                if (ps.c == 0) mbar_wait(q_full + x, ps.tiles() & 1, wctx, kErrLoadWait);
                mbar_wait(k_full + rk.at, rk.phase, wctx, kErrLoadWait);
                tc_fence_after();
                const uint32_t q_lo = q_lo0 + x * (C::BYTES >> 4), k_lo = k_lo0 + rk.at * (C::BYTES >> 4);
                const uint32_t t_s = tmem_base + C::TMEM_S + x * kRows;
                const bool end = ps.c + 1 == ps.mine(), last = ps.last();
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        constexpr int kPerSlab = C::SLAB_C / 16;
                        const int at = (((kk / kPerSlab) * C::SLAB) >> 4) + 2 * (kk % kPerSlab);
                        umma_ss(t_s, desc64(hi, q_lo + at), desc64(hi, k_lo + at), idesc_s, kk > 0);
                    }
                    umma_commit(s_full + x);                                  // and P V of the group's chunk before
                    if (last) umma_commit(k_empty + rk.at);
                    if (end) umma_commit(q_empty + x);
                }
                __syncwarp();
                if (last) rk.next(NST);
            }
            ps.next(g, cut);
        };
        auto outputs = [&]() {
            const int x = po.x;
            if (po.c < po.mine()) {
                if (po.c == 0) mbar_wait(o_free + x, (po.tiles() & 1) ^ 1, wctx, kErrMmaWait);      // the tile before has been read out
                mbar_wait(v_full + rv.at, rv.phase, wctx, kErrLoadWait);
                if (g.lengths) mbar_wait(v_clear + rv.at, rv.phase, wctx, kErrOther);
                mbar_wait(p_full + x, po.chunks() & 1, wctx, kErrMmaWait);
                tc_fence_after();
                const uint32_t v_lo = v_lo0 + rv.at * (C::BYTES >> 4);
                const uint32_t t_p = tmem_base + C::TMEM_S + x * kRows, t_o = tmem_base + C::TMEM_O + x * D;
                const bool end = po.c + 1 == po.mine(), last = po.last();
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < kRows / 16; ++kk)
                        umma_ts(t_o, t_p + 8 * kk, desc64(hi, v_lo + ((kk * 16 * C::ROWB) >> 4)), idesc_o, (po.c > 0) || (kk > 0));
                    if (last) umma_commit(v_empty + rv.at);
                    if (end) umma_commit(o_full + x);
                }
                __syncwarp();
                if (last) rv.next(NST);
            }
            po.next(g, cut);
        };
        // A group's next scores go into the buffer that its P V has just read; the pipe runs its MMAs in the order they were issued.
        for (int s = 0; s < 2 && ps.item < cut.items; ++s) scores();
        while (po.item < cut.items) {
            outputs();
            if (ps.item < cut.items) scores();
        }
    } else if (warp >= 12) {
        // ------------------------------------------------------------------ epilogue warps
        reg_dec<kDkvRegsEpi>();
        const int quarter = warp & 3;
        const int row = quarter * 32 + lane;                 // row of the tile = tensor-memory lane
        const uint32_t tmem_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        uint8_t* stage = sOut + quarter * 2 * OutStage<32>::BYTES;
        const bool by_tma = g.hp == 1 && cut.splits == 1;
        uint32_t it[2] = {0, 0}, seq = 0;
        for (int item = blockIdx.x; item < cut.items; item += gridDim.x) {
            FwdPart p[2];
            fwd_parts<PAIR>(g, cut, item, p);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (!p[x].any) continue;
                int n, t;
                const bool ok = p[x].tile.row(g, row, n, t);
                const size_t at = row_index(g, p[x].tile.b, n, t);
                const bool none = p[x].n == 0;               // no key: zeros
                float total = 0.f, fin = 0.f;
                if (!none) {
                    mbar_wait(o_full + x, it[x] & 1, wctx, kErrMmaWait);          // also: the group's sums are written
                    tc_fence_after();
                    total = x_sum[(x * 2 + (it[x] & 1)) * kRows + row];
                    fin = x_fin[(x * 2 + (it[x] & 1)) * kRows + row];
                }
                const float inv = total == 0.f ? 0.f : 1.f / total;
                const int h_first = p[x].tile.h0, t_first = p[x].tile.t0 + quarter * 32;
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    uint32_t v[32];
                    if (!none) {
                        tmem_ld_32x32(tmem_lane + C::TMEM_O + x * D + 32 * j, v);
                        tmem_ld_wait();
                        if (j + 1 == D / 32) {                                    // O has been read
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(o_free + x);
                        }
                        if (total == 0.f) {                                       // a row that sees nothing: what P V made of it is not read
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] = 0u;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = 0u;
                    }
                    if (32 * j >= g.C) continue;
                    if (by_tma) {
                        if (t_first < g.Tq)
                            na2d_tc::stage_and_store<DT, 32, 2>(&tm_o, stage, v, inv, 32 * j, t_first, h_first, p[x].tile.b, 0, lane, &seq);
                    } else if (ok && cut.splits == 1) {
                        uint4* dst = reinterpret_cast<uint4*>(o_rows + p[x].tile.b * o_st.b + n * o_st.n + t * o_st.t + 32 * j);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (32 * j + 8 * e < g.C) {
                                uint32_t w[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    w[i] = pack2<DT>(__uint_as_float(v[8 * e + 2 * i]) * inv, __uint_as_float(v[8 * e + 2 * i + 1]) * inv);
                                dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                    } else if (ok && !none) {
                        float4* dst = reinterpret_cast<float4*>(cut.part_o + (p[x].split * (static_cast<size_t>(g.B) * g.N * g.Tq) + at) * g.C + 32 * j);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (32 * j + 4 * e < g.C)
                                dst[e] = make_float4(__uint_as_float(v[4 * e]) * inv, __uint_as_float(v[4 * e + 1]) * inv,
                                                     __uint_as_float(v[4 * e + 2]) * inv, __uint_as_float(v[4 * e + 3]) * inv);
                    }
                }
                if (ok) {
                    float* to = cut.splits == 1 ? lse + at : cut.part_lse + p[x].split * (static_cast<size_t>(g.B) * g.N * g.Tq) + at;
                    *to = total == 0.f ? -CUDART_INF_F : (fin + log2f(total)) * kLn2;
                }
                if (!none) ++it[x];
            }
        }
        if (lane == 0) bulk_wait<0>();                       // the staging buffers have been read, the rows written
    } else {
        // ------------------------------------------------------------------ softmax warps
        reg_inc<kDkvRegsSoftmax>();
        const int quarter = warp & 3, group = warp >> 2;
        const int row = quarter * 32 + lane;                 // row of the tile = tensor-memory lane
        const uint32_t tmem_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t s_addr = tmem_lane + C::TMEM_S + group * kRows, o_addr = tmem_lane + C::TMEM_O + group * D;
        uint32_t m = 0, it = 0;                              // chunks and tiles of this group so far
        const uint64_t scale2 = pair2(g.sl2, g.sl2);
        for (int item = blockIdx.x; item < cut.items; item += gridDim.x) {
            FwdPart both[2];
            fwd_parts<PAIR>(g, cut, item, both);
            const FwdPart p = group ? both[1] : both[0];
            if (p.n == 0) continue;
            int n, t;
            const bool ok = p.tile.row(g, row, n, t);
            const bool idle = !__any_sync(0xffffffffu, ok);  // no row of this warp is one of the tile: nothing is read of what it writes
            const int seen = (ok ? keys_seen(g, p.tile.count, t) : 0) - p.c0 * kRows;      // keys of this row, from the part's first chunk on
            float run_max = -CUDART_INF_F, run_sum = 0.f;
            for (int c = 0; c < p.n; ++c, ++m) {
                mbar_wait(s_full + group, m & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if (!idle) {
                    uint32_t s[4][32];
#pragma unroll
                    for (int a = 0; a < 4; ++a) tmem_ld_32x32(s_addr + 32 * a, s[a]);
                    tmem_ld_wait();
                    const int open = seen - c * kRows;       // columns of this chunk that the row sees
                    if (__any_sync(0xffffffffu, open < kRows)) {
                        // by selection: columns that are not seen may hold anything
#pragma unroll
                        for (int a = 0; a < 4; ++a)
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (32 * a + e >= open) s[a][e] = __float_as_uint(-CUDART_INF_F);
                    }
                    float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
                    for (int a = 0; a < 4; ++a)
#pragma unroll
                        for (int e = 0; e < 32; e += 2)
                            mx[a] = max3(mx[a], __uint_as_float(s[a][e]), __uint_as_float(s[a][e + 1]));
                    const float cmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * g.sl2;
                    const bool grow = cmax > run_max + kGrow || run_max == -CUDART_INF_F;
                    if (c > 0 && __any_sync(0xffffffffu, grow && cmax != -CUDART_INF_F)) {
                        // (O holds the chunks before: their P V went ahead of this chunk's scores)
                        const float alpha = grow && run_max != -CUDART_INF_F ? fast_exp2(run_max - cmax) : 1.f;
                        const uint64_t alpha2 = pair2(alpha, alpha);
#pragma unroll
                        for (int piece = 0; piece < D / 16; ++piece) {
                            uint32_t v[16];
                            tmem_ld_32x16(o_addr + 16 * piece, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                const uint64_t y = mul2(pair2(v[e], v[e + 1]), alpha2);
                                v[e] = __float_as_uint(lo2(y));
                                v[e + 1] = __float_as_uint(hi2(y));
                            }
                            tmem_st_32x16(o_addr + 16 * piece, v);
                        }
                        run_sum *= alpha;
                    }
                    if (grow) run_max = cmax;
                    const float safe_max = run_max == -CUDART_INF_F ? 0.f : run_max;
                    // P = exp2(s * scale * log2e - max) as packed 16-bit pairs -> tensor memory (over S), row sum
                    uint64_t sum2[2] = {0, 0};
                    const uint64_t max2 = pair2(-safe_max, -safe_max);
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        uint32_t w[16];
#pragma unroll
                        for (int e2 = 0; e2 < 16; ++e2) {
                            const uint64_t y = fma2(pair2(s[a][2 * e2], s[a][2 * e2 + 1]), scale2, max2);
                            const float p0 = fast_exp2(lo2(y)), p1 = fast_exp2(hi2(y));
                            sum2[e2 & 1] = add2(sum2[e2 & 1], pair2(p0, p1));
                            w[e2] = pack2<DT>(p0, p1);
                        }
                        tmem_st_32x16(s_addr + 16 * a, w);
                    }
                    const uint64_t sum = add2(sum2[0], sum2[1]);
                    run_sum += lo2(sum) + hi2(sum);
                    if (c + 1 == p.n) {              // for the epilogue warps, ahead of the arrival that lets the last P V go
                        x_sum[(group * 2 + (it & 1)) * kRows + row] = run_sum;
                        x_fin[(group * 2 + (it & 1)) * kRows + row] = safe_max;
                    }
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + group);
            }
            ++it;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// Joins the parts of a row: lse = ln sum_s e^lse_s, o = sum_s e^(lse_s - lse) o_s.  A warp a row, 4 channels a lane.
template <typename DT>
__global__ void __launch_bounds__(256)
attn_combine_kernel(const float* __restrict__ part_o, const float* __restrict__ part_lse, DT* __restrict__ o, const Operand o_st,
                    float* __restrict__ lse, const Geom g, const int splits) {
    after_previous_grid();
    next_grid_may_start();
    const size_t rows = static_cast<size_t>(g.B) * g.N * g.Tq;
    const size_t row = static_cast<size_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= rows) return;
    float top = -CUDART_INF_F;
    for (int s = lane; s < splits; s += 32) top = fmaxf(top, part_lse[s * rows + row]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    // (a NaN of a part stays one: the maximum skips it, its weight does not)
    const float base = top == -CUDART_INF_F ? 0.f : top;
    float total = 0.f;
    for (int s = lane; s < splits; s += 32) total += expf(part_lse[s * rows + row] - base);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int t = (int)(row % g.Tq);
    const size_t bn = row / g.Tq;
    DT* dst = o + (bn / g.N) * o_st.b + (bn % g.N) * o_st.n + t * o_st.t;
    for (int c = 4 * lane; c < g.C; c += 128) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < splits; ++s) {
            const float part = part_lse[s * rows + row];
            if (part == -CUDART_INF_F) continue;             // nothing was written for it
            const float w = expf(part - base) * inv;
            const float4 v = *reinterpret_cast<const float4*>(part_o + (s * rows + row) * g.C + c);
            acc.x = fmaf(w, v.x, acc.x);
            acc.y = fmaf(w, v.y, acc.y);
            acc.z = fmaf(w, v.z, acc.z);
            acc.w = fmaf(w, v.w, acc.w);
        }
        *reinterpret_cast<uint2*>(dst + c) = make_uint2(pack2<DT>(acc.x, acc.y), pack2<DT>(acc.z, acc.w));
    }
    if (lane == 0) lse[row] = total == 0.f ? -CUDART_INF_F : base + logf(total);
}

template <typename DT, int D, bool PAIR>
int launch_fwd_as(const Place& at, const Geom& g, const FwdCut& cut, const Operand& q, const Operand& k, const Operand& v,
                  const Operand& o, float* lse) {
    using C = FwdCfg<D>;
    CUtensorMap tq, tk, tv, to;
    int rc = operand_map(&tq, q, at.dtype, g.B, g.N, g.Tq, g.C, g.tt, g.hp, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&tk, k, at.dtype, g.B, g.Nk, g.Tk, g.C, kRows, 1, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&tv, v, at.dtype, g.B, g.Nk, g.Tk, g.C, kRows, 1, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&to, o, at.dtype, g.B, g.N, g.Tq, g.C, 32, 1, 32);
    if (rc != NA2D_OK) return rc;
    auto kern = attn_fwd_kernel<DT, D, PAIR>;
    static std::atomic<unsigned long long> opted{0};
    if (na2d_tc::opt_in_smem(kern, C::SMEM, at.device, opted) != cudaSuccess) return NA2D_ERR_CUDA;
    const int sms = na2d_tc::sm_count(at.device);
    *at.launched += 1;
    if (na2d_launch::launch(false, kern, cut.items < sms ? cut.items : sms, 512, C::SMEM, at.st, tq, tk, tv, to, (DT*)o.ptr, o, lse,
                            at.errors, g, cut) != cudaSuccess)
        return NA2D_ERR_CUDA;
    if (cut.splits == 1) return NA2D_OK;
    const long long rows = (long long)g.B * g.N * g.Tq;
    *at.launched += 1;
    return na2d_launch::launch(true, attn_combine_kernel<DT>, (unsigned)((rows + 7) / 8), 256, 0, at.st, (const float*)cut.part_o,
                               (const float*)cut.part_lse, (DT*)o.ptr, o, lse, g, cut.splits) == cudaSuccess
               ? NA2D_OK
               : NA2D_ERR_CUDA;
}

template <typename DT, int D>
int launch_fwd(const Place& at, const Geom& g, const FwdCut& cut, const Operand& q, const Operand& k, const Operand& v,
               const Operand& o, float* lse) {
    return g.tiles > 1 ? launch_fwd_as<DT, D, true>(at, g, cut, q, k, v, o, lse) : launch_fwd_as<DT, D, false>(at, g, cut, q, k, v, o, lse);
}

}  // namespace na2d_attn
