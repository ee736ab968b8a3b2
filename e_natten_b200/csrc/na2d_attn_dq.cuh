// Attention over all keys, query half of the backward, on tcgen05 (bf16 / fp16, head dims up to 128).
//
//     S = Q K_c^T,  dP = dO V_c^T                          (tensor memory, fp32)
//     P = exp(S - lse),  dS = P (dP - delta)               (softmax warps)
//     dQ += dS K_c                                         (dS from tensor memory, 16 bit)
// with delta = dO . o of the row, formed ahead by delta_kernel.  dS goes into its product as two numbers of 16 bits, what it rounds to and
// the rest: rounded to one, it put dQ 1.4 to 1.5 times as far from its 64-bit value as dQ's own rounding does, and together with the rounding of
// o in delta up to 1.7 times; now that is up to 1.3 times.  The softmax scale comes in the epilogue, and in fp16, whose numbers end at 2^-24 and
// 2^16, so does the power of two that each row's dS carries (ds_shift; P has it as a summand of its exponent).
//
// Bound as the key half is: 8 heads x 16384 x 128, causal, bf16: 1024 us, 805 TFLOP/s over three products (with dS in one number: 782 us).
//
// Where tiles and CTAs do not go into one another (few rows and many keys, one tile more than a round), the chunks of all tiles lie on one
// line, of which every CTA takes the same stretch; what it has of a tile that it does not see all keys of goes to a workspace as fp32 sums,
// which attn_join_rows_kernel adds in their order (4 x 4 heads x 4096 x 128, 512 tiles, dS
// in one number: 178 us for 228; in two: 223).
//
// Persistent, one CTA per SM, one tile of 128 query rows at a time, keys in chunks of 128.  S has two buffers, so that the
// exponentials of chunk n + 1 run while dQ and dP of chunks n and n + 1 are on the tensor pipe; dS goes over dP.
//   warps 0-7   softmax: warps w and w + 4 share 32 rows and take 64 columns each;
//   warp 8      producer (Q, dO, K, V);  warp 9  MMA issue;  warp 11  clears the rows of K beyond a batch entry's keys;
//   warps 12-15 epilogue.
#pragma once

#include "na2d_attn_fwd.cuh"

namespace na2d_attn {

// delta = dO . o of each row, 8 channels a lane; fp16: the norms of dO and, by the blocks behind row_blocks, of V, too.  LPR lanes a row:
// C / 8, rounded up to a power of two.  A lane has kDeltaRows rows of one head, 256 / LPR apart, all under way at once (8 x 16 heads x 3136 x
// 64: 16.5 us, 6.2 TB/s, with the norms 19; with one row a lane 24).
constexpr int kDeltaRows = 4;
template <typename DT, int LPR>
__global__ void __launch_bounds__(256)
attn_delta_kernel(const DT* __restrict__ d_o, const Operand st_do, const DT* __restrict__ o, const Operand st_o, float* __restrict__ delta,
                  const Geom g, const Div by_tiles, const Div by_heads, const Operand v, const Bounds bounds, const Div by_key_tiles,
                  const unsigned row_blocks) {
    after_previous_grid();
    next_grid_may_start();
    constexpr int kStep = 256 / LPR;
    // the largest of the block's squares, none of them infinite -> `to` (a maximum has no order; every warp by itself, 2000 at one
    // address, took 20 us longer)
    auto largest = [](float x, float* to) {
        __shared__ unsigned warps[8];
        const unsigned top = __reduce_max_sync(0xffffffffu, __float_as_uint(x));
        if (threadIdx.x % 32 == 0) warps[threadIdx.x / 32] = top;
        __syncthreads();
        if (threadIdx.x >= 32) return;
        const unsigned all = __reduce_max_sync(0xffffffffu, warps[threadIdx.x % 8]);
        if (threadIdx.x == 0 && all) atomicMax(reinterpret_cast<unsigned*>(to), all);
    };
    if (!IsBf16<DT>::value && blockIdx.x >= row_blocks) {
        int tile, m;
        const int unit = by_key_tiles.split(blockIdx.x - row_blocks, tile), b = g.by_nk.split(unit, m), part = threadIdx.x % LPR;
        const int k0 = tile * kDeltaRows * kStep + threadIdx.x / LPR, count = key_count(g, b);
        const DT* x = static_cast<const DT*>(v.ptr) + b * v.b + m * v.n + 8 * part;
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kDeltaRows; ++i) {
            const int key = k0 + i * kStep;
            const uint4 vx = key < count && 8 * part < g.C ? __ldg(reinterpret_cast<const uint4*>(x + key * v.t)) : make_uint4(0u, 0u, 0u, 0u);
            float square = na2d_delta::dot8<DT>(vx, vx, 0.f);
#pragma unroll
            for (int d = LPR / 2; d > 0; d >>= 1) square += __shfl_xor_sync(0xffffffffu, square, d);
            if (square < CUDART_INF_F) top = fmaxf(top, square);
        }
        largest(top, bounds.unit + 2 * unit + 1);
        return;
    }
    int tile, n;
    const int bn = by_tiles.split(blockIdx.x, tile), b = by_heads.split(bn, n);
    const int part = threadIdx.x % LPR, t0 = tile * kDeltaRows * kStep + threadIdx.x / LPR;
    const DT *x = d_o + b * st_do.b + n * st_do.n + 8 * part, *y = o + b * st_o.b + n * st_o.n + 8 * part;
    uint4 vx[kDeltaRows], vy[kDeltaRows];
#pragma unroll
    for (int i = 0; i < kDeltaRows; ++i) {
        const int t = t0 + i * kStep;
        vx[i] = vy[i] = make_uint4(0u, 0u, 0u, 0u);
        if (t < g.Tq && 8 * part < g.C) {
            vx[i] = __ldg(reinterpret_cast<const uint4*>(x + t * st_do.t));
            vy[i] = __ldg(reinterpret_cast<const uint4*>(y + t * st_o.t));
        }
    }
    const int count = IsBf16<DT>::value ? 0 : key_count(g, b);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < kDeltaRows; ++i) {
        float acc = na2d_delta::dot8<DT>(vx[i], vy[i], 0.f);
#pragma unroll
        for (int d = LPR / 2; d > 0; d >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, d);
        const int t = t0 + i * kStep;
        if (part == 0 && t < g.Tq) delta[static_cast<size_t>(bn) * g.Tq + t] = acc;
        if constexpr (!IsBf16<DT>::value) {
            float square = na2d_delta::dot8<DT>(vx[i], vx[i], 0.f);
#pragma unroll
            for (int d = LPR / 2; d > 0; d >>= 1) square += __shfl_xor_sync(0xffffffffu, square, d);
            if (part == 0 && t < g.Tq) bounds.row[static_cast<size_t>(bn) * g.Tq + t] = square;
            if (t < g.Tq && keys_seen(g, count, t) > 0 && square < CUDART_INF_F) top = fmaxf(top, square);
        }
    }
    if constexpr (!IsBf16<DT>::value) largest(top, bounds.unit + 2 * (b * g.Nk + n / g.G));
}

struct RowCut {
    int items;              // tiles
    int line;               // the chunks of all tiles on one line, that many CTAs take; 0: an item is a tile
    float* part;            // line: (2 a CTA, rows of a tile, C)
};

// One item: chunks [c0, c0 + n) of a tile of rows.
struct RowItem {
    RowTile tile;
    int c0, n;
    int part;               // its place in the workspace, -1 where it has all of the tile's chunks
};
// The items of a CTA, which every role walks by itself.  (LINE when compiled: the other form's code in every role of a kernel whose items are
// short costs it 15 %.)
template <bool LINE>
struct RowWalk {
    int item, at, end;
    __device__ __forceinline__ RowWalk(const Geom& g, const RowCut& cut, const int* before) : item(blockIdx.x), at(0), end(0) {
        if constexpr (!LINE) return;
        const int all = before[g.B] * g.Nk * g.tiles, each = (all + cut.line - 1) / cut.line;
        at = min((int)blockIdx.x * each, all);
        end = min(at + each, all);
    }
    __device__ __forceinline__ bool more(const RowCut& cut) const { return LINE ? at < end : item < cut.items; }
    __device__ __forceinline__ RowItem get(const Geom& g, const RowCut& cut, const int* before) const {
        RowItem x;
        int unit, tile;
        if constexpr (LINE) {
            const int per_entry = g.Nk * g.tiles;
            int lo = 0, hi = g.B;                        // before[lo] per_entry <= at < before[hi] per_entry
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (before[mid] * per_entry <= at) lo = mid;
                else hi = mid;
            }
            const int own = at - before[lo] * per_entry, len = before[lo + 1] - before[lo], which = own / len;
            x.c0 = own - which * len;
            x.n = min(len - x.c0, end - at);
            x.part = x.n == len ? -1 : 2 * (int)blockIdx.x + (x.c0 == 0);
            unit = lo * g.Nk + g.by_tiles.split(which, tile);
            x.tile = RowTile(g, unit, tile);
        } else {
            if (g.causal) {                              // the longer tiles first
                tile = g.tiles - 1 - g.by_units.split(item, unit);
            } else {
                unit = g.by_tiles.split(item, tile);
            }
            x.tile = RowTile(g, unit, tile);
            x.c0 = 0;
            x.n = (x.tile.keys(g) + kRows - 1) / kRows;
            x.part = -1;
        }
        return x;
    }
    __device__ __forceinline__ void next(const RowItem& x) {
        if constexpr (LINE) at += x.n;
        else item += gridDim.x;
    }
};

template <int D>
struct DqCfg : TileCfg<D> {
    using T = TileCfg<D>;
    static constexpr int NST = D == 128 ? 2 : 4;                         // chunks of K, and of V
    static constexpr int NQ = D == 128 ? 1 : 2;                          // tiles of Q and dO: the next one's while this one's are read
    static constexpr int OUT_BYTES = 4 * 2 * OutStage<32>::BYTES;
    static constexpr int SMEM = 2 * NQ * T::BYTES + 2 * NST * T::BYTES + OUT_BYTES + 512 /*barriers*/ + 1024 /*alignment*/;
    static constexpr int TMEM_S = 0, TMEM_DP = 256, TMEM_DQ = 384;       // S: two buffers of 128 columns
    static_assert(SMEM <= kSmemLimit, "dQ kernel shared memory");
};

template <typename DT, int D, bool LINE>
__global__ void __launch_bounds__(512, 1)
attn_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
               const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
               const __grid_constant__ CUtensorMap tm_dq, DT* __restrict__ dq_rows, const Operand dq_st, const float* __restrict__ lse,
               const float* __restrict__ delta, const Bounds bounds, const ErrorState* __restrict__ errors, const Geom g, const RowCut cut) {
    using C = DqCfg<D>;
    constexpr int NST = C::NST, NQ = C::NQ;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int before[LINE ? kLineEntries + 1 : 1];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;
    uint8_t* sG = sQ + NQ * C::BYTES;                     // dO
    uint8_t* sK = sG + NQ * C::BYTES;                     // NST x K chunk
    uint8_t* sV = sK + NST * C::BYTES;                    // NST x V chunk
    uint8_t* sOut = sV + NST * C::BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sOut + C::OUT_BYTES);
    uint64_t* q_full = bars;                 // [2] TMA -> MMA: Q and dO
    uint64_t* q_empty = bars + 2;            // [2] MMA (commit) -> TMA
    uint64_t* s_full = bars + 4;             // [2] MMA (commit) -> softmax
    uint64_t* s_free = bars + 6;             // [2] softmax -> MMA: S is in registers
    uint64_t* dq_full = bars + 8;            //     MMA (commit) -> epilogue
    uint64_t* dq_free = bars + 9;            //     epilogue -> MMA
    uint64_t* dp_full = bars + 10;           //     MMA (commit) -> softmax
    uint64_t* ds_full = bars + 11;           //     softmax -> MMA
    uint64_t* k_full = bars + 12;            // [4] TMA -> MMA: K and V chunk
    uint64_t* k_empty = bars + 16;           // [4] MMA (commit) -> TMA
    uint64_t* k_clear = bars + 20;           // [4] warp 11 -> MMA
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
    const WaitCtx wctx{reinterpret_cast<WaitState*>(bars + 25)};

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        wait_state_init(wctx.st, errors, kWaitLimitNs);
        mbar_init(dq_full, 1);
        mbar_init(dq_free, 4);
        mbar_init(dp_full, 1);
        mbar_init(ds_full, 8);
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + i, 1);
            mbar_init(q_empty + i, 1);
            mbar_init(s_full + i, 1);
            mbar_init(s_free + i, 8);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(k_full + i, 1);
            mbar_init(k_empty + i, 1);
            mbar_init(k_clear + i, 1);
        }
        mbar_fence_init();
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_do);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        tma_prefetch_desc(&tm_dq);
    }
    after_previous_grid();
    if (warp == 0) {
        __syncwarp();
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (LINE && warp == 1) line_table(g, before, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    next_grid_may_start();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 8) {
        // ------------------------------------------------------------------ producer
        reg_dec<kDkvRegsCtl>();
        if (lane == 0) {
            LoadTracker lt(bars);
            Ring ring;
            uint32_t it = 0;
            for (RowWalk<LINE> walk(g, cut, before); walk.more(cut) && lt.ok;) {
                const RowItem x = walk.get(g, cut, before);
                const RowTile& t = x.tile;
                const int n = x.n;
                walk.next(x);
                if (n == 0) continue;
                const uint32_t to = it % NQ, phase = (it / NQ) & 1;
                if (!lt.acquire(q_empty + to, phase ^ 1, wctx)) break;
                lt.arm(q_full + to, phase, 2 * C::load_bytes(g.hp * g.tt));
#pragma unroll
                for (int s = 0; s < C::NS; ++s) {
                    tma_load_5d(sQ + to * C::BYTES + s * C::SLAB, &tm_q, q_full + to, s * 64, t.t0, t.h0, t.b, 0);
                    tma_load_5d(sG + to * C::BYTES + s * C::SLAB, &tm_do, q_full + to, s * 64, t.t0, t.h0, t.b, 0);
                }
                ++it;
                for (int c = 0; c < n; ++c) {
                    if (!lt.acquire(k_empty + ring.at, ring.phase ^ 1, wctx)) break;
                    lt.arm(k_full + ring.at, ring.phase, 2 * C::BYTES);
#pragma unroll
                    for (int s = 0; s < C::NS; ++s) {
                        tma_load_5d(sK + ring.at * C::BYTES + s * C::SLAB, &tm_k, k_full + ring.at, s * 64, (x.c0 + c) * kRows, t.m, t.b, 0);
                        tma_load_5d(sV + ring.at * C::BYTES + s * C::SLAB, &tm_v, k_full + ring.at, s * 64, (x.c0 + c) * kRows, t.m, t.b, 0);
                    }
                    ring.next(NST);
                }
            }
            lt.drain(wctx);
        }
    } else if (warp == 11) {
        // ------------------------------------------------------------------ zeros beyond the keys
        reg_dec<kDkvRegsCtl>();
        if (g.lengths) {
            Ring ring;
            for (RowWalk<LINE> walk(g, cut, before); walk.more(cut);) {
                const RowItem x = walk.get(g, cut, before);
                const RowTile& t = x.tile;
                const int n = x.n, ragged = fwd_ragged_chunk(g, t.count, x.c0, n);
                walk.next(x);
                for (int c = 0; c < n; ++c) {
                    if (c == ragged) {
                        mbar_wait(k_full + ring.at, ring.phase, wctx, kErrLoadWait);
                        __syncwarp();
                        clear_rows<D>(sK + ring.at * C::BYTES, t.count % kRows, lane);
                        if (lane == 0) mbar_arrive(k_clear + ring.at);
                    } else if (lane == 0) {
                        mbar_wait(k_full + ring.at, ring.phase, wctx, kErrLoadWait);
                        mbar_arrive(k_clear + ring.at);
                    }
                    ring.next(NST);
                }
            }
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------------ MMA issue
        // Order on the tensor pipe: S(0) dP(0) S(1) | dQ(0) dP(1) S(2) | dQ(1) dP(2) S(3) | ...
        reg_dec<kDkvRegsCtl>();
        constexpr uint32_t idesc_s = umma_idesc(kRows, kRows, IsBf16<DT>::value, IsBf16<DT>::value, false, false);
        constexpr uint32_t idesc_o = umma_idesc(kRows, D, IsBf16<DT>::value, IsBf16<DT>::value, false, true);
        constexpr uint32_t hi = smem_desc_hi(C::ATOM, C::SWZ);
        const uint32_t q_lo = smem_desc_lo(smem_u32(sQ), 16), g_lo = smem_desc_lo(smem_u32(sG), 16);
        const uint32_t k_lo0 = smem_desc_lo(smem_u32(sK), 16), v_lo0 = smem_desc_lo(smem_u32(sV), 16);
        const uint32_t km_lo0 = smem_desc_lo(smem_u32(sK), C::SLAB);
        // D (128 columns) = A B^T of two K-major operands
        auto product = [&](uint32_t t_d, uint32_t a_lo, uint32_t b_lo) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                constexpr int kPerSlab = C::SLAB_C / 16;
                const int at = (((kk / kPerSlab) * C::SLAB) >> 4) + 2 * (kk % kPerSlab);
                umma_ss(t_d, desc64(hi, a_lo + at), desc64(hi, b_lo + at), idesc_s, kk > 0);
            }
        };
        Ring rs, rp, ro;                     // places of the chunks that S, dP and dQ are at
        uint32_t ns = 0, no = 0, it = 0;     // chunks that S and dQ are at, tiles
        auto scores = [&](uint32_t tile) {
            mbar_wait(k_full + rs.at, rs.phase, wctx, kErrLoadWait);
            if (g.lengths) mbar_wait(k_clear + rs.at, rs.phase, wctx, kErrOther);
            mbar_wait(s_free + (ns & 1), ((ns >> 1) & 1) ^ 1, wctx, kErrMmaWait);
            tc_fence_after();
            if (elect_one()) {
                product(tmem_base + C::TMEM_S + (ns & 1) * kRows, q_lo + tile % NQ * (C::BYTES >> 4), k_lo0 + rs.at * (C::BYTES >> 4));
                umma_commit(s_full + (ns & 1));
            }
            __syncwarp();
            ++ns;
            rs.next(NST);
        };
        auto grads = [&](bool last) {        // (by the elected lane; its chunk has landed: S came before)
            product(tmem_base + C::TMEM_DP, g_lo + it % NQ * (C::BYTES >> 4), v_lo0 + rp.at * (C::BYTES >> 4));
            umma_commit(dp_full);
            if (last) umma_commit(q_empty + it % NQ);
        };
        bool ahead = false;                  // the tile's first scores have been issued
        RowWalk<LINE> walk(g, cut, before);
        // chunks of the walk's item (asked for ahead: a length is a load from memory)
        auto take = [&]() {
            if (!walk.more(cut)) return -1;
            const RowItem x = walk.get(g, cut, before);
            walk.next(x);
            return x.n;
        };
        int next = take();
        while (next >= 0) {
            const int n = next;
            next = take();
            if (n == 0) continue;
            if (!ahead) {
                mbar_wait(q_full + it % NQ, (it / NQ) & 1, wctx, kErrLoadWait);
                scores(it);
            }
            if (elect_one()) grads(n == 1);  // (dS of the chunk before has been read: dQ came before on the pipe)
            __syncwarp();
            rp.next(NST);
            for (int c = 0; c < n; ++c, ++no) {
                if (lane == 0) NA2D_TR(2, 0, no);
                if (c + 1 < n) {
                    scores(it);
                } else {                     // with room for its Q: the next tile's first scores, under this one's last chunk
                    ahead = NQ > 1 && next > 0;
                    if (ahead) {
                        mbar_wait(q_full + (it + 1) % NQ, ((it + 1) / NQ) & 1, wctx, kErrLoadWait);
                        scores(it + 1);
                    }
                }
                if (lane == 0) NA2D_TR(2, 1, no);
                if (c == 0) mbar_wait(dq_free, (it & 1) ^ 1, wctx, kErrMmaWait);
                mbar_wait(ds_full, no & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if (lane == 0) NA2D_TR(2, 2, no);
                if (elect_one()) {
                    const uint32_t km_lo = km_lo0 + ro.at * (C::BYTES >> 4);
#pragma unroll
                    for (int kk = 0; kk < kRows / 8; ++kk)       // a warp's half of dS: 32 columns of pairs over its own half of dP, then the rests
                        umma_ts(tmem_base + C::TMEM_DQ, tmem_base + C::TMEM_DP + (kk % 8 / 4) * 64 + kk / 8 * 32 + (kk % 4) * 8,
                                desc64(hi, km_lo + ((kk % 8 * 16 * C::ROWB) >> 4)), idesc_o, (c > 0) || (kk > 0));
                    umma_commit(k_empty + ro.at);
                    if (c + 1 < n) grads(c + 2 == n);
                    else umma_commit(dq_full);
                }
                __syncwarp();
                if (c + 1 < n) rp.next(NST);
                ro.next(NST);
                if (lane == 0) NA2D_TR(2, 3, no);
            }
            ++it;
        }
    } else if (warp == 10) {
        reg_dec<kDkvRegsCtl>();
    } else if (warp >= 12) {
        // ------------------------------------------------------------------ epilogue warps
        reg_dec<kDkvRegsEpi>();
        const int quarter = warp & 3;
        const int row = quarter * 32 + lane;
        const uint32_t tmem_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        uint8_t* stage = sOut + quarter * 2 * OutStage<32>::BYTES;
        uint32_t it = 0, seq = 0;
        for (RowWalk<LINE> walk(g, cut, before); walk.more(cut);) {
            const RowItem x = walk.get(g, cut, before);
            const RowTile& tile = x.tile;
            const bool none = x.n == 0;
            walk.next(x);
            int n, t;
            const bool ok = tile.row(g, row, n, t);
            const int t_first = tile.t0 + quarter * 32;
            float scale = g.scale;
            if constexpr (!IsBf16<DT>::value) {
                if (ok && !none)
                    scale *= exp2i(-ds_shift(__ldg(bounds.row + row_index(g, tile.b, n, t)), __ldg(bounds.unit + 2 * (tile.b * g.Nk + tile.m) + 1)));
            }
            const bool blind = g.causal && keys_seen(g, tile.count, t) == 0;         // (beside rows that see: dS = 0 meets any key of theirs)
            if (!none) {
                mbar_wait(dq_full, it & 1, wctx, kErrMmaWait);
                tc_fence_after();
            }
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                uint32_t v[32];
                if (!none) {
                    tmem_ld_32x32(tmem_lane + C::TMEM_DQ + 32 * j, v);
                    tmem_ld_wait();
                    if (j + 1 == D / 32) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(dq_free);
                    }
                }
                if (none || blind) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = 0u;
                }
                if (32 * j >= g.C) continue;
                if (LINE && x.part >= 0) {
                    float4* dst = reinterpret_cast<float4*>(cut.part + (static_cast<size_t>(x.part) * kRows + row) * g.C + 32 * j);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (ok && 32 * j + 4 * e < g.C)
                            dst[e] = make_float4(__uint_as_float(v[4 * e]) * scale, __uint_as_float(v[4 * e + 1]) * scale,
                                                 __uint_as_float(v[4 * e + 2]) * scale, __uint_as_float(v[4 * e + 3]) * scale);
                } else if (g.hp == 1) {
                    if (t_first < g.Tq)
                        na2d_tc::stage_and_store<DT, 32, 2>(&tm_dq, stage, v, scale, 32 * j, t_first, tile.h0, tile.b, 0, lane, &seq);
                } else if (ok) {
                    uint4* dst = reinterpret_cast<uint4*>(dq_rows + tile.b * dq_st.b + n * dq_st.n + t * dq_st.t + 32 * j);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (32 * j + 8 * e < g.C) {
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                w[i] = pack2<DT>(__uint_as_float(v[8 * e + 2 * i]) * scale, __uint_as_float(v[8 * e + 2 * i + 1]) * scale);
                            dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                }
            }
            if (!none) ++it;
        }
        if (lane == 0) bulk_wait<0>();
    } else {
        // ------------------------------------------------------------------ softmax warps
        reg_inc<kDkvRegsSoftmax>();
        const int quarter = warp & 3, half = warp >> 2;
        const int row = quarter * 32 + lane;
        const uint32_t tmem_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t dp_addr = tmem_lane + C::TMEM_DP + 64 * half;
        const uint64_t scale2 = pair2(g.sl2, g.sl2);
        uint32_t m = 0;                                      // chunks so far
        // lse and delta of a row (fp16: and the squares that its dS are bounded by): read an item ahead, since few chunks to an item would
        // not cover the way to memory
        RowItem next;
        float next_lse, next_delta, next_row = 0.f, next_unit = 0.f;
        RowWalk<LINE> walk(g, cut, before);
        auto fetch = [&]() {
            next.n = -1;
            next_lse = -CUDART_INF_F;
            next_delta = 0.f;
            if (!walk.more(cut)) return;
            next = walk.get(g, cut, before);
            walk.next(next);
            int n, t;
            if (!next.tile.row(g, row, n, t)) return;
            const size_t at = row_index(g, next.tile.b, n, t);
            next_lse = __ldg(lse + at);
            next_delta = __ldg(delta + at);
            if constexpr (!IsBf16<DT>::value) {
                next_row = __ldg(bounds.row + at);
                next_unit = __ldg(bounds.unit + 2 * (next.tile.b * g.Nk + next.tile.m) + 1);
            }
        };
        fetch();
        while (next.n >= 0) {
            const RowTile tile = next.tile;
            const int chunks = next.n, c0 = next.c0;
            const float row_lse = next_lse, row_delta = next_delta, shift = IsBf16<DT>::value ? 0.f : (float)ds_shift(next_row, next_unit);
            fetch();
            if (chunks == 0) continue;
            int n, t;
            const bool ok = tile.row(g, row, n, t);
            const bool idle = !__any_sync(0xffffffffu, ok);
            // a row that sees nothing has weights of zero: exp2(-infinity)
            const float neg = row_lse == -CUDART_INF_F ? -CUDART_INF_F : IsBf16<DT>::value ? -row_lse * kLog2e : shift - row_lse * kLog2e;
            const uint64_t neg2 = pair2(neg, neg), delta2 = pair2(-row_delta, -row_delta);
            const int seen = (ok ? keys_seen(g, tile.count, t) : 0) - 64 * half - c0 * kRows;      // from the item's first chunk on
            for (int c = 0; c < chunks; ++c, ++m) {
                uint64_t pr[32];
                if ((tid & 127) == 0) NA2D_TR(half ? 0 : 3, 0, m);
                mbar_wait(s_full + (m & 1), (m >> 1) & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if ((tid & 127) == 0) NA2D_TR(half ? 0 : 3, 1, m);
                if (!idle) {
                    uint32_t s[2][32];
                    const uint32_t s_addr = tmem_lane + C::TMEM_S + (m & 1) * kRows + 64 * half;
                    tmem_ld_32x32(s_addr, s[0]);
                    tmem_ld_32x32(s_addr + 32, s[1]);
                    tmem_ld_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_free + (m & 1));
#pragma unroll
                    for (int e2 = 0; e2 < 32; ++e2) {
                        const uint64_t y = fma2(pair2(s[e2 / 16][2 * (e2 % 16)], s[e2 / 16][2 * (e2 % 16) + 1]), scale2, neg2);
                        pr[e2] = pair2(fast_exp2(lo2(y)), fast_exp2(hi2(y)));
                    }
                } else if (lane == 0) {
                    mbar_arrive(s_free + (m & 1));
                }
                if ((tid & 127) == 0) NA2D_TR(half ? 0 : 3, 2, m);
                mbar_wait(dp_full, m & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if ((tid & 127) == 0) NA2D_TR(half ? 0 : 3, 3, m);
                if (!idle) {
                    uint32_t dp[2][32], w[2][16];
                    tmem_ld_32x32(dp_addr, dp[0]);
                    tmem_ld_32x32(dp_addr + 32, dp[1]);
                    tmem_ld_wait();
#pragma unroll
                    for (int e2 = 0; e2 < 32; ++e2)
                        pr[e2] = mul2(pr[e2], add2(pair2(dp[e2 / 16][2 * (e2 % 16)], dp[e2 / 16][2 * (e2 % 16) + 1]), delta2));
                    const int open = seen - c * kRows;       // columns of this half that the row sees
                    if (__any_sync(0xffffffffu, open < 64)) {
                        // by selection: columns that are not seen may hold anything
#pragma unroll
                        for (int e = 0; e < 64; e += 2)
                            pr[e / 2] = pair2(e >= open ? 0.f : lo2(pr[e / 2]), e + 1 >= open ? 0.f : hi2(pr[e / 2]));
                    }
#pragma unroll
                    for (int e2 = 0; e2 < 32; ++e2) w[e2 / 16][e2 % 16] = pack2<DT>(lo2(pr[e2]), hi2(pr[e2]));
                    // (over columns of dP that this warp has read: dS in the first half of its own, its rests in the second)
                    tmem_st_32x16(dp_addr, w[0]);
                    tmem_st_32x16(dp_addr + 16, w[1]);
#pragma unroll
                    for (int e2 = 0; e2 < 32; ++e2) w[e2 / 16][e2 % 16] = pack_rest<DT>(pr[e2], w[e2 / 16][e2 % 16]);
                    tmem_st_32x16(dp_addr + 32, w[0]);
                    tmem_st_32x16(dp_addr + 48, w[1]);
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ds_full);
                if ((tid & 127) == 0) NA2D_TR(half ? 0 : 3, 4, m);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

template <typename DT>
int launch_delta(const Place& at, const Geom& g, const Operand& d_o, const Operand& o, const Operand& v, float* delta, const Bounds& bounds) {
    const int lanes = g.C <= 32 ? 4 : g.C <= 64 ? 8 : 16, rows = kDeltaRows * 256 / lanes, tiles = (g.Tq + rows - 1) / rows;
    const int key_tiles = (g.Tk + rows - 1) / rows;
    const long long row_blocks = (long long)g.B * g.N * tiles, blocks = row_blocks + (IsBf16<DT>::value ? 0 : (long long)g.units * key_tiles);
    if (blocks > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    if (!IsBf16<DT>::value && cudaMemsetAsync(bounds.unit, 0, (size_t)g.units * 2 * sizeof(float), at.st) != cudaSuccess) return NA2D_ERR_CUDA;
    auto kern = lanes == 4 ? attn_delta_kernel<DT, 4> : lanes == 8 ? attn_delta_kernel<DT, 8> : attn_delta_kernel<DT, 16>;
    *at.launched += 1;
    return na2d_launch::launch(false, kern, (unsigned)blocks, 256, 0, at.st, (const DT*)d_o.ptr, d_o, (const DT*)o.ptr, o, delta, g, Div(tiles),
                               Div(g.N), v, bounds, Div(key_tiles), (unsigned)row_blocks) == cudaSuccess
               ? NA2D_OK
               : NA2D_ERR_CUDA;
}

// Line: a block joins the parts of an eighth of one tile of rows, or writes zeros where the batch entry has no keys.  (A block a tile
// read sixteen times one after the other: 24 us for 19 MB.)
constexpr int kJoinBlocks = 8, kJoinRows = kRows / kJoinBlocks;
template <typename DT>
__global__ void __launch_bounds__(256)
attn_join_rows_kernel(const float* __restrict__ part, DT* __restrict__ dq, const Operand st, const Geom g, const RowCut cut) {
    after_previous_grid();
    next_grid_may_start();
    int which, m, before = 0, all = 0;                   // chunks of a tile of the entries before b, and of all
    const int unit = g.by_tiles.split(blockIdx.x, which), b = g.by_nk.split(unit, m), lane = threadIdx.x & 31;
    for (int i = lane; i < g.B; i += 32) {
        const int chunks = (key_count(g, i) + kRows - 1) / kRows;
        all += chunks;
        if (i < b) before += chunks;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, d);
        before += __shfl_xor_sync(0xffffffffu, before, d);
    }
    const RowTile tile(g, unit, which);
    const int chunks = (tile.count + kRows - 1) / kRows, each = (all * g.Nk * g.tiles + cut.line - 1) / cut.line;
    const int at = (before * g.Nk + m * chunks) * g.tiles + which * chunks;
    const int lo = chunks ? at / each : 0, hi = chunks ? (at + chunks - 1) / each : 0;       // CTAs that have some of it
    if (chunks && lo == hi) return;                      // one had them all
    const int vectors = g.C / 4;
    for (int i = threadIdx.x; i < kJoinRows * vectors; i += 256) {
        const int own = i / vectors, c = 4 * (i - own * vectors), r = blockIdx.y * kJoinRows + own;
        int n, t;
        if (!tile.row(g, r, n, t)) continue;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (chunks) {
#pragma unroll 4
            for (int s = lo; s <= hi; ++s) {             // lo has the tile's first chunk
                const float4 v = *reinterpret_cast<const float4*>(part + ((2 * s + (s == lo)) * static_cast<size_t>(kRows) + r) * g.C + c);
                acc.x += v.x;
                acc.y += v.y;
                acc.z += v.z;
                acc.w += v.w;
            }
        }
        *reinterpret_cast<uint2*>(dq + tile.b * st.b + n * st.n + t * st.t + c) = make_uint2(pack2<DT>(acc.x, acc.y), pack2<DT>(acc.z, acc.w));
    }
}

template <typename DT, int D>
int launch_dq(const Place& at, const Geom& g, RowCut cut, const Operand& q, const Operand& k, const Operand& v, const Operand& d_o, const float* lse,
              const float* delta, const Bounds& bounds, const Operand& d_q) {
    using C = DqCfg<D>;
    CUtensorMap tq, tg, tk, tv, tdq;
    int rc = operand_map(&tq, q, at.dtype, g.B, g.N, g.Tq, g.C, g.tt, g.hp, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&tg, d_o, at.dtype, g.B, g.N, g.Tq, g.C, g.tt, g.hp, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&tk, k, at.dtype, g.B, g.Nk, g.Tk, g.C, kRows, 1, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&tv, v, at.dtype, g.B, g.Nk, g.Tk, g.C, kRows, 1, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&tdq, d_q, at.dtype, g.B, g.N, g.Tq, g.C, 32, 1, 32);
    if (rc != NA2D_OK) return rc;
    const long long items = (long long)g.units * g.tiles;
    if (items > 0x3fffffffLL) return NA2D_ERR_TOO_LARGE;
    cut.items = (int)items;
    auto kern = cut.line ? attn_dq_kernel<DT, D, true> : attn_dq_kernel<DT, D, false>;
    static std::atomic<unsigned long long> opted[2]{};
    if (na2d_tc::opt_in_smem(kern, C::SMEM, at.device, opted[cut.line > 0]) != cudaSuccess) return NA2D_ERR_CUDA;
    const int sms = na2d_tc::sm_count(at.device);
    *at.launched += 1;
    if (na2d_launch::launch(true, kern, cut.line ? cut.line : items < sms ? (int)items : sms, 512, C::SMEM, at.st, tq, tg, tk, tv, tdq, (DT*)d_q.ptr,
                            d_q, lse, delta, bounds, at.errors, g, cut) != cudaSuccess)
        return NA2D_ERR_CUDA;
    if (!cut.line) return NA2D_OK;
    *at.launched += 1;
    return na2d_launch::launch(true, attn_join_rows_kernel<DT>, dim3((unsigned)items, kJoinBlocks), 256, 0, at.st, (const float*)cut.part, (DT*)d_q.ptr, d_q, g,
                               cut) == cudaSuccess
               ? NA2D_OK
               : NA2D_ERR_CUDA;
}

}  // namespace na2d_attn
