// Attention over all keys, key half of the backward, on tcgen05 (bf16 / fp16, head dims up to 128).
//
//     S^T = K Q_c^T,  dP^T = V dO_c^T                      (tensor memory, fp32)
//     P^T = exp(S^T - lse),  dS^T = P^T (dP^T - delta)     (softmax warps)
//     dV += P^T dO_c,  dK += dS^T Q_c                      (P^T, dS^T from tensor memory, 16 bit)
// over the query chunks of every head that shares the key head, accumulated in tensor memory: no atomics, and the order of the sums is
// the same in every call.  P is rounded once to 16 bits for its product (dV is 1.4 times as far from 64 bits as its own rounding puts it, like
// o); dS goes into its own as what it rounds to and the rest, as in the query half, in fp16 times a power of two (ds_shift, one for all
// rows of a unit, since they are summed).
//
// Bound by the chain from a chunk's scores to its dS: the tensor pipe works about half of the time (8 heads x 16384 x 128, causal: 1340 us,
// 820 TFLOP/s over four products; 4 x 4 heads x 4096 x 128: 284 us; 8 x 16 heads on 4 key heads, 3136 rows on up to 333 keys of 64: 102 us.
// With dS in one number 1115, 256 and 90 us; with items in place of the line the last one took 129).
//
// Persistent, one CTA per SM, one tile of 128 keys (row r of every MMA) at a time, queries in chunks of 128.  All 512 columns of
// tensor memory are in use, S^T and dP^T having one buffer each; the two halves of a chunk's arithmetic take turns with the MMAs:
//     softmax   P(n)         | dS(n)        | P(n+1)        | dS(n+1)
//     tensor          dP(n)  | dV(n) S(n+1) | dK(n) dP(n+1) | dV(n+1) ...
// Where tiles and CTAs do not go into one another, or batch entries have lengths of their own, the chunks of all tiles that hold a key lie on
// one line, of which every CTA takes the same stretch (causal calls, whose tiles see different numbers of chunks, cut a tile's chunks into
// `splits` parts where the tiles are few).  What a CTA has of a tile that it does not see all chunks of goes to a workspace as fp32 sums,
// which attn_join_kernel (attn_sum_kernel) adds in their order.
//   warps 0-7   softmax: warps w and w + 4 share 32 keys and take 64 queries each;
//   warp 8      producer of the Q / dO chunks and of the chunks' lse and delta;  warp 11  producer of the K, V tile;
//   warp 9      MMA issue;  warps 12-15 epilogue.
#pragma once

#include "na2d_attn_dq.cuh"
#include "na2d_attn_fwd.cuh"

namespace na2d_attn {

struct KeyCut {
    int key_tiles;
    int splits;
    int items;
    int each;               // chunks of a part
    int line;               // the chunks of all tiles that hold keys on one line, that many CTAs take; 0: not
    Div by_splits, by_key_tiles;
    float* part_dk;         // (splits, B, Nk, Tk, C), where splits > 1; line: (2 a CTA, keys of a tile, C)
    float* part_dv;
};

// A tile of keys by its number on the line; `before` as line_table writes it.
struct LineTile {
    int b, m, k0;
    __device__ __forceinline__ LineTile(const Geom& g, const int* before, int tile) {
        int lo = 0, hi = g.B;                            // before[lo] Nk <= tile < before[hi] Nk
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (before[mid] * g.Nk <= tile) lo = mid;
            else hi = mid;
        }
        const int own = tile - before[lo] * g.Nk, len = before[lo + 1] - before[lo];
        b = lo;
        m = own / len;
        k0 = (own - m * len) * kRows;
    }
};

// One item: chunks [first, first + n) of those that see a key tile.
struct KeyItem {
    int b, m, k0, count;
    int split;              // line: the part's place in the workspace, -1 for a whole tile
    int lo, per_head;       // the tile's chunks: query tiles lo .. lo + per_head - 1 of each (group of) heads
    int first, n, head, in_head;
    __device__ __forceinline__ KeyItem(const Geom& g, const KeyCut& cut, int item) {
        int tile, unit;
        const int rest = cut.by_splits.split(item, split);
        if (g.causal) {     // the first tiles are the longer ones
            tile = g.by_units.split(rest, unit);
        } else {
            unit = cut.by_key_tiles.split(rest, tile);
        }
        b = g.by_nk.split(unit, m);
        k0 = tile * kRows;
        count = key_count(g, b);
        const int t_min = g.causal ? max(k0 + g.Tq - count, 0) : 0;        // the first token that sees the tile
        lo = t_min / kRows;
        per_head = k0 < count && t_min < g.Tq ? g.tiles_t - lo : 0;
        const int all = per_head * g.groups;
        first = min(split * cut.each, all);
        n = min(cut.each, all - first);
        head = per_head > 0 ? first / per_head : 0;
        in_head = first - head * per_head;
    }
    // chunks from `at` on of a line that ends at `end`
    __device__ __forceinline__ KeyItem(const Geom& g, const int* before, int at, int end) {
        const int tile = g.by_tiles.split(at, first);
        const LineTile x(g, before, tile);
        b = x.b;
        m = x.m;
        k0 = x.k0;
        count = key_count(g, b);
        lo = 0;
        per_head = g.tiles_t;
        n = min(g.tiles - first, end - at);
        head = first / per_head;
        in_head = first - head * per_head;
        split = n == g.tiles ? -1 : 2 * (int)blockIdx.x + (first == 0);
    }
    // first head and token of the first chunk
    __device__ __forceinline__ void start(const Geom& g, int& h0, int& t0) const {
        h0 = m * g.G + head * g.hp;
        t0 = (lo + in_head) * kRows;
    }
    // and of the one behind
    __device__ __forceinline__ void step(const Geom& g, int& h0, int& t0) const {
        t0 += kRows;
        if (t0 == (lo + per_head) * kRows) {
            t0 = lo * kRows;
            h0 += g.hp;
        }
    }
};

// The items of a CTA, which every role walks by itself.
template <bool LINE>
struct KeyWalk {
    int item, at, end;
    __device__ __forceinline__ KeyWalk(const Geom& g, const KeyCut& cut, const int* before) : item(blockIdx.x), at(0), end(0) {
        if constexpr (!LINE) return;
        const int all = before[g.B] * g.Nk * g.tiles, each = (all + cut.line - 1) / cut.line;
        at = min((int)blockIdx.x * each, all);
        end = min(at + each, all);
    }
    __device__ __forceinline__ bool more(const KeyCut& cut) const { return LINE ? at < end : item < cut.items; }
    __device__ __forceinline__ KeyItem get(const Geom& g, const KeyCut& cut, const int* before) const {
        if constexpr (LINE) return KeyItem(g, before, at, end);
        else return KeyItem(g, cut, item);
    }
    __device__ __forceinline__ void next(const KeyItem& k) {
        if constexpr (LINE) at += k.n;
        else item += gridDim.x;
    }
};

template <int D>
struct KeyCfg : TileCfg<D> {
    using T = TileCfg<D>;
    static constexpr int NST = D == 128 ? 2 : 4;                         // chunks of Q and dO
    static constexpr int NKV = D == 128 ? 1 : 2;                         // tiles of K and V: the next one's while this one's are read
    static constexpr int OUT_BYTES = 4 * 2 * OutStage<32>::BYTES;
    // [ring slot]{-lse * log2(e), -delta}[row]; [ring slot] what dP is scaled by, twice
    static constexpr int X_BYTES = NST * 2 * kRows * 4 + NST * 8;
    static constexpr int SMEM = 2 * NKV * T::BYTES + 2 * NST * T::BYTES + OUT_BYTES + X_BYTES + 512 /*barriers*/ + 1024 /*alignment*/;
    static constexpr int TMEM_S = 0, TMEM_DP = 128, TMEM_DV = 256, TMEM_DK = 384;
    static_assert(SMEM <= kSmemLimit, "dK/dV kernel shared memory");
};

// P for its product, times 2^kShift: in fp16 the weights of long sequences would fall among the subnormal numbers.
template <typename DT> struct Weight {
    static constexpr int kBits = IsBf16<DT>::value ? 0 : 6;
    static constexpr float kShift = kBits, kUnit = IsBf16<DT>::value ? 1.f : 1.f / 64.f;
};
// The power of two that dS of a unit goes into its product with.
template <typename DT>
__device__ __forceinline__ int unit_shift(const Geom& g, const Bounds& bounds, const KeyItem& k) {
    if constexpr (IsBf16<DT>::value) return 0;
    const float2 squares = __ldg(reinterpret_cast<const float2*>(bounds.unit) + k.b * g.Nk + k.m);
    return ds_shift(squares.x, squares.y, g.joint ? __ldg(bounds.delta + k.b * g.Nk + k.m) : 0.f);
}

template <typename DT, int D, bool LINE>
__global__ void __launch_bounds__(512, 1)
attn_dkdv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                 const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                 const __grid_constant__ CUtensorMap tm_dk, const __grid_constant__ CUtensorMap tm_dv, const float* __restrict__ lse,
                 const float* __restrict__ delta, const Bounds bounds, const ErrorState* __restrict__ errors, const Geom g, const KeyCut cut) {
    using C = KeyCfg<D>;
    constexpr int NST = C::NST, NKV = C::NKV;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int before[LINE ? kLineEntries + 1 : 1];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sK = smem;
    uint8_t* sV = sK + NKV * C::BYTES;
    uint8_t* sQ = sV + NKV * C::BYTES;                    // NST x Q chunk
    uint8_t* sG = sQ + NST * C::BYTES;                    // NST x dO chunk
    uint8_t* sOut = sG + NST * C::BYTES;
    float* s_x = reinterpret_cast<float*>(sOut + C::OUT_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_x + C::X_BYTES / 4);
    uint64_t* kv_full = bars;                // [2] TMA -> MMA
    uint64_t* kv_empty = bars + 2;           // [2] MMA (commit) -> TMA
    uint64_t* acc_full = bars + 4;           //     MMA (commit) -> epilogue
    uint64_t* acc_free = bars + 5;           //     epilogue -> MMA
    uint64_t* s_full = bars + 6;             //     MMA (commit) -> softmax
    uint64_t* p_full = bars + 7;             //     softmax -> MMA
    uint64_t* dp_full = bars + 8;            //     MMA (commit) -> softmax
    uint64_t* ds_full = bars + 9;            //     softmax -> MMA
    uint64_t* qd_full = bars + 12;           // [4] TMA -> MMA
    uint64_t* qd_empty = bars + 16;          // [4] MMA (commit) -> TMA
    uint64_t* x_full = bars + 20;            // [4] producer -> MMA (and through it softmax): lse and delta
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
    const WaitCtx wctx{reinterpret_cast<WaitState*>(bars + 25)};

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        wait_state_init(wctx.st, errors, kWaitLimitNs);
        for (int i = 0; i < 2; ++i) {
            mbar_init(kv_full + i, 1);
            mbar_init(kv_empty + i, 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_free, 4);
        mbar_init(s_full, 1);
        mbar_init(p_full, 8);
        mbar_init(dp_full, 1);
        mbar_init(ds_full, 8);
        for (int i = 0; i < 4; ++i) {
            mbar_init(qd_full + i, 1);
            mbar_init(qd_empty + i, 1);
            mbar_init(x_full + i, 1);
        }
        mbar_fence_init();
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_do);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        tma_prefetch_desc(&tm_dk);
        tma_prefetch_desc(&tm_dv);
    }
    // Rows of a chunk that no copy writes (several heads of few tokens that do not fill 128 rows) are contraction rows all the same.
    if (g.hp * g.tt < kRows) {
        for (int i = tid; i < 2 * NST * C::BYTES / 16; i += 512) na2d_tc::st_shared_v4(smem_u32(sQ) + 16 * i, 0u, 0u, 0u, 0u);
        fence_proxy_async();
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
        // ------------------------------------------------------------------ producer of the Q / dO chunks
        reg_dec<kDkvRegsCtl>();
        LoadTracker lt(bars);
        Ring ring;
        for (KeyWalk<LINE> walk(g, cut, before); walk.more(cut) && lt.ok;) {
            const KeyItem k = walk.get(g, cut, before);
            walk.next(k);
            int h0, t0;
            k.start(g, h0, t0);
            const float unit = exp2i(unit_shift<DT>(g, bounds, k) - Weight<DT>::kBits);      // dS over P as it is here, and dP
            for (int i = 0; i < k.n; ++i, k.step(g, h0, t0)) {
                float x_lse[4], x_delta[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {                // (read ahead of the wait for a free slot)
                    const int r = lane + 32 * u, h = g.hp == 1 ? 0 : g.by_tt.quotient(r), t = t0 + r - h * g.tt;
                    x_lse[u] = -CUDART_INF_F;
                    x_delta[u] = 0.f;
                    if (h < g.hp && t < g.Tq) {
                        const size_t at = row_index(g, k.b, h0 + h, t);
                        x_lse[u] = lse[at];
                        x_delta[u] = delta[at];
                    }
                }
                if (!lt.acquire_warp(qd_empty + ring.at, ring.phase ^ 1, wctx)) break;
                if (lane == 0) {
                    lt.arm(qd_full + ring.at, ring.phase, 2 * C::load_bytes(g.hp * g.tt));
#pragma unroll
                    for (int s = 0; s < C::NS; ++s) {
                        tma_load_5d(sQ + ring.at * C::BYTES + s * C::SLAB, &tm_q, qd_full + ring.at, s * 64, t0, h0, k.b, 0);
                        tma_load_5d(sG + ring.at * C::BYTES + s * C::SLAB, &tm_do, qd_full + ring.at, s * 64, t0, h0, k.b, 0);
                    }
                }
                float* x = s_x + ring.at * 2 * kRows;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    // rows that see nothing, or are none: weights of exp2(-infinity)
                    x[lane + 32 * u] = x_lse[u] == -CUDART_INF_F ? -CUDART_INF_F : Weight<DT>::kShift - x_lse[u] * kLog2e;
                    x[kRows + lane + 32 * u] = -x_delta[u] * unit;
                }
                if (!IsBf16<DT>::value && lane == 0) reinterpret_cast<uint64_t*>(s_x + NST * 2 * kRows)[ring.at] = pair2(unit, unit);
                __syncwarp();
                if (lane == 0) mbar_arrive(x_full + ring.at);
                ring.next(NST);
            }
        }
        if (lane == 0) lt.drain(wctx);
    } else if (warp == 11) {
        // ------------------------------------------------------------------ producer of the K, V tile
        reg_dec<kDkvRegsCtl>();
        if (lane == 0) {
            LoadTracker lt(bars);
            uint32_t it = 0;
            for (KeyWalk<LINE> walk(g, cut, before); walk.more(cut);) {
                const KeyItem k = walk.get(g, cut, before);
                walk.next(k);
                if (k.n == 0) continue;
                const uint32_t to = it % NKV, phase = (it / NKV) & 1;
                if (!lt.acquire(kv_empty + to, phase ^ 1, wctx)) break;
                lt.arm(kv_full + to, phase, 2 * C::BYTES);
#pragma unroll
                for (int s = 0; s < C::NS; ++s) {
                    tma_load_5d(sK + to * C::BYTES + s * C::SLAB, &tm_k, kv_full + to, s * 64, k.k0, k.m, k.b, 0);
                    tma_load_5d(sV + to * C::BYTES + s * C::SLAB, &tm_v, kv_full + to, s * 64, k.k0, k.m, k.b, 0);
                }
                ++it;
            }
            lt.drain(wctx);
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------------ MMA issue
        reg_dec<kDkvRegsCtl>();
        constexpr uint32_t idesc_s = umma_idesc(kRows, kRows, IsBf16<DT>::value, IsBf16<DT>::value, false, false);
        constexpr uint32_t idesc_o = umma_idesc(kRows, D, IsBf16<DT>::value, IsBf16<DT>::value, false, true);
        constexpr uint32_t hi = smem_desc_hi(C::ATOM, C::SWZ);
        const uint32_t k_lo = smem_desc_lo(smem_u32(sK), 16), v_lo = smem_desc_lo(smem_u32(sV), 16);
        const uint32_t q_lo0 = smem_desc_lo(smem_u32(sQ), 16), g_lo0 = smem_desc_lo(smem_u32(sG), 16);
        const uint32_t qm_lo0 = smem_desc_lo(smem_u32(sQ), C::SLAB), gm_lo0 = smem_desc_lo(smem_u32(sG), C::SLAB);
        auto product = [&](uint32_t t_d, uint32_t a_lo, uint32_t b_lo) {          // D = A B^T of two K-major operands
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                constexpr int kPerSlab = C::SLAB_C / 16;
                const int at = (((kk / kPerSlab) * C::SLAB) >> 4) + 2 * (kk % kPerSlab);
                umma_ss(t_d, desc64(hi, a_lo + at), desc64(hi, b_lo + at), idesc_s, kk > 0);
            }
        };
        // D += A B, A the 16-bit pairs over a softmax warp's half of t_a's columns, B a chunk
        auto gather = [&](uint32_t t_d, uint32_t t_a, uint32_t b_lo, uint32_t accumulate) {
#pragma unroll
            for (int kk = 0; kk < kRows / 16; ++kk)
                umma_ts(t_d, t_a + (kk / 4) * 64 + (kk % 4) * 8, desc64(hi, b_lo + ((kk * 16 * C::ROWB) >> 4)), idesc_o,
                        accumulate | (kk > 0));
        };
        Ring rs, ro;                          // places of the chunks that S and the outputs are at
        uint32_t no = 0, it = 0;
        // what the elected lane issues
        auto scores = [&]() {
            product(tmem_base + C::TMEM_S, k_lo + it % NKV * (C::BYTES >> 4), q_lo0 + rs.at * (C::BYTES >> 4));
            umma_commit(s_full);
        };
        auto grads = [&](bool last) {
            product(tmem_base + C::TMEM_DP, v_lo + it % NKV * (C::BYTES >> 4), g_lo0 + rs.at * (C::BYTES >> 4));
            umma_commit(dp_full);
            if (last) umma_commit(kv_empty + it % NKV);
        };
        auto chunk_wait = [&]() {
            mbar_wait(qd_full + rs.at, rs.phase, wctx, kErrLoadWait);
            mbar_wait(x_full + rs.at, rs.phase, wctx, kErrLoadWait);
        };
        for (KeyWalk<LINE> walk(g, cut, before); walk.more(cut);) {
            const KeyItem k = walk.get(g, cut, before);
            walk.next(k);
            if (k.n == 0) continue;
            mbar_wait(kv_full + it % NKV, (it / NKV) & 1, wctx, kErrLoadWait);
            chunk_wait();
            tc_fence_after();
            if (elect_one()) {
                scores();
                grads(k.n == 1);
            }
            __syncwarp();
            rs.next(NST);
            for (int i = 0; i < k.n; ++i, ++no) {
                const bool more = i + 1 < k.n;
                if (i == 0) mbar_wait(acc_free, (it & 1) ^ 1, wctx, kErrMmaWait);
                if (more) chunk_wait();      // (of the next one, ahead of what holds this one up)
                if (lane == 0) NA2D_TR(2, 0, no);
                mbar_wait(p_full, no & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if (lane == 0) NA2D_TR(2, 1, no);
                if (elect_one()) {
                    gather(tmem_base + C::TMEM_DV, tmem_base + C::TMEM_S, gm_lo0 + ro.at * (C::BYTES >> 4), i > 0);
                    if (more) scores();
                }
                __syncwarp();
                if (lane == 0) NA2D_TR(2, 3, no);
                mbar_wait(ds_full, no & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if (lane == 0) NA2D_TR(2, 4, no);
                if (elect_one()) {
                    gather(tmem_base + C::TMEM_DK, tmem_base + C::TMEM_DP, qm_lo0 + ro.at * (C::BYTES >> 4), i > 0);
                    gather(tmem_base + C::TMEM_DK, tmem_base + C::TMEM_DP + 32, qm_lo0 + ro.at * (C::BYTES >> 4), 1);
                    umma_commit(qd_empty + ro.at);
                    if (more) grads(i + 2 == k.n);
                    else umma_commit(acc_full);
                }
                __syncwarp();
                if (more) rs.next(NST);
                ro.next(NST);
                if (lane == 0) NA2D_TR(2, 5, no);
            }
            ++it;
        }
    } else if (warp == 10) {
        reg_dec<kDkvRegsCtl>();
    } else if (warp >= 12) {
        // ------------------------------------------------------------------ epilogue warps
        reg_dec<kDkvRegsEpi>();
        const int quarter = warp & 3;
        const uint32_t tmem_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        uint8_t* stage = sOut + quarter * 2 * OutStage<32>::BYTES;
        uint32_t it = 0, seq = 0;
        for (KeyWalk<LINE> walk(g, cut, before); walk.more(cut);) {
            const KeyItem k = walk.get(g, cut, before);
            walk.next(k);
            const int first = k.k0 + quarter * 32, key = first + lane;
            const bool there = k.n > 0 && key < k.count;     // else no query sees the tile, or the key is none (its weights of 0 meet any dO and Q)
            const float scale_dk = g.scale * exp2i(-unit_shift<DT>(g, bounds, k));
            if (k.n > 0) {
                mbar_wait(acc_full, it & 1, wctx, kErrMmaWait);
                tc_fence_after();
            }
#pragma unroll
            for (int j = 0; j < 2 * (D / 32); ++j) {
                const int which = j / (D / 32), r = j % (D / 32);        // dV, then dK
                const float scale = which ? scale_dk : Weight<DT>::kUnit;
                uint32_t v[32];
                if (k.n > 0) {
                    tmem_ld_32x32(tmem_lane + (which ? C::TMEM_DK : C::TMEM_DV) + 32 * r, v);
                    tmem_ld_wait();
                    if (j + 1 == 2 * (D / 32)) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(acc_free);
                    }
                }
                if (!there) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = 0u;
                }
                if (32 * r >= g.C || first >= g.Tk) continue;
                if (LINE ? k.split < 0 : cut.splits == 1) {
                    na2d_tc::stage_and_store<DT, 32, 2>(which ? &tm_dk : &tm_dv, stage, v, scale, 32 * r, first, k.m, k.b, 0, lane, &seq);
                } else if (key < g.Tk) {
                    const size_t at = LINE ? static_cast<size_t>(k.split) * kRows + quarter * 32 + lane
                                               : (static_cast<size_t>(k.split) * g.units + static_cast<size_t>(k.b) * g.Nk + k.m) * g.Tk + key;
                    float4* dst = reinterpret_cast<float4*>((which ? cut.part_dk : cut.part_dv) + at * g.C + 32 * r);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (32 * r + 4 * e < g.C)
                            dst[e] = make_float4(__uint_as_float(v[4 * e]) * scale, __uint_as_float(v[4 * e + 1]) * scale,
                                                 __uint_as_float(v[4 * e + 2]) * scale, __uint_as_float(v[4 * e + 3]) * scale);
                }
            }
            if (k.n > 0) ++it;
        }
        if (lane == 0) bulk_wait<0>();
    } else {
        // ------------------------------------------------------------------ softmax warps
        reg_inc<kDkvRegsSoftmax>();
        const int quarter = warp & 3, half = warp >> 2;
        const int row = quarter * 32 + lane;                 // key of the tile = tensor-memory lane
        const uint32_t tmem_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t s_addr = tmem_lane + C::TMEM_S + 64 * half, dp_addr = tmem_lane + C::TMEM_DP + 64 * half;
        const uint64_t scale2 = pair2(g.sl2, g.sl2);
        uint32_t m = 0;
        Ring ring;
        for (KeyWalk<LINE> walk(g, cut, before); walk.more(cut);) {
            const KeyItem k = walk.get(g, cut, before);
            walk.next(k);
            const int key = k.k0 + row;
            // the first token that sees this key
            const int t_lo = key >= k.count ? 0x7fffffff : g.causal ? max(key + g.Tq - k.count, 0) : 0;
            int h0, t0;
            k.start(g, h0, t0);
            for (int i = 0; i < k.n; ++i, ++m, k.step(g, h0, t0)) {
                const int closed = key >= k.count ? 64 : t_lo - t0 - 64 * half;     // columns of this half that do not see the key come first
                const bool cover = __any_sync(0xffffffffu, closed > 0);
                const float* x_lse = s_x + ring.at * 2 * kRows + 64 * half;
                const float* x_delta = x_lse + kRows;
                uint64_t pr[32];
                if ((tid & 127) == 0) NA2D_TR(half ? 0 : 3, 0, m);
                mbar_wait(s_full, m & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if ((tid & 127) == 0) NA2D_TR(half ? 0 : 3, 1, m);
                uint32_t s[2][32];
                tmem_ld_32x32(s_addr, s[0]);
                tmem_ld_32x32(s_addr + 32, s[1]);
                tmem_ld_wait();
#pragma unroll
                for (int e4 = 0; e4 < 16; ++e4) {
                    const ulonglong2 nl = *reinterpret_cast<const ulonglong2*>(x_lse + 4 * e4);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int e = 4 * e4 + 2 * h;
                        const uint64_t y = fma2(pair2(s[e / 32][e % 32], s[e / 32][e % 32 + 1]), scale2, h ? nl.y : nl.x);
                        pr[e / 2] = pair2(fast_exp2(lo2(y)), fast_exp2(hi2(y)));
                    }
                }
                if (cover) {                                 // by selection: what is not seen may hold anything
#pragma unroll
                    for (int e = 0; e < 64; e += 2)
                        pr[e / 2] = pair2(e < closed ? 0.f : lo2(pr[e / 2]), e + 1 < closed ? 0.f : hi2(pr[e / 2]));
                }
                uint32_t w[2][16];
#pragma unroll
                for (int e2 = 0; e2 < 32; ++e2) w[e2 / 16][e2 % 16] = pack2<DT>(lo2(pr[e2]), hi2(pr[e2]));
                tmem_st_32x16(s_addr, w[0]);                 // over columns that this warp has read
                tmem_st_32x16(s_addr + 16, w[1]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full);
                if ((tid & 127) == 0) NA2D_TR(half ? 0 : 3, 2, m);
                mbar_wait(dp_full, m & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if ((tid & 127) == 0) NA2D_TR(half ? 0 : 3, 3, m);
                tmem_ld_32x32(dp_addr, s[0]);
                tmem_ld_32x32(dp_addr + 32, s[1]);
                tmem_ld_wait();
                const uint64_t unit2 = reinterpret_cast<const uint64_t*>(s_x + NST * 2 * kRows)[ring.at];
#pragma unroll
                for (int e4 = 0; e4 < 16; ++e4) {
                    const ulonglong2 nd = *reinterpret_cast<const ulonglong2*>(x_delta + 4 * e4);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int e = 4 * e4 + 2 * h;
                        const uint64_t dp = pair2(s[e / 32][e % 32], s[e / 32][e % 32 + 1]);
                        pr[e / 2] = mul2(pr[e / 2], IsBf16<DT>::value ? add2(dp, h ? nd.y : nd.x) : fma2(dp, unit2, h ? nd.y : nd.x));
                    }
                }
                if (cover) {
#pragma unroll
                    for (int e = 0; e < 64; e += 2)
                        pr[e / 2] = pair2(e < closed ? 0.f : lo2(pr[e / 2]), e + 1 < closed ? 0.f : hi2(pr[e / 2]));
                }
#pragma unroll
                for (int e2 = 0; e2 < 32; ++e2) w[e2 / 16][e2 % 16] = pack2<DT>(lo2(pr[e2]), hi2(pr[e2]));
                tmem_st_32x16(dp_addr, w[0]);
                tmem_st_32x16(dp_addr + 16, w[1]);
#pragma unroll
                for (int e2 = 0; e2 < 32; ++e2) w[e2 / 16][e2 % 16] = pack_rest<DT>(pr[e2], w[e2 / 16][e2 % 16]);
                tmem_st_32x16(dp_addr + 32, w[0]);           // (dP's other columns, read, too)
                tmem_st_32x16(dp_addr + 48, w[1]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ds_full);
                if ((tid & 127) == 0) NA2D_TR(half ? 0 : 3, 4, m);
                ring.next(NST);
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

// Adds the parts of dK and dV: `elements` of each part, 4 a thread.
template <typename DT>
__global__ void __launch_bounds__(256)
attn_sum_kernel(const float* __restrict__ part_dk, const float* __restrict__ part_dv, DT* __restrict__ dk, DT* __restrict__ dv,
                const long long elements, const int splits) {
    after_previous_grid();
    next_grid_may_start();
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= elements) return;
    const float* src = (blockIdx.y ? part_dv : part_dk) + i;
    float4 acc = *reinterpret_cast<const float4*>(src);
#pragma unroll 4
    for (int s = 1; s < splits; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(src + s * elements);
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
    }
    *reinterpret_cast<uint2*>((blockIdx.y ? dv : dk) + i) = make_uint2(pack2<DT>(acc.x, acc.y), pack2<DT>(acc.z, acc.w));
}

// Line: a block joins the parts of an eighth of one tile of keys, or writes zeros where the tile holds none.
template <typename DT>
__global__ void __launch_bounds__(256)
attn_join_kernel(const float* __restrict__ part_dk, const float* __restrict__ part_dv, DT* __restrict__ dk, DT* __restrict__ dv,
                 const Geom g, const KeyCut cut) {
    after_previous_grid();
    next_grid_may_start();
    int tile, m, before = 0, all = 0;                    // tiles of one key head of the entries before b, and of all
    const int unit = cut.by_key_tiles.split(blockIdx.x, tile), b = g.by_nk.split(unit, m), lane = threadIdx.x & 31;
    for (int i = lane; i < g.B; i += 32) {
        const int tiles = (key_count(g, i) + kRows - 1) / kRows;
        all += tiles;
        if (i < b) before += tiles;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, d);
        before += __shfl_xor_sync(0xffffffffu, before, d);
    }
    const int tiles = (key_count(g, b) + kRows - 1) / kRows, each = (all * g.Nk * g.tiles + cut.line - 1) / cut.line;
    const int at = (before * g.Nk + m * tiles + tile) * g.tiles;
    const int lo = tile < tiles ? at / each : 0, hi = tile < tiles ? (at + g.tiles - 1) / each : 0;      // CTAs that have some of it
    if (tile < tiles && lo == hi) return;                // one had them all
    const int vectors = g.C / 4, first = blockIdx.z * kJoinRows, rows = min(first + kJoinRows, min(kRows, g.Tk - tile * kRows));
    const float* part = blockIdx.y ? part_dv : part_dk;
    DT* dst = (blockIdx.y ? dv : dk) + (static_cast<size_t>(unit) * g.Tk + static_cast<size_t>(tile) * kRows) * g.C;
    for (int i = first * vectors + threadIdx.x; i < rows * vectors; i += 256) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (tile < tiles) {
#pragma unroll 4
            for (int s = lo; s <= hi; ++s) {             // lo has the tile's first chunk
                const float4 v = *reinterpret_cast<const float4*>(part + (2 * s + (s == lo)) * static_cast<size_t>(kRows) * g.C + 4 * i);
                acc.x += v.x;
                acc.y += v.y;
                acc.z += v.z;
                acc.w += v.w;
            }
        }
        *reinterpret_cast<uint2*>(dst + 4 * i) = make_uint2(pack2<DT>(acc.x, acc.y), pack2<DT>(acc.z, acc.w));
    }
}

template <typename DT, int D>
int launch_dkdv(const Place& at, const Geom& g, const KeyCut& cut, const Operand& q, const Operand& k, const Operand& v, const Operand& d_o,
                const float* lse, const float* delta, const Bounds& bounds, const Operand& d_k, const Operand& d_v) {
    using C = KeyCfg<D>;
    CUtensorMap tq, tg, tk, tv, tdk, tdv;
    int rc = operand_map(&tq, q, at.dtype, g.B, g.N, g.Tq, g.C, g.tt, g.hp, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&tg, d_o, at.dtype, g.B, g.N, g.Tq, g.C, g.tt, g.hp, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&tk, k, at.dtype, g.B, g.Nk, g.Tk, g.C, kRows, 1, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&tv, v, at.dtype, g.B, g.Nk, g.Tk, g.C, kRows, 1, C::SLAB_C);
    if (rc == NA2D_OK) rc = operand_map(&tdk, d_k, at.dtype, g.B, g.Nk, g.Tk, g.C, 32, 1, 32);
    if (rc == NA2D_OK) rc = operand_map(&tdv, d_v, at.dtype, g.B, g.Nk, g.Tk, g.C, 32, 1, 32);
    if (rc != NA2D_OK) return rc;
    auto kern = cut.line ? attn_dkdv_kernel<DT, D, true> : attn_dkdv_kernel<DT, D, false>;
    static std::atomic<unsigned long long> opted[2]{};
    if (na2d_tc::opt_in_smem(kern, C::SMEM, at.device, opted[cut.line > 0]) != cudaSuccess) return NA2D_ERR_CUDA;
    const int sms = na2d_tc::sm_count(at.device);
    *at.launched += 1;
    if (na2d_launch::launch(true, kern, cut.line ? cut.line : cut.items < sms ? cut.items : sms, 512, C::SMEM, at.st, tq, tg, tk, tv, tdk, tdv,
                            lse, delta, bounds, at.errors, g, cut) != cudaSuccess)
        return NA2D_ERR_CUDA;
    if (cut.line) {
        *at.launched += 1;
        return na2d_launch::launch(true, attn_join_kernel<DT>, dim3((unsigned)(g.units * cut.key_tiles), 2, kJoinBlocks), 256, 0, at.st,
                                   (const float*)cut.part_dk, (const float*)cut.part_dv, (DT*)d_k.ptr, (DT*)d_v.ptr, g, cut) == cudaSuccess
                   ? NA2D_OK
                   : NA2D_ERR_CUDA;
    }
    if (cut.splits == 1) return NA2D_OK;
    const long long elements = (long long)g.units * g.Tk * g.C;
    *at.launched += 1;
    return na2d_launch::launch(true, attn_sum_kernel<DT>, dim3((unsigned)((elements / 4 + 255) / 256), 2), 256, 0, at.st,
                               (const float*)cut.part_dk, (const float*)cut.part_dv, (DT*)d_k.ptr, (DT*)d_v.ptr, elements,
                               cut.splits) == cudaSuccess
               ? NA2D_OK
               : NA2D_ERR_CUDA;
}

}  // namespace na2d_attn
