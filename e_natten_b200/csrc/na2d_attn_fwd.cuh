// Attention over all keys, forward, on tcgen05 (bf16 / fp16, head dims up to 128).
//
// Persistent, one CTA per SM, two tiles of 128 query rows in flight: group a (softmax warps 0-3, issuer warp 9) has one, group b (warps 4-7,
// issuer 11) the other, each with an S / P buffer and an output accumulator of its own in tensor memory.  Keys are walked in chunks of
// 128; on the tensor pipe a group's P V(c) S(c + 1) run under the other group's exponentials.  PAIR: the two tiles are neighbours of
// one unit and share every chunk of K and V in shared memory; else (units of a single tile) each has its own.
//
// Few rows and many keys: the keys of a row are taken in parts, whose o (fp32) and lse go to a workspace and are joined by
// attn_combine_kernel.  Units of several tiles: `splits` parts of each, every one an item.  Units of one tile (single tokens on caches): all
// units' chunks lie on one line, of which every group takes the same length, wherever units begin and end; with parts of a unit for
// items, caches of different lengths left some CTAs 1.4 times the mean's work (16 x 4 caches of up to 32768 keys: 141 us).
//
// P goes into its product rounded once to 16 bits, as tensor memory and the pipe take it: o is 1.3 to 1.4 times as far from its 64-bit value as
// its own rounding puts it (bf16 2.3e-3 for 1.7e-3, fp16 2.9e-4 for 2.1e-4), the two roundings' sum of squares.  A second number, as the
// backward's dS has, would be a third product to these two.  Sums and maxima are of the weights in 32 bits.
//
// Bound by the chain S - maximum - exponentials - P V of a group, of which the other group's covers all but about 700 of 3700 cycles a pair of
// chunks; the special-function unit is at 60 % (a polynomial for a quarter of the exponentials: 179 us for 155).  8 heads x 16384 x 128,
// causal, bf16: 620-643 us, 870 TFLOP/s; 4 x 4 heads x 4096 x 128: 156 us.
//
//   warps 0-7   softmax: a thread owns a row, reads its 128 scores, writes P over S as packed 16-bit pairs;
//   warp 8      producer of Q, K and V;    warps 9, 11  MMA issue, one a group: a warp that served both in turn had 3000 cycles of
//               bookkeeping and waits a chunk, three times the MMAs' (4 x 4 x 4096 x 128: 198 us);
//   warp 10     clears the rows of V beyond a batch entry's keys;
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
#ifdef NA2D_TRACE
using na2d_tc::trace;
#endif

// How the work is cut: items of two tiles (or two parts of tiles).
struct FwdCut {
    int splits;
    int pairs;              // PAIR: items of a unit and split
    int items;
    int each;               // chunks of a part
    int line;               // not PAIR: the chunks of all units on one line, that many groups take; 0: not
    Div by_splits, by_pairs;
    float* part_o;          // (splits, B, N, Tq, C), where splits > 1; line: (groups + units, rows of a unit, C)
    float* part_lse;        // (splits, B, N, Tq); line: (groups + units, rows of a unit)
};

// One group's half of an item: chunks [c0, c0 + n) of a tile.
struct FwdPart {
    RowTile tile;
    bool any;               // there is a tile
    int slot, c0, n;        // slot: the part's place in the workspace
};

// Batch entries on the line, at most (units are fewer than the groups where it is used).
constexpr int kLineEntries = 1024;
// before[b]: chunks of one key head of the entries before b; of all of them at before[B].  Written by one warp.
__device__ __forceinline__ void line_table(const Geom& g, int* before, int lane) {
    int sum = 0;
    for (int b0 = 0; b0 < g.B; b0 += 32) {
        int n = b0 + lane < g.B ? (key_count(g, b0 + lane) + kRows - 1) / kRows : 0;
        const int own = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, n, d);
            if (lane >= d) n += up;
        }
        if (b0 + lane < g.B) before[b0 + lane] = sum + n - own;
        sum += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) before[g.B] = sum;
}
// A group's stretch [at, end) of the line, and the unit that `at` lies in.
struct Stretch {
    int at, end, b, m;
    __device__ __forceinline__ void start(const Geom& g, const int* before, int group, int groups) {
        const int all = before[g.B] * g.Nk, each = (all + groups - 1) / max(groups, 1);
        at = min(group * each, all);
        end = min(at + each, all);
        if (at >= end) return;
        int lo = 0, hi = g.B;                            // before[lo] <= at's < before[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (before[mid] * g.Nk <= at) lo = mid;
            else hi = mid;
        }
        b = lo;
        m = (at - before[b] * g.Nk) / (before[b + 1] - before[b]);
    }
    __device__ __forceinline__ bool any() const { return at < end; }
    __device__ __forceinline__ int length(const int* before) const { return before[b + 1] - before[b]; }       // of the unit
    __device__ __forceinline__ int first(const Geom& g, const int* before) const { return before[b] * g.Nk + m * length(before); }
    // to the next unit
    __device__ __forceinline__ void next(const Geom& g, const int* before) {
        at = min(end, first(g, before) + length(before));
        if (at < end && ++m == g.Nk) {
            m = 0;
            do ++b;
            while (length(before) == 0);                 // (at < end: there is one)
        }
    }
};

// The items of a CTA, which every role walks by itself.
template <bool PAIR>
struct FwdWalk {
    int item;
    Stretch s[2];
    __device__ __forceinline__ FwdWalk(const Geom& g, const FwdCut& cut, const int* before) : item(blockIdx.x) {
        if constexpr (!PAIR) {
            if (cut.line) {
                s[0].start(g, before, 2 * blockIdx.x, 2 * gridDim.x);
                s[1].start(g, before, 2 * blockIdx.x + 1, 2 * gridDim.x);
            }
        }
    }
    __device__ __forceinline__ bool more(const FwdCut& cut) const {
        if constexpr (!PAIR)
            if (cut.line) return s[0].any() || s[1].any();
        return item < cut.items;
    }
    __device__ __forceinline__ void next(const Geom& g, const FwdCut& cut, const int* before) {
        item += gridDim.x;
        if constexpr (!PAIR) {
            if (cut.line) {
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    if (s[x].any()) s[x].next(g, before);
            }
        }
    }
    __device__ __forceinline__ void parts(const Geom& g, const FwdCut& cut, const int* before, FwdPart (&p)[2]) const {
        if constexpr (PAIR) {
            int split, pair, unit;
            const int rest = cut.by_splits.split(item, split);
            if (g.causal) {     // the later tiles are the longer ones: they go first, so that no CTA is left with one at the end
                pair = cut.pairs - 1 - g.by_units.split(rest, unit);
            } else {
                unit = cut.by_pairs.split(rest, pair);
            }
            int chunks[2], most = 0;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                p[x].any = 2 * pair + x < g.tiles;
                p[x].tile = RowTile(g, unit, p[x].any ? 2 * pair + x : 2 * pair);
                chunks[x] = p[x].any ? (p[x].tile.keys(g) + kRows - 1) / kRows : 0;
                most = max(most, chunks[x]);
            }
            const int c0 = min(split * cut.each, most), c1 = min(c0 + cut.each, most);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                p[x].slot = split;
                p[x].c0 = c0;
                p[x].n = max(min(chunks[x], c1) - c0, 0);
            }
        } else if (cut.line) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                p[x].any = s[x].any();
                const int unit = p[x].any ? s[x].b * g.Nk + s[x].m : 0;
                p[x].tile = RowTile(g, unit, 0);
                p[x].slot = 2 * blockIdx.x + x + unit;   // from part to part either the group or the unit is one more
                const int first = p[x].any ? s[x].first(g, before) : 0;
                p[x].c0 = p[x].any ? s[x].at - first : 0;
                p[x].n = p[x].any ? min(s[x].end, first + s[x].length(before)) - s[x].at : 0;
            }
        } else {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int unit = 2 * item + x;
                p[x].any = unit < g.units;
                p[x].tile = RowTile(g, p[x].any ? unit : 0, 0);
                p[x].slot = p[x].c0 = 0;
                p[x].n = p[x].any ? (p[x].tile.keys(g) + kRows - 1) / kRows : 0;
            }
        }
    }
};

// The part's chunk that holds keys beyond its batch entry's (and not beyond Tk, where TMA fills with zeros), or -1.
__device__ __forceinline__ int fwd_ragged_chunk(const Geom& g, int count, int c0, int n) {
    const int at = count / kRows - c0;
    return count % kRows != 0 && count < g.Tk && at >= 0 && at < n ? at : -1;
}

template <int D>
struct FwdCfg : TileCfg<D> {
    using T = TileCfg<D>;
    static constexpr int NST = D == 128 ? 2 : 4;                         // chunks of K, and of V
    static constexpr int NQ = D == 128 ? 1 : 2;                          // Q tiles of a group
    static constexpr int OUT_BYTES = 4 * 2 * OutStage<32>::BYTES;        // two staging buffers for each epilogue warp
    static constexpr int X_BYTES = 2 * 2 * 2 * kRows * 4;                // row sum, final maximum [group][tile parity][row]
    static constexpr int LINE_BYTES = (kLineEntries + 1) * 4;
    static constexpr int SMEM = 2 * NQ * T::BYTES + 2 * NST * T::BYTES + OUT_BYTES + X_BYTES + 512 /*barriers*/ + LINE_BYTES + 1024 /*alignment*/;
    static constexpr int TMEM_S = 0, TMEM_O = 256;                       // of group x: S + 128 x, O + D x
    static_assert(SMEM <= kSmemLimit && NST <= 8, "forward kernel shared memory");
};

// Logarithm (base 2) by which a row's maximum may grow before its sums are rescaled: the weights stay below 2^8, within fp16 by far,
// and most chunks after the first rescale nothing.
constexpr float kGrow = 8.f;
// Weights go into their sums and products times 2^kLift: fp16 ends at 2^-24, and 2^17 keys whose weights rounded to nothing, or to twice what they
// are, beside one of large weight were a result off by hundredths.  kGrow + kLift stays within its 2^16.
template <typename DT> constexpr float kLift = IsBf16<DT>::value ? 0.f : 7.f;

// What rounding a pair to `w` left of it, rounded itself: the two together have 16 (22) bits.
template <typename DT>
__device__ __forceinline__ uint32_t pack_rest(uint64_t pair, uint32_t w) {
    uint64_t had;
    if constexpr (IsBf16<DT>::value) {
        had = na2d_ptx::pair2(w << 16, w & 0xffff0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        had = na2d_ptx::pair2(f.x, f.y);
    }
    const uint64_t rest = na2d_ptx::fma2(had, na2d_ptx::pair2(-1.f, -1.f), pair);
    return pack2<DT>(na2d_ptx::lo2(rest), na2d_ptx::hi2(rest));
}

// Columns of P whose product starts ahead of the others (64: 166 us for 156).
constexpr int kMost = 96;

template <typename DT, int D, bool PAIR>
__global__ void __launch_bounds__(512, 1)
attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o, DT* __restrict__ o_rows,
                const Operand o_st, float* __restrict__ lse, const ErrorState* __restrict__ errors, const Geom g, const FwdCut cut) {
    using C = FwdCfg<D>;
    constexpr int NST = C::NST, NQ = C::NQ;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;                                   // [group][NQ] Q tiles
    uint8_t* sK = sQ + 2 * NQ * C::BYTES;               // NST x K chunk
    uint8_t* sV = sK + NST * C::BYTES;                    // NST x V chunk
    uint8_t* sOut = sV + NST * C::BYTES;                  // output staging
    float* x_sum = reinterpret_cast<float*>(sOut + C::OUT_BYTES);     // [group][tile parity][row]
    float* x_fin = x_sum + 4 * kRows;
    uint64_t* bars = reinterpret_cast<uint64_t*>(x_fin + 4 * kRows);
    uint64_t* q_full = bars;                 // [2][2] TMA -> MMA, per group and buffer
    uint64_t* q_empty = bars + 4;            // [2][2] MMA (commit) -> TMA
    uint64_t* o_full = bars + 8;             // [2] MMA (commit) -> epilogue
    uint64_t* o_free = bars + 10;            // [2] epilogue -> MMA
    uint64_t* s_full = bars + 52;            // [2] MMA (commit) -> softmax
    uint64_t* p_full = bars + 54;            // [2] softmax -> MMA
    uint64_t* p_most = bars + 56;            // [2] softmax -> MMA: the first kMost columns of P
    uint64_t* k_full = bars + 12;            // [8] TMA -> MMA
    uint64_t* v_full = bars + 20;            // [8] TMA -> MMA
    uint64_t* k_empty = bars + 28;           // [8] MMA (commit) -> TMA
    uint64_t* v_empty = bars + 36;           // [8] MMA (commit) -> TMA
    uint64_t* v_clear = bars + 44;           // [8] warp 10 -> MMA: rows beyond the keys are zeros
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 58);
    const WaitCtx wctx{reinterpret_cast<WaitState*>(bars + 59)};
    int* before = reinterpret_cast<int*>(bars + 64);      // the line's table

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        wait_state_init(wctx.st, errors, kWaitLimitNs);
        for (int i = 0; i < 2; ++i) {
            mbar_init(o_full + i, 1);
            mbar_init(o_free + i, 4);
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 4);
            mbar_init(p_most + i, 4);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(q_full + i, 1);
            mbar_init(q_empty + i, 1);
        }
        for (int i = 0; i < NST; ++i) {
            mbar_init(k_full + i, 1);
            mbar_init(k_empty + i, PAIR ? 2 : 1);        // a pair's chunks are read by both groups
            mbar_init(v_full + i, 1);
            mbar_init(v_empty + i, PAIR ? 2 : 1);
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
    if (!PAIR && warp == 1 && cut.line) line_table(g, before, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    next_grid_may_start();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 8) {
        // ------------------------------------------------------------------ producer
        // K is a chunk ahead of V: the buffers come free in that order (on the pipe P V(c - 2), S(c - 1), P V(c - 1), S(c)).
        reg_dec<kDkvRegsCtl>();
        if (lane == 0) {
            LoadTracker lt(bars);
            Ring rk, rv;
            uint32_t it[2] = {0, 0};
            auto load = [&](const FwdPart& p, int c, bool values) {
                const int key = (p.c0 + c) * kRows;
                // (the tensor map is named in each call: a map chosen through a run-time pointer may be copied to local memory, where
                // TMA cannot read it)
                if (!values) {
                    if (!lt.acquire(k_empty + rk.at, rk.phase ^ 1, wctx)) return;
                    lt.arm(k_full + rk.at, rk.phase, C::BYTES);
#pragma unroll
                    for (int s = 0; s < C::NS; ++s)
                        tma_load_5d(sK + rk.at * C::BYTES + s * C::SLAB, &tm_k, k_full + rk.at, s * 64, key, p.tile.m, p.tile.b, 0);
                    rk.next(NST);
                } else {
                    if (!lt.acquire(v_empty + rv.at, rv.phase ^ 1, wctx)) return;
                    lt.arm(v_full + rv.at, rv.phase, C::BYTES);
#pragma unroll
                    for (int s = 0; s < C::NS; ++s)
                        tma_load_5d(sV + rv.at * C::BYTES + s * C::SLAB, &tm_v, v_full + rv.at, s * 64, key, p.tile.m, p.tile.b, 0);
                    rv.next(NST);
                }
            };
            for (FwdWalk<PAIR> walk(g, cut, before); walk.more(cut) && lt.ok; walk.next(g, cut, before)) {
                FwdPart p[2];
                walk.parts(g, cut, before, p);
                const int most = max(p[0].n, p[1].n);
                for (int c = 0; c <= most && lt.ok; ++c) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (c == 0 && p[x].n > 0) {
                            const uint32_t to = 2 * x + it[x] % NQ, phase = (it[x] / NQ) & 1;
                            if (!lt.acquire(q_empty + to, phase ^ 1, wctx)) break;
                            lt.arm(q_full + to, phase, C::load_bytes(g.hp * g.tt));
#pragma unroll
                            for (int s = 0; s < C::NS; ++s)
                                tma_load_5d(sQ + (x * NQ + it[x] % NQ) * C::BYTES + s * C::SLAB, &tm_q, q_full + to, s * 64, p[x].tile.t0,
                                            p[x].tile.h0, p[x].tile.b, 0);
                            ++it[x];
                        }
                        if (PAIR ? x == 0 && c < most : c < p[x].n) load(p[x], c, false);    // (a pair has its unit and first chunk in common)
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        if (c > 0 && lt.ok && (PAIR ? x == 0 : c <= p[x].n)) load(p[x], c - 1, true);
                }
            }
            lt.drain(wctx);
        }
    } else if (warp == 10) {
        // ------------------------------------------------------------------ zeros beyond the keys
        reg_dec<kDkvRegsCtl>();
        if (g.lengths) {
            Ring ring;
            for (FwdWalk<PAIR> walk(g, cut, before); walk.more(cut); walk.next(g, cut, before)) {
                FwdPart p[2];
                walk.parts(g, cut, before, p);
                const int most = max(p[0].n, p[1].n);
                const int at[2] = {fwd_ragged_chunk(g, p[0].tile.count, p[0].c0, PAIR ? most : p[0].n),
                                   PAIR ? -1 : fwd_ragged_chunk(g, p[1].tile.count, p[1].c0, p[1].n)};
                for (int c = 0; c < most; ++c) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (PAIR ? x == 1 : c >= p[x].n) continue;
                        mbar_wait(v_full + ring.at, ring.phase, wctx, kErrLoadWait);
                        __syncwarp();
                        if (c == at[x]) clear_rows<D>(sV + ring.at * C::BYTES, p[x].tile.count % kRows, lane);
                        if (lane == 0) mbar_arrive(v_clear + ring.at);
                        ring.next(NST);
                    }
                }
            }
        }
    } else if (warp == 9 || warp == 11) {
        // ------------------------------------------------------------------ MMA issue of a group
        // (the whole warp walks the loop so that addresses stay warp-uniform; one lane issues)
        reg_dec<kDkvRegsCtl>();
        constexpr uint32_t idesc_s = umma_idesc(kRows, kRows, IsBf16<DT>::value, IsBf16<DT>::value, false, false);
        constexpr uint32_t idesc_o = umma_idesc(kRows, D, IsBf16<DT>::value, IsBf16<DT>::value, false, true);
        constexpr uint32_t hi = smem_desc_hi(C::ATOM, C::SWZ);
        const int x = warp == 11;
        const uint32_t q_lo0 = smem_desc_lo(smem_u32(sQ) + x * NQ * C::BYTES, 16), k_lo0 = smem_desc_lo(smem_u32(sK), 16);
        const uint32_t v_lo0 = smem_desc_lo(smem_u32(sV), C::SLAB);
        const uint32_t t_s = tmem_base + C::TMEM_S + x * kRows, t_o = tmem_base + C::TMEM_O + x * D;
        // Loads of the item that come before the group's chunk c.
        struct Item {
            int n, other;                    // chunks of the group, and of the other one
            __device__ __forceinline__ Item(const Geom& g, const FwdCut& cut, const int* before, const FwdWalk<PAIR>& walk, int x) {
                n = other = 0;
                if (!walk.more(cut)) return;
                FwdPart p[2];
                walk.parts(g, cut, before, p);
                n = x ? p[1].n : p[0].n;
                other = x ? p[0].n : p[1].n;
            }
            __device__ __forceinline__ uint32_t loads() const { return PAIR ? max(n, other) : n + other; }
            __device__ __forceinline__ uint32_t ahead(int c, int x) const { return PAIR ? c : c + min(c + x, other); }
        };
        uint32_t base = 0, chunks = 0, tiles = 0;        // loads, this group's chunks and tiles so far
        // (by the elected lane, K there)
        auto scores = [&](const Item& t, int c) {
            const uint32_t at = (base + t.ahead(c, x)) % NST, q_lo = q_lo0 + tiles % NQ * (C::BYTES >> 4), k_lo = k_lo0 + at * (C::BYTES >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                constexpr int kPerSlab = C::SLAB_C / 16;
                const int slab = kk / kPerSlab, in = 2 * (kk % kPerSlab);
                umma_ss(t_s, desc64(hi, q_lo + ((slab * C::SLAB) >> 4) + in), desc64(hi, k_lo + ((slab * C::SLAB) >> 4) + in), idesc_s, kk > 0);
            }
            umma_commit(s_full + x);                                          // and P V of the group's chunk before
            umma_commit(k_empty + at);
            if (c + 1 == t.n) umma_commit(q_empty + 2 * x + tiles % NQ);
        };
        auto key_wait = [&](const Item& t, int c) {
            mbar_wait(k_full + (base + t.ahead(c, x)) % NST, ((base + t.ahead(c, x)) / NST) & 1, wctx, kErrLoadWait);
        };
        FwdWalk<PAIR> walk(g, cut, before);
        Item t(g, cut, before, walk, x);
        while (walk.more(cut)) {
            if (t.n > 0) {
                mbar_wait(q_full + 2 * x + tiles % NQ, (tiles / NQ) & 1, wctx, kErrLoadWait);
                key_wait(t, 0);
                tc_fence_after();
                if (elect_one()) scores(t, 0);
                __syncwarp();
            }
            walk.next(g, cut, before);
            const Item next(g, cut, before, walk, x);
            for (int c = 0; c < t.n; ++c, ++chunks) {
                const uint32_t at = (base + t.ahead(c, x)) % NST, phase = ((base + t.ahead(c, x)) / NST) & 1;
                if (c == 0) mbar_wait(o_free + x, (tiles & 1) ^ 1, wctx, kErrMmaWait);      // the tile before has been read out
                mbar_wait(v_full + at, phase, wctx, kErrLoadWait);
                if (g.lengths) mbar_wait(v_clear + at, phase, wctx, kErrOther);
                const bool more = c + 1 < t.n;
                if (more) key_wait(t, c + 1);            // (its load does not wait for this chunk's P V)
                if (lane == 0) NA2D_TR(1 + x, 0, chunks);
                const uint32_t v_lo = v_lo0 + at * (C::BYTES >> 4);
                auto product = [&](int from, int to) {
#pragma unroll
                    for (int kk = from; kk < to; ++kk)
                        umma_ts(t_o, t_s + 8 * kk, desc64(hi, v_lo + ((kk * 16 * C::ROWB) >> 4)), idesc_o, (c > 0) || (kk > 0));
                };
                mbar_wait(p_most + x, chunks & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if (elect_one()) product(0, kMost / 16);
                __syncwarp();
                mbar_wait(p_full + x, chunks & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if (lane == 0) NA2D_TR(1 + x, 1, chunks);
                if (elect_one()) {
                    product(kMost / 16, kRows / 16);
                    umma_commit(v_empty + at);
                    if (!more) umma_commit(o_full + x);
                    else scores(t, c + 1);               // into the buffer that P V has just read: a thread's MMAs run in their order
                    NA2D_TR(1 + x, 2, chunks);
                }
                __syncwarp();
            }
            // chunks that only the pair's other tile has: their buffers wait for both groups
            for (int c = t.n; PAIR && c < t.other; ++c) {
                const uint32_t at = (base + c) % NST, phase = ((base + c) / NST) & 1;
                mbar_wait(k_full + at, phase, wctx, kErrLoadWait);
                if (lane == 0) mbar_arrive(k_empty + at);
                mbar_wait(v_full + at, phase, wctx, kErrLoadWait);
                if (lane == 0) mbar_arrive(v_empty + at);
                __syncwarp();
            }
            base += t.loads();
            if (t.n > 0) ++tiles;
            t = next;
        }
    } else if (warp >= 12) {
        // ------------------------------------------------------------------ epilogue warps
        reg_dec<kDkvRegsEpi>();
        const int quarter = warp & 3;
        const int row = quarter * 32 + lane;                 // row of the tile = tensor-memory lane
        const uint32_t tmem_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        uint8_t* stage = sOut + quarter * 2 * OutStage<32>::BYTES;
        const bool in_parts = cut.splits > 1 || cut.line, by_tma = g.hp == 1 && !in_parts;
        const size_t part_rows = cut.line ? (size_t)g.G * g.Tq : static_cast<size_t>(g.B) * g.N * g.Tq;     // of the workspace
        uint32_t it[2] = {0, 0}, seq = 0;
        for (FwdWalk<PAIR> walk(g, cut, before); walk.more(cut); walk.next(g, cut, before)) {
            FwdPart p[2];
            walk.parts(g, cut, before, p);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (!p[x].any) continue;
                int n, t;
                const bool ok = p[x].tile.row(g, row, n, t);
                const size_t at = row_index(g, p[x].tile.b, n, t);
                const size_t part_at = p[x].slot * part_rows + (cut.line ? (size_t)(n - p[x].tile.m * g.G) * g.Tq + t : at);
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
                    } else if (ok && !in_parts) {
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
                        float4* dst = reinterpret_cast<float4*>(cut.part_o + part_at * g.C + 32 * j);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (32 * j + 4 * e < g.C)
                                dst[e] = make_float4(__uint_as_float(v[4 * e]) * inv, __uint_as_float(v[4 * e + 1]) * inv,
                                                     __uint_as_float(v[4 * e + 2]) * inv, __uint_as_float(v[4 * e + 3]) * inv);
                    }
                }
                if (ok) {
                    float* to = in_parts ? cut.part_lse + part_at : lse + at;
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
        // The groups take turns at the exponentials: left to themselves they fall into step, both at them at half the rate and then both
        // waiting for their MMAs (4 x 4 x 4096 x 128: 4640 cycles a chunk of either).  Both go through the turns of an item's longer half.
        const uint32_t my_turn = 1 + group, other_turn = 2 - group;
        if (group) bar_arrive(other_turn, 256);              // a goes first
        for (FwdWalk<PAIR> walk(g, cut, before); walk.more(cut); walk.next(g, cut, before)) {
            FwdPart both[2];
            walk.parts(g, cut, before, both);
            const FwdPart p = group ? both[1] : both[0];
            const int turns = max(both[0].n, both[1].n);
            int n, t;
            const bool ok = p.tile.row(g, row, n, t);
            const bool idle = !__any_sync(0xffffffffu, ok);  // no row of this warp is one of the tile: nothing is read of what it writes
            const int seen = (ok ? keys_seen(g, p.tile.count, t) : 0) - p.c0 * kRows;      // keys of this row, from the part's first chunk on
            float run_max = -CUDART_INF_F, run_sum = 0.f;
            for (int c = 0; c < turns; ++c) {
                if (c >= p.n || idle) {
                    if (c < p.n) {
                        mbar_wait(s_full + group, m & 1, wctx, kErrMmaWait);
                        tc_fence_after();
                    }
                    bar_sync(my_turn, 256);
                    bar_arrive(other_turn, 256);
                    if (c < p.n) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(p_most + group);
                            mbar_arrive(p_full + group);
                        }
                        ++m;
                    }
                    continue;
                }
                if ((tid & 127) == 0) NA2D_TR(group ? 0 : 3, 0, m);
                mbar_wait(s_full + group, m & 1, wctx, kErrMmaWait);
                tc_fence_after();
                if ((tid & 127) == 0) NA2D_TR(group ? 0 : 3, 1, m);
                uint32_t s[4][32];
#pragma unroll
                for (int a = 0; a < 4; ++a) tmem_ld_32x32(s_addr + 32 * a, s[a]);
                tmem_ld_wait();
                const int open = seen - c * kRows;           // columns of this chunk that the row sees
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
                const float safe_max = (run_max == -CUDART_INF_F ? 0.f : run_max) - kLift<DT>;
                if ((tid & 127) == 0) NA2D_TR(group ? 0 : 3, 2, m);
                bar_sync(my_turn, 256);
                if ((tid & 127) == 0) NA2D_TR(group ? 0 : 3, 3, m);
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
                    if (32 * (a + 1) == kMost) {             // most of P V goes under the last exponentials
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_most + group);
                    }
                }
                bar_arrive(other_turn, 256);
                const uint64_t sum = add2(sum2[0], sum2[1]);
                run_sum += lo2(sum) + hi2(sum);
                if (c + 1 == p.n) {                          // for the epilogue warps, ahead of the arrival that lets the last P V go
                    x_sum[(group * 2 + (it & 1)) * kRows + row] = run_sum;
                    x_fin[(group * 2 + (it & 1)) * kRows + row] = safe_max;
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + group);
                if ((tid & 127) == 0) NA2D_TR(group ? 0 : 3, 5, m);
                ++m;
            }
            if (p.n > 0) ++it;
        }
        if (!group) bar_sync(my_turn, 256);                  // b's last arrival
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// Joins the parts of a row: lse = ln sum_s e^lse_s, o = sum_s e^(lse_s - lse) o_s.  A block a row: its four warps share the parts, 4 channels
// a lane.
template <typename DT>
__global__ void __launch_bounds__(128)
attn_combine_kernel(const float* __restrict__ part_o, const float* __restrict__ part_lse, DT* __restrict__ o, const Operand o_st,
                    float* __restrict__ lse, const Geom g, const int splits, const int line_groups) {
    __shared__ float4 sums[3][32];
    after_previous_grid();
    next_grid_may_start();
    const size_t row = blockIdx.x, bn = row / g.Tq;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int t = (int)(row % g.Tq), c = 4 * lane, b = (int)(bn / g.N), n = (int)(bn - (size_t)b * g.N);
    // the row's parts: places first, first + stride, ... of the workspace
    size_t first = row, stride = static_cast<size_t>(g.B) * g.N * g.Tq;
    int parts = splits;
    if (line_groups > 0) {
        int before = 0, all = 0;                         // chunks of one key head of the entries before b, and of all
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
        all *= g.Nk;
        const int m = n / g.G, each = max(1, (all + line_groups - 1) / line_groups);
        const int chunks = (key_count(g, b) + kRows - 1) / kRows, at = before * g.Nk + m * chunks;
        const int lo = at / each, hi = (at + chunks - 1) / each;         // groups that have some of them
        parts = chunks > 0 ? hi - lo + 1 : 0;
        stride = static_cast<size_t>(g.G) * g.Tq;
        first = (lo + b * g.Nk + m) * stride + static_cast<size_t>(n - m * g.G) * g.Tq + t;
    }
    float top = -CUDART_INF_F;
    for (int s = lane; s < parts; s += 32) top = fmaxf(top, part_lse[first + s * stride]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    // (a NaN of a part stays one: the maximum skips it, its weight does not)
    const float base = top == -CUDART_INF_F ? 0.f : top;
    float total = 0.f;
    for (int s = lane; s < parts; s += 32) total += expf(part_lse[first + s * stride] - base);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < g.C) {
#pragma unroll 4
        for (int s = warp; s < parts; s += 4) {
            const float part = part_lse[first + s * stride];
            if (part == -CUDART_INF_F) continue;             // nothing was written for it
            const float w = expf(part - base) * inv;
            const float4 v = *reinterpret_cast<const float4*>(part_o + (first + s * stride) * g.C + c);
            acc.x = fmaf(w, v.x, acc.x);
            acc.y = fmaf(w, v.y, acc.y);
            acc.z = fmaf(w, v.z, acc.z);
            acc.w = fmaf(w, v.w, acc.w);
        }
    }
    if (warp > 0) sums[warp - 1][lane] = acc;
    __syncthreads();
    if (warp > 0 || c >= g.C) return;
    for (int w = 0; w < 3; ++w) {
        acc.x += sums[w][lane].x;
        acc.y += sums[w][lane].y;
        acc.z += sums[w][lane].z;
        acc.w += sums[w][lane].w;
    }
    DT* dst = o + b * o_st.b + n * o_st.n + t * o_st.t;
    *reinterpret_cast<uint2*>(dst + c) = make_uint2(pack2<DT>(acc.x, acc.y), pack2<DT>(acc.z, acc.w));
    if (lane == 0) lse[row] = total == 0.f ? -CUDART_INF_F : base + logf(total);
}

template <typename DT>
int launch_combine(const Place& at, const Geom& g, const FwdCut& cut, const Operand& o, float* lse) {
    const long long rows = (long long)g.B * g.N * g.Tq;
    *at.launched += 1;
    return na2d_launch::launch(true, attn_combine_kernel<DT>, (unsigned)rows, 128, 0, at.st, (const float*)cut.part_o,
                               (const float*)cut.part_lse, (DT*)o.ptr, o, lse, g, cut.splits, cut.line) == cudaSuccess
               ? NA2D_OK
               : NA2D_ERR_CUDA;
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
    const int grid = cut.line ? cut.line / 2 : cut.items < sms ? cut.items : sms;
    if (na2d_launch::launch(false, kern, grid, 512, C::SMEM, at.st, tq, tk, tv, to, (DT*)o.ptr, o, lse,
                            at.errors, g, cut) != cudaSuccess)
        return NA2D_ERR_CUDA;
    return cut.splits == 1 && !cut.line ? NA2D_OK : launch_combine<DT>(at, g, cut, o, lse);
}

template <typename DT, int D>
int launch_fwd(const Place& at, const Geom& g, const FwdCut& cut, const Operand& q, const Operand& k, const Operand& v,
               const Operand& o, float* lse) {
    if (g.tiles > 1) return launch_fwd_as<DT, D, true>(at, g, cut, q, k, v, o, lse);
    return launch_fwd_as<DT, D, false>(at, g, cut, q, k, v, o, lse);
}

}  // namespace na2d_attn
