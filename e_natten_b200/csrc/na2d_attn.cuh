// Attention over all keys (no window): the geometry that its kernels and launchers share.
//
//   s_ij = scale q_i . k_j over the keys that row i sees,   p_i = softmax(s_i),   o_i = sum_j p_ij v_j
//
// Operands are (B, heads, T, C); N query heads, Nk key heads, each shared by G = N / Nk query heads.  Batch entry b has
// lengths[b] keys (all Tk without lengths); with `causal`, row i of Tq sees the first lengths[b] - Tq + 1 + i of them: the queries are
// the last ones of the keys' sequence.  A row that sees nothing has o = 0, lse = -infinity and gradients of 0.
//
// A unit is one (batch entry, key head).  Its query rows, of all heads that share the key head, are cut into tiles of up to 128 rows:
// 128 tokens of one head, or, where there are few tokens, hp heads with all their tt tokens (row h * tt + t), so that keys and
// values are read once for all of them.  hp divides G: no tile holds rows of another unit.
#pragma once

#include "na2d_tc.cuh"

namespace na2d_attn {

constexpr int kRows = 128;      // rows of a tile of queries or keys

// Division of 0 <= x < 2^31 by a number that the host knows, as a multiplication: every role of a kernel works out where its tiles lie, and
// with divisions (in 64 bits for the parts) a tile began 2500 cycles late.
struct Div {
    unsigned d, m, s;
    Div() = default;
    explicit Div(int by) : d((unsigned)by), m(0), s(0) {
        while ((1ull << s) < d) ++s;
        m = (unsigned)((((1ull << s) - d) << 32) / d + 1);
    }
#ifdef __CUDACC__
    __device__ __forceinline__ int quotient(int x) const { return (int)((__umulhi((unsigned)x, m) + (unsigned)x) >> s); }
    __device__ __forceinline__ int split(int x, int& rest) const {
        const int q = quotient(x);
        rest = x - q * (int)d;
        return q;
    }
#endif
};

struct Geom {
    int B, N, Nk, G, Tq, Tk, C;
    int units;                              // B * Nk
    int hp, tt;                             // heads and tokens of a query tile
    int tiles_t, groups, tiles;             // query tiles of a unit: along the tokens, (groups of) heads, in all
    int causal;
    const int* lengths;                     // (B,) on the device, or null
    float scale, sl2;                       // the softmax scale, and times log2(e)
    Div by_nk, by_tt, by_tiles_t, by_tiles, by_units;
    int parts = 0;                          // forward, units of several tiles: parts of each unit's keys, all of the same length; 0: by a rule
    bool joint = false;                     // rows see other keys, too: o and lse are over all of them
};

// Rows in tiles (host); several heads in one only with `pack`.
inline void cut_rows(Geom& g, bool pack = true) {
    g.G = g.N / g.Nk;
    g.units = g.B * g.Nk;
    g.hp = 1;
    for (int h = 2; pack && h <= g.G && (long long)h * g.Tq <= kRows; ++h)
        if (g.G % h == 0) g.hp = h;
    g.tt = g.Tq < kRows ? g.Tq : kRows;
    g.tiles_t = g.hp > 1 ? 1 : (g.Tq + kRows - 1) / kRows;
    g.groups = g.G / g.hp;
    g.tiles = g.tiles_t * g.groups;
    g.by_nk = Div(g.Nk);
    g.by_tt = Div(g.tt);
    g.by_tiles_t = Div(g.tiles_t);
    g.by_tiles = Div(g.tiles);
    g.by_units = Div(g.units);
}

#ifdef __CUDACC__

__device__ __forceinline__ int key_count(const Geom& g, int b) { return g.lengths ? min(max(__ldg(g.lengths + b), 0), g.Tk) : g.Tk; }
// Keys that token t sees, of the `count` of its batch entry.
__device__ __forceinline__ int keys_seen(const Geom& g, int count, int t) {
    return g.causal ? max(count - g.Tq + 1 + t, 0) : count;
}

// One tile of query rows.
struct RowTile {
    int b, m;               // batch entry, key head
    int h0, t0;             // its first head and token
    int count;              // keys of the batch entry
    __device__ __forceinline__ RowTile() {}
    __device__ __forceinline__ RowTile(const Geom& g, int unit, int tile) {
        b = g.by_nk.split(unit, m);
        int ti;
        const int th = g.by_tiles_t.split(tile, ti);
        t0 = ti * kRows;
        h0 = m * g.G + th * g.hp;
        count = key_count(g, b);
    }
    // keys that its last token sees: those that any of its rows sees
    __device__ __forceinline__ int keys(const Geom& g) const { return keys_seen(g, count, min(t0 + g.tt, g.Tq) - 1); }
    // head and token of a row; false where the tile has no such row
    __device__ __forceinline__ bool row(const Geom& g, int r, int& n, int& t) const {
        const int h = g.hp == 1 ? 0 : g.by_tt.quotient(r);
        n = h0 + h;
        t = t0 + r - h * g.tt;
        return h < g.hp && t < g.Tq;
    }
};

// Index of a row in (B, N, Tq).
__device__ __forceinline__ size_t row_index(const Geom& g, int b, int n, int t) {
    return (static_cast<size_t>(b) * g.N + n) * g.Tq + t;
}

// An operand tile of 128 rows in shared memory, in slabs of up to 64 channels as the tensor maps' swizzle lays them.  D is the head
// dim rounded up to 32, 64 or 128: TMA fills the channels beyond C with zeros.
template <int D>
struct TileCfg {
    static constexpr int NS = (D + 63) / 64, SLAB_C = D < 64 ? D : 64, ROWB = SLAB_C * 2;
    static constexpr uint32_t SWZ = ROWB == 128 ? 2u : 4u;
    static constexpr int ATOM = 8 * ROWB, SLAB = kRows * ROWB, BYTES = NS * SLAB;
    // bytes that a copy of `rows` rows brings
    static __device__ __forceinline__ uint32_t load_bytes(int rows) { return (uint32_t)(NS * rows * ROWB); }
};

// Zeros in rows [first, 128) of a tile, by one warp: keys that a batch entry does not have may hold anything, and as contraction rows
// they meet weights of zero.
template <int D>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int first, int lane) {
    using T = TileCfg<D>;
    const int pieces = (kRows - first) * (T::ROWB / 16);
#pragma unroll
    for (int s = 0; s < T::NS; ++s) {
        const uint32_t at = na2d_ptx::smem_u32(tile) + s * T::SLAB + first * T::ROWB;
        for (int i = lane; i < pieces; i += 32) na2d_tc::st_shared_v4(at + 16 * i, 0u, 0u, 0u, 0u);
    }
    na2d_ptx::fence_proxy_async();
    __syncwarp();
}

#endif

// fp16: what bounds |dO . V| and |delta|, from which the backward takes the power of two that its dS go into their products with (ds_shift).
struct Bounds {
    float* unit;            // (units, 2): the largest squared norms of the dO rows that see keys and of V's rows
    float* row;             // (B, N, Tq): the squared norm of a dO row
    float* delta;           // joint rows: (units,): the largest square of the delta of rows that see keys; else null
};

#ifdef __CUDACC__
// s so that |dS| 2^s stays below 2^15, given the squared norms of dO and V: |dP| and |delta| are at most the norms' product.  (Of joint rows
// |delta| is not, o being of other values, too: they give the square of delta.)  dS and the rest that rounding leaves of it are then within fp16's 2^-24 of a largest value near its end, whatever the size of gradients
// (unshifted, weights of 2^-14 times gradients of 1e-2 were half lost, and dS beyond 65504 infinite).
__device__ __forceinline__ int ds_shift(float d_o_square, float v_square, float delta_square = 0.f) {
    const float square = fmaxf(d_o_square * v_square, delta_square);         // 2^-96 to 2^78 for numbers of fp16
    if (!(square > 0.f) || square == CUDART_INF_F) return 0;
    const int e = (__float_as_int(square) >> 23) - 127;      // square < 2^(e + 1)
    return 14 - ((e + 2) >> 1);
}
// x^2, or 0 where that is infinite or no number: what such a delta gives is no number whatever the shift.
__device__ __forceinline__ float finite_square(float x) { return x * x < CUDART_INF_F ? x * x : 0.f; }
__device__ __forceinline__ float exp2i(int s) { return __int_as_float((s + 127) << 23); }      // |s| < 127
#endif

// What a launcher gets: geometry, element type, place, error state, launch counter.
struct Place {
    int dtype, device;
    cudaStream_t st;
    const na2d_ptx::ErrorState* errors;
    int* launched;
};

// A (B, heads, T, C) operand: element strides, channels contiguous.
struct Operand {
    void* ptr;
    long long b, n, t;
    bool wide = false;      // a result in fp32, dense, whatever the operands' type: a sum that others join
};

// Tensor map with coordinates (channel, token, head, batch, 0) and boxes of box_t tokens of box_n heads.
inline int operand_map(CUtensorMap* map, const Operand& x, int dtype, int B, int heads, int T, int C, int box_t, int box_n, int box_c) {
    return na2d_tc::make_map(map, na2d_tc::TensorArg{x.ptr, Na2dStride{x.b, x.b, x.n, x.t}}, dtype, 1, B, heads, T, C, box_t, box_n, box_c);
}

}  // namespace na2d_attn
