// Translation unit of the tcgen05 kernels of attention over all keys for one 16-bit element type
// (-DNA2D_TC_DT=1: bf16, 2: fp16).
#include "na2d_attn_entry.h"
#include "na2d_delta.cuh"
#include "na2d_attn_fwd.cuh"
#include "na2d_attn_dq.cuh"
#include "na2d_attn_dkdv.cuh"

namespace na2d_attn {

#if NA2D_TC_DT == 1
#define NA2D_TC_TYPE __nv_bfloat16
#define NA2D_TC_NAME(base) base##_bf16
#elif NA2D_TC_DT == 2
#define NA2D_TC_TYPE __half
#define NA2D_TC_NAME(base) base##_f16
#else
#error "compile with -DNA2D_TC_DT=1 (bf16) or 2 (fp16)"
#endif

namespace {

// f(head dim rounded up to one that kernels are built for)
template <typename F>
int by_head_dim(int C, F&& f) {
    if (C <= 32) return f(std::integral_constant<int, 32>{});
    if (C <= 64) return f(std::integral_constant<int, 64>{});
    return f(std::integral_constant<int, 128>{});
}

}  // namespace

int NA2D_TC_NAME(forward)(const Place& at, const Geom& g, const Parts& parts, const Operand& q, const Operand& k, const Operand& v,
                          const Operand& o, float* lse) {
    FwdCut cut{parts.count, (g.tiles + 1) / 2, 0, Div(parts.count), Div((g.tiles + 1) / 2), parts.a, parts.b};
    const long long items = g.tiles > 1 ? (long long)g.units * cut.pairs * cut.splits : ((long long)g.units * cut.splits + 1) / 2;
    if (items > 0x3fffffffLL) return NA2D_ERR_TOO_LARGE;
    cut.items = (int)items;
    return by_head_dim(g.C, [&](auto d) { return launch_fwd<NA2D_TC_TYPE, decltype(d)::value>(at, g, cut, q, k, v, o, lse); });
}

int NA2D_TC_NAME(backward)(const Place& at, const Geom& g, const Parts& parts, const Backward& x) {
    int rc = launch_delta<NA2D_TC_TYPE>(at, g, x.d_o, x.o, x.delta);
    if (rc != NA2D_OK) return rc;
    return by_head_dim(g.C, [&](auto d) {
        constexpr int D = decltype(d)::value;
        int rc = NA2D_OK;
        if (x.d_q.ptr) rc = launch_dq<NA2D_TC_TYPE, D>(at, g, x.q, x.k, x.v, x.d_o, x.lse, x.delta, x.d_q);
        if (rc != NA2D_OK || !x.d_k.ptr) return rc;
        Geom gk = g;
        if (g.causal) cut_rows(gk, false);               // a chunk's masks go by the column alone
        const int key_tiles = (g.Tk + kRows - 1) / kRows;
        KeyCut cut{key_tiles, parts.count, 0, Div(parts.count), Div(key_tiles), parts.a, parts.b};
        const long long items = (long long)gk.units * cut.key_tiles * cut.splits;
        if (items > 0x3fffffffLL) return (int)NA2D_ERR_TOO_LARGE;
        cut.items = (int)items;
        return launch_dkdv<NA2D_TC_TYPE, D>(at, gk, cut, x.q, x.k, x.v, x.d_o, x.lse, x.delta, x.d_k, x.d_v);
    });
}

#if NA2D_TC_DT == 1
// Parts of the keys in the forward: where the tiles are fewer than the groups that the SMs have (two a CTA), so many that each group has
// about eight, since lengths that differ make parts that differ; of at least 4 chunks each.
int forward_parts(const Geom& g, int sms) {
    const long long tiles = (long long)g.units * g.tiles;
    const int chunks = (g.Tk + kRows - 1) / kRows;
    if (tiles >= 2 * sms) return 1;
    const long long want = (16LL * sms + tiles - 1) / tiles;
    return (int)std::max(1LL, std::min<long long>(want, chunks / 4));
}

// Parts of the queries in the key half, by the same rule with one tile a CTA, and fewer: a part costs its sums' way through memory.
int key_parts(const Geom& g, int sms) {
    const long long tiles = (long long)g.units * ((g.Tk + kRows - 1) / kRows);
    if (tiles >= sms) return 1;
    const long long want = (4LL * sms + tiles - 1) / tiles;
    return (int)std::max(1LL, std::min<long long>(want, g.tiles / 4));
}
#endif

}  // namespace na2d_attn

#ifdef NA2D_TRACE
// Development aid: the trace that CTA 0 of this unit's kernels recorded (see na2d_tc.cuh).
extern "C" int NA2D_TC_NAME(na2d_debug_trace_attn)(unsigned long long* out, int max_entries) {
    return na2d_tc::copy_trace(out, max_entries);
}
#endif
