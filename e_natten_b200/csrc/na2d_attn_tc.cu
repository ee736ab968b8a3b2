// Translation unit of the tcgen05 kernels of attention over all keys for one 16-bit element type
// (-DNA2D_TC_DT=1: bf16, 2: fp16).
#include "na2d_attn_entry.h"
#include "na2d_delta.cuh"
#include "na2d_attn_fwd.cuh"
#include "na2d_attn_few.cuh"
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

// Whether the chunks of all units go on one line: units of one tile, fewer than the groups of the SMs (two a CTA).  The line against units as
// items, bf16, 128 channels, lengths from none to the largest: 16 x 4 caches of up to 32768 keys with 4 heads each 98 us for 683, with 40 rows
// (16 x 4 of up to 8192) 65 for 176; 36 x 8 caches of up to 8192, one head each, 117 for 189.  With more units the 128-row kernel has items
// enough (64 x 8 of up to 4096, 40 rows: 146 us, 204 on the line).  The kernel for few rows would win there, too, where caches are long
// (32 x 16 of up to 8192: 188 for 273) and lose where they are short (64 x 8 of up to 512: 48 for 34): it has the bound of the other.
bool on_line(const Geom& g, int sms) { return g.tiles == 1 && g.units < 2 * sms && g.B <= kLineEntries && g.Tk > kRows; }

// Whether the kernel for few rows takes them.
bool few_rows(const Geom& g) { return g.G * g.Tq <= kFewRows; }

// Takers of the line: CTAs, or their groups (two a CTA); fewer where that would leave them less than 2 chunks each.
int line_groups(const Geom& g, int sms) {
    const long long chunks = (long long)g.units * ((g.Tk + kRows - 1) / kRows);
    if (few_rows(g)) return (int)std::max(1LL, std::min((long long)sms, (chunks + 1) / 2));
    return 2 * (int)std::max(1LL, std::min((long long)sms, (chunks + 3) / 4));
}

// Parts of the keys in the forward of units of several tiles: where the tiles are fewer than the groups, so many that each group has about
// four, since where lengths differ many of them are empty; of at least 4 chunks each.  In parts and whole, bf16, 128 channels, 8 heads: 512
// rows on 16384 keys 86 us for 266, 1024 rows 141 for 298; 4 heads x 2048, causal, 38 for 44.  Near the bound the whole tiles, one round of
// nearly all SMs, would be faster: 2 x 8 heads x 2048 rows on 8192 keys 240 for 158, 8 heads x 4096, causal, 121 for 80.
int forward_parts(const Geom& g, int sms) {
    const long long tiles = (long long)g.units * g.tiles;
    const int chunks = (g.Tk + kRows - 1) / kRows;
    if (g.tiles == 1 || tiles >= 2 * sms) return 1;
    return (int)std::max(1LL, std::min<long long>((8LL * sms + tiles - 1) / tiles, chunks / 4));
}

// CTAs that share the line of the key half's chunks, at least 4 chunks each; 0 where every tile is a CTA's item.  By items a CTA has a
// whole number of tiles, and with lengths some of them are empty; the line costs its parts' way through memory.  Line and items, bf16,
// backward of the key half: 4 x 4 heads x 4096 x 128 290 us for 309, 8 x 4 x 3136 x 4 rows on 333 keys of 64 161 for 205, with lengths 117
// for 213; lengths of up to 1024 keys of 64, 8 x 16 heads: 2048 rows 176 for 191, 1024 rows 116 for 106, 512 rows 77 for 63 (not on the line).
int key_line(const Geom& g, int sms) {
    const long long tiles = (long long)g.units * ((g.Tk + kRows - 1) / kRows), chunks = tiles * g.tiles;
    if (g.causal || g.B > kLineEntries || chunks + sms > 0x7fffffffLL) return 0;
    const bool pays = g.lengths ? g.tiles >= 8 : (tiles + sms - 1) / sms * g.tiles > (chunks + sms - 1) / sms + 4;
    return pays ? (int)std::max(1LL, std::min<long long>(sms, chunks / 4)) : 0;
}

// The same for the query half, whose tiles are of rows and whose chunks of keys: 4 x 4 heads x 4096 x 128 238 us for 275, 2 x 4 heads x 512 rows
// on 8192 keys 51 for 123; where whole rounds of items do as well, 4 x 4 x 3136 x 8 rows on 333 keys of 64, 190 for 139 (not on the line).
int row_line(const Geom& g, int sms) {
    const long long tiles = (long long)g.units * g.tiles, each = (g.Tk + kRows - 1) / kRows, chunks = tiles * each;
    if (g.causal || g.B > kLineEntries || chunks + sms > 0x7fffffffLL) return 0;
    const bool pays = (tiles + sms - 1) / sms * each > (chunks + sms - 1) / sms + 4;
    return pays ? (int)std::max(1LL, std::min<long long>(sms, chunks / 4)) : 0;
}

// Parts of the queries in the key half of causal calls, where tiles are fewer than CTAs: a part costs its sums' way through memory.  In parts
// and whole, bf16, 128 channels: 2 x 4 heads on one key head x 4096 181 us for 270, 2 heads x 4096 71 for 77; 8 heads x 2048 79 for 52, which
// whole tiles would do better; 8 heads x 4096, more tiles than CTAs, 111 whole for 146.
int key_parts(const Geom& g, int sms) {
    const long long tiles = (long long)g.units * ((g.Tk + kRows - 1) / kRows);
    if (!g.causal || tiles >= sms) return 1;
    return (int)std::max(1LL, std::min<long long>((4LL * sms + tiles - 1) / tiles, g.tiles / 4));
}

size_t line_rows(const Geom& g, int sms) { return (size_t)(line_groups(g, sms) + g.units) * g.G * g.Tq; }
size_t all_rows(const Geom& g) { return (size_t)g.B * g.N * g.Tq; }
size_t key_part(const Geom& g) { return (size_t)g.units * g.Tk * g.C; }
size_t row_part(const Geom& g, int line) { return (size_t)line * 2 * kRows * g.C; }             // 2 a CTA
size_t bound_units(const Geom& g) { return ((size_t)g.units * 2 + 3) / 4 * 4; }                 // floats, in whole 16 bytes
size_t bound_floats(const Geom& g) { return bound_units(g) + (all_rows(g) + 3) / 4 * 4; }
size_t line_part(const Geom& g, int line) { return (size_t)line * 2 * 2 * kRows * g.C; }        // of dK and dV, 2 a CTA

}  // namespace

int NA2D_TC_NAME(forward)(const Place& at, const Geom& g, const Scratch& scratch, const Operand& q, const Operand& k, const Operand& v,
                          const Operand& o, float* lse) {
    const int sms = na2d_tc::sm_count(at.device);
    FwdCut cut{};
    cut.pairs = (g.tiles + 1) / 2;
    if (on_line(g, sms) && scratch.floats >= line_rows(g, sms) * (g.C + 1)) {
        cut.line = line_groups(g, sms);
        cut.part_o = scratch.at;
        cut.part_lse = scratch.at + line_rows(g, sms) * g.C;
    }
    cut.splits = (int)std::min<size_t>(forward_parts(g, sms), std::max<size_t>(1, scratch.floats / (all_rows(g) * (g.C + 1))));
    if (cut.splits > 1) {
        cut.part_o = scratch.at;
        cut.part_lse = scratch.at + cut.splits * all_rows(g) * g.C;
    }
    const int chunks = (g.Tk + kRows - 1) / kRows;
    cut.each = (chunks + cut.splits - 1) / cut.splits;
    cut.by_splits = Div(cut.splits);
    cut.by_pairs = Div(cut.pairs);
    const long long items = g.tiles > 1 ? (long long)g.units * cut.pairs * cut.splits : ((long long)g.units + 1) / 2;
    if (items > 0x3fffffffLL) return NA2D_ERR_TOO_LARGE;
    cut.items = (int)items;
    return by_head_dim(g.C, [&](auto d) {
        return cut.line && few_rows(g) ? launch_few<NA2D_TC_TYPE, decltype(d)::value>(at, g, cut, q, k, v, o, lse)
                                       : launch_fwd<NA2D_TC_TYPE, decltype(d)::value>(at, g, cut, q, k, v, o, lse);
    });
}

int NA2D_TC_NAME(backward)(const Place& at, const Geom& g, const Scratch& given, const Backward& x) {
    // fp16's bounds come first in the workspace; without one they lie in the stream's memory pool for the time of the call
    struct Own {
        float* at = nullptr;
        cudaStream_t st;
        ~Own() {
            if (at) cudaFreeAsync(at, st);
        }
    } own;
    own.st = at.st;
    Bounds bounds{};
    Scratch scratch = given;
    if (!IsBf16<NA2D_TC_TYPE>::value) {
        if (given.floats >= bound_floats(g)) {
            bounds.unit = given.at;
            scratch = Scratch{given.at + bound_floats(g), given.floats - bound_floats(g)};
        } else {
            if (cudaMallocAsync(reinterpret_cast<void**>(&own.at), bound_floats(g) * sizeof(float), at.st) != cudaSuccess) return NA2D_ERR_CUDA;
            bounds.unit = own.at;
        }
        bounds.row = bounds.unit + bound_units(g);
    }
    int rc = launch_delta<NA2D_TC_TYPE>(at, g, x.d_o, x.o, x.v, x.delta, bounds);
    if (rc != NA2D_OK) return rc;
    return by_head_dim(g.C, [&](auto d) {
        constexpr int D = decltype(d)::value;
        int rc = NA2D_OK;
        const int sms = na2d_tc::sm_count(at.device), rows = row_line(g, sms);
        RowCut row_cut{};
        if (rows && scratch.floats >= row_part(g, rows)) {
            row_cut.line = rows;
            row_cut.part = scratch.at;
        }
        if (x.d_q.ptr) rc = launch_dq<NA2D_TC_TYPE, D>(at, g, row_cut, x.q, x.k, x.v, x.d_o, x.lse, x.delta, bounds, x.d_q);
        if (rc != NA2D_OK || !x.d_k.ptr) return rc;
        Geom gk = g;
        if (g.causal) cut_rows(gk, false);               // a chunk's masks go by the column alone
        KeyCut cut{};
        cut.key_tiles = (g.Tk + kRows - 1) / kRows;
        const int line = key_line(g, sms);
        if (line && scratch.floats >= line_part(g, line)) cut.line = line;
        cut.splits = (int)std::min<size_t>(key_parts(g, sms), std::max<size_t>(1, scratch.floats / (2 * key_part(g))));
        cut.each = (gk.tiles + cut.splits - 1) / cut.splits;
        cut.by_splits = Div(cut.splits);
        cut.by_key_tiles = Div(cut.key_tiles);
        if (cut.line || cut.splits > 1) {
            cut.part_dk = scratch.at;
            cut.part_dv = scratch.at + (cut.line ? line_part(g, cut.line) / 2 : cut.splits * key_part(g));
        }
        const long long items = (long long)gk.units * cut.key_tiles * cut.splits;
        if (items > 0x3fffffffLL) return (int)NA2D_ERR_TOO_LARGE;
        cut.items = (int)items;
        return launch_dkdv<NA2D_TC_TYPE, D>(at, gk, cut, x.q, x.k, x.v, x.d_o, x.lse, x.delta, bounds, x.d_k, x.d_v);
    });
}

#if NA2D_TC_DT == 1
size_t forward_floats(const Geom& g, int sms) {
    if (on_line(g, sms)) return line_rows(g, sms) * (g.C + 1);
    const int parts = forward_parts(g, sms);
    return parts > 1 ? parts * all_rows(g) * (g.C + 1) : 0;
}
size_t backward_floats(const Geom& g, int sms, bool f16, bool d_q, bool d_k) {       // the halves' one after the other
    const size_t bounds = f16 ? bound_floats(g) : 0;
    size_t floats = d_q ? row_part(g, row_line(g, sms)) : 0;
    if (!d_k) return bounds + floats;
    if (const int line = key_line(g, sms)) return bounds + std::max(floats, line_part(g, line));
    const int parts = key_parts(g, sms);
    return bounds + std::max(floats, parts > 1 ? 2 * parts * key_part(g) : 0);
}
#endif

}  // namespace na2d_attn

#ifdef NA2D_TRACE
// Development aid: the trace that CTA 0 of this unit's kernels recorded (see na2d_tc.cuh).
extern "C" int NA2D_TC_NAME(na2d_debug_trace_attn)(unsigned long long* out, int max_entries) {
    return na2d_tc::copy_trace(out, max_entries);
}
#endif
