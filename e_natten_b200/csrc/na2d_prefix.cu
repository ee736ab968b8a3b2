// Attention over a prefix that several batch entries share, and each entry's own keys (include/na2d.h).
//
//   s_ij = scale q_i . k_j over the prefix's keys and the own keys that row i sees, one softmax over both:
//   o_i = sum_x e^(lse_x - lse) o_x,   lse = ln sum_x e^lse_x,   x in {prefix, own}
//
// The rows of all entries of a prefix are the rows of one attention problem, (S, N, A Tq, C) for S prefixes of A entries: the prefix's
// keys and values are read once for all of them, and its tiles of 128 rows are full where entries have few rows.  Own keys are another
// problem, (B, N, Tq, C).  Both run on the kernels of attention over all keys, with results in fp32, which are joined here.
// The backward forms the weights of both from the joint lse, so that each half's dQ is a summand, and dK and dV are final: the prefix's
// are sums over the rows of all its entries without atomics.  Few rows (serving) have a kernel of their own, na2d_prefix_tokens.cuh.
// The joins are bound by memory: 65536 rows of 128, 84 MB, 19 us each.
#include <algorithm>
#include <cmath>

#include "na2d_attn_entry.h"
#include "na2d_host.h"
#include "na2d_launch.h"
#include "na2d_prefix_entry.h"
#include "na2d_vec.cuh"

namespace {

using na2d_attn::Geom;
using na2d_attn::Operand;
using na2d_attn::Scratch;
using na2d_vec::narrow;
using na2d_vec::Vec;

constexpr int kThreads = 256;

// Rows of the whole batch: entry b = s A + a has prefix s.
struct Rows {
    int A, N, Tq, C;
    long long all;          // B N Tq, at most 2^31 - kThreads
    na2d_attn::Div by_a, by_n, by_tq;
};
struct Row {
    int b, n, t;
    long long by_prefix;    // its place in (S, N, A, Tq)
};
// Row `r` of (B, N, Tq).
__device__ __forceinline__ Row row_of(const Rows& g, int r) {
    Row x;
    x.b = g.by_n.split(g.by_tq.split(r, x.t), x.n);
    int a = 0, s = x.b;
    if (g.A > 1) s = g.by_a.split(x.b, a);
    x.by_prefix = (((long long)s * g.N + x.n) * g.A + a) * g.Tq + x.t;
    return x;
}
// The row and the piece of it, of `by.d`, that a thread has; a block has whole rows.
__device__ __forceinline__ bool piece_of(const Rows& g, const na2d_attn::Div& by, int& r, int& piece) {
    const int rows = kThreads / (int)by.d, own = by.split(threadIdx.x, piece);
    r = blockIdx.x * rows + own;
    return own < rows && r < g.all;
}
unsigned blocks_of(const Rows& g, int pieces) { return (unsigned)((g.all + kThreads / pieces - 1) / (kThreads / pieces)); }

// ---- rows in the prefixes' order ----------------------------------------------------------------------------------------
struct Gather {
    const void* from[3];    // (B, N, Tq, C), bytes
    long long b[3], n[3], t[3];
    void* to[3];            // (S, N, A Tq, C), dense
    const float* lse;       // null: none
    float* lse_to;
    int tensors;
    na2d_attn::Div by_pieces;           // of a row
};
template <typename V>
__global__ void __launch_bounds__(kThreads) gather_rows_kernel(const __grid_constant__ Rows g, const __grid_constant__ Gather x) {
    int r, c;
    const bool there = piece_of(g, x.by_pieces, r, c);
    const Row row = row_of(g, there ? r : 0);
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    if (!there) return;
    const int which = blockIdx.y;
    if (which == x.tensors) {
        if (c == 0) x.lse_to[row.by_prefix] = x.lse[r];
        return;
    }
    const char* from = static_cast<const char*>(x.from[which]) + row.b * x.b[which] + row.n * x.n[which] + row.t * x.t[which];
    reinterpret_cast<V*>(x.to[which])[row.by_prefix * (int)x.by_pieces.d + c] = __ldg(reinterpret_cast<const V*>(from) + c);
}

// ---- joins ----------------------------------------------------------------------------------------------------------------
// o and lse of a row from the prefix's and its own, either in parts of all rows; a thread has N channels.
template <typename DT, int N>
__global__ void __launch_bounds__(kThreads)
join_outputs_kernel(const __grid_constant__ Rows g, const na2d_attn::Div by_pieces, const float* __restrict__ o_prefix,
                    const float* __restrict__ lse_prefix, const float* __restrict__ o_own, const float* __restrict__ lse_own, const int prefix_parts,
                    const int own_parts, DT* __restrict__ o, float* __restrict__ lse) {
    int r, c;
    const bool there = piece_of(g, by_pieces, r, c);
    const Row row = row_of(g, there ? r : 0);
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    if (!there) return;
    const int parts = prefix_parts + own_parts;
    auto place = [&](int i) { return i < prefix_parts ? i * g.all + row.by_prefix : (i - prefix_parts) * g.all + r; };
    auto lse_of = [&](int i) { return (i < prefix_parts ? lse_prefix : lse_own)[place(i)]; };
    float top = lse_of(0);
    for (int i = 1; i < parts; ++i) top = fmaxf(top, lse_of(i));
    // (a NaN stays one: the maximum skips it, its weight does not)
    const float base = top == -CUDART_INF_F ? 0.f : top;
    float out[N], total = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) out[k] = 0.f;
#pragma unroll 2
    for (int i = 0; i < parts; ++i) {
        const float of = lse_of(i);
        if (of == -CUDART_INF_F) continue;               // of rows that see nothing, nothing was written
        Vec<float, N> v;
        v.load((i < prefix_parts ? o_prefix : o_own) + place(i) * g.C + c * N);
        const float w = expf(of - base);
        total += w;
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = fmaf(v.at[k], w, out[k]);
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int k = 0; k < N; ++k) out[k] *= inv;
    Vec<DT, N> to;
    to.round(out);
    to.store(o + (long long)r * g.C + c * N);
    if (c == 0) lse[r] = total == 0.f ? -CUDART_INF_F : base + logf(total);
}

// dq of a row: the sum of the prefix's parts and its own, in their order.
template <typename DT, int N>
__global__ void __launch_bounds__(kThreads)
join_gradients_kernel(const __grid_constant__ Rows g, const na2d_attn::Div by_pieces, const float* __restrict__ prefix, const float* __restrict__ own,
                      const int prefix_parts, const int own_parts, DT* __restrict__ d_q) {
    int r, c;
    const bool there = piece_of(g, by_pieces, r, c);
    const Row row = row_of(g, there ? r : 0);
    na2d_ptx::after_previous_grid();
    na2d_ptx::next_grid_may_start();
    if (!there) return;
    float out[N];
#pragma unroll
    for (int k = 0; k < N; ++k) out[k] = 0.f;
#pragma unroll 2
    for (int i = 0; i < prefix_parts + own_parts; ++i) {
        Vec<float, N> x;
        x.load((i < prefix_parts ? prefix + (i * g.all + row.by_prefix) * g.C : own + ((i - prefix_parts) * g.all + r) * g.C) + c * N);
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] += x.at[k];
    }
    Vec<DT, N> to;
    to.round(out);
    to.store(d_q + (long long)r * g.C + c * N);
}

// ---- the problem ------------------------------------------------------------------------------------------------------------
struct Problem {
    Rows rows;
    Geom prefix, own;       // own: unused without own keys
    bool any_own, tensor;
    bool heads_as_rows;     // CUDA cores, one token: the heads that share a key head are rows of one tile of own's
    int B, S, dtype;
    Operand q, k, v, pk, pv, o, d_o;       // as given
    bool follow[3];         // whether q's (o's, d_o's) rows of an entry follow those of the one before
};

// Parts of a prefix's keys where the tiles of rows, two an item, are at most half as many as the SMs: as many as make one round.  32 heads on 8
// key heads of 16384 keys, 64 answers of one token with 1 to 1024 own keys, the call: 70.8 us with one round, 79.7 with two, 95.8 with four, 78.9
// with attention's own rule; 16 heads on 4 of 30011 keys of 64, 24 answers of five tokens: 68.6, 62.5, 76.8, 79.3.
int even_parts(const Geom& g, int sms) {
    const long long items = (long long)g.units * ((g.tiles + 1) / 2);
    if (g.tiles == 1 || items > sms / 2) return 0;
    return (int)(sms / items);
}

int make_problem(const na2d_prefix_attention_args* a, Problem* p) {
    if (!a || a->struct_size < sizeof(na2d_prefix_attention_args)) return NA2D_ERR_BAD_ARG;
    if (a->B <= 0 || a->S <= 0 || a->N <= 0 || a->Nk <= 0 || a->Tq <= 0 || a->P <= 0 || a->Tk < 0 || a->C <= 0) return NA2D_ERR_BAD_ARG;
    if (a->B % a->S != 0 || a->N % a->Nk != 0) return NA2D_ERR_BAD_ARG;
    if (a->dtype != NA2D_F32 && a->dtype != NA2D_BF16 && a->dtype != NA2D_F16) return NA2D_ERR_UNSUPPORTED;
    if (a->path != NA2D_PATH_AUTO && a->path != NA2D_PATH_SIMT && a->path != NA2D_PATH_TENSOR) return NA2D_ERR_BAD_ARG;
    if (!(a->scale > 0.f) || !(a->scale < 3.0e38f)) return NA2D_ERR_BAD_ARG;
    const int A = a->B / a->S;
    if (a->Tk > (1 << 29) || a->P > (1 << 29) || (long long)A * a->Tq > (1 << 29) || (long long)a->B * a->N > (1 << 24)) return NA2D_ERR_TOO_LARGE;
    if (a->C > na2d_attn::kSimtMaxC) return NA2D_ERR_UNSUPPORTED;
    p->any_own = a->Tk > 0;
    p->B = a->B;
    p->S = a->S;
    p->dtype = a->dtype;
    p->rows = Rows{A, a->N, a->Tq, a->C, (long long)a->B * a->N * a->Tq, na2d_attn::Div(A), na2d_attn::Div(a->N), na2d_attn::Div(a->Tq)};
    if (p->rows.all > (1LL << 31) - kThreads) return NA2D_ERR_TOO_LARGE;         // (the last block's rows that are none are counted, too)
    auto geometry = [&](int B, int Tq, int Tk, bool causal, const int* lengths) {
        Geom g{};
        g.B = B; g.N = a->N; g.Nk = a->Nk; g.Tq = Tq; g.Tk = Tk; g.C = a->C;
        g.causal = causal;
        g.lengths = lengths;
        g.joint = a->Tk > 0;
        g.scale = a->scale;
        g.sl2 = a->scale * 1.4426950408889634f;
        na2d_attn::cut_rows(g);
        return g;
    };
    p->prefix = geometry(a->S, A * a->Tq, a->P, false, a->prefix_lengths);
    p->prefix.parts = even_parts(p->prefix, na2d_host::sm_count(a->device));
    if (p->any_own) p->own = geometry(a->B, a->Tq, a->Tk, a->causal != 0, a->key_lengths);
    auto operand = [&](const na2d_heads& x, int B, int heads, int T) {
        const na2d_host::HeadStrides s = na2d_host::head_strides(x, B, heads, T, a->C);
        return Operand{x.ptr, s.b, s.n, s.t};
    };
    p->q = operand(a->q, a->B, a->N, a->Tq);
    p->o = operand(a->o, a->B, a->N, a->Tq);
    p->d_o = operand(a->d_o, a->B, a->N, a->Tq);
    p->pk = operand(a->prefix_k, a->S, a->Nk, a->P);
    p->pv = operand(a->prefix_v, a->S, a->Nk, a->P);
    if (p->any_own) {
        p->k = operand(a->k, a->B, a->Nk, a->Tk);
        p->v = operand(a->v, a->B, a->Nk, a->Tk);
    }
    const Operand* by_rows[3] = {&p->q, &p->o, &p->d_o};
    for (int i = 0; i < 3; ++i) p->follow[i] = A == 1 || a->Tq == 1 || by_rows[i]->b == a->Tq * by_rows[i]->t;
    bool fits = a->dtype != NA2D_F32 && a->C <= 128 && a->C % 8 == 0;
    for (const Operand* x : {&p->q, &p->k, &p->v, &p->pk, &p->pv, &p->o, &p->d_o}) fits = fits && (!x->ptr || na2d_attn::tma_ready(*x));
    for (const na2d_heads* x : {&a->d_k, &a->d_v, &a->d_prefix_k, &a->d_prefix_v}) fits = fits && reinterpret_cast<uintptr_t>(x->ptr) % 16 == 0;      // (dense)
    if (a->path == NA2D_PATH_TENSOR && !fits) return NA2D_ERR_UNSUPPORTED;
    p->tensor = fits && a->path != NA2D_PATH_SIMT;
    p->heads_as_rows = p->any_own && !p->tensor && a->Tq == 1 && a->N > a->Nk;
    if (p->heads_as_rows) {                              // (the one token sees all own keys, causal or not)
        Geom& g = p->own;
        g.Tq = g.G;
        g.N = g.Nk;
        g.causal = 0;
        na2d_attn::cut_rows(g);
    }
    return NA2D_OK;
}

size_t esize_of(const Problem& p) { return p.dtype == NA2D_F32 ? 4 : 2; }

// Where things lie in the workspace, in bytes; every part on a 256-byte boundary.
struct Layout {
    size_t size = 0;
    size_t take(size_t bytes) {
        const size_t at = size;
        size += (bytes + 255) / 256 * 256;
        return at;
    }
};
// Which kind of keys goes on the line of few rows (na2d_prefix_tokens.cuh): its units' rows fit.  Where a prefix's do, its entries' own do.
struct OnLine {
    bool prefix, own;
    bool any() const { return prefix || own; }
};
OnLine on_line(const Problem& p) {
    const Rows& g = p.rows;
    const long long most = na2d_prefix::kTokenRows, own = (long long)p.prefix.G * g.Tq;
    const long long steps = (p.S * ((p.prefix.Tk + 15LL) / 16 + na2d_prefix::kUnitSteps) +
                             (p.any_own ? p.B * ((p.own.Tk + 15LL) / 16 + na2d_prefix::kUnitSteps) : 0)) * p.prefix.Nk;
    if (!p.tensor || (long long)p.S + p.B > na2d_prefix::kTokenEntries || steps > (1 << 30)) return {false, false};
    return {own * g.A <= most, p.any_own && own <= most};
}
// Rows of the parts of one side on the line: from part to part either the warp or the unit is one more.
size_t line_rows(const Geom& g, int sms) { return ((size_t)g.units + na2d_prefix::token_warps(sms)) * g.G * g.Tq; }

// Steps that a warp of the line takes, at least, where units are few: a third of the root of a unit's.  A unit's parts are then thrice as many as
// a part has steps: the joins take as long as the parts.  One unit of 2049 steps: 31 us with 8 or 16, 52 with 4, 97 with 2; four of 126:
// 16 with 4, 17 with 2, 25 with 16; eight of 33: 13 with 2, 15 with 4.
int least_steps(const Problem& p) {
    const int longest = (std::max(p.prefix.Tk, p.any_own ? p.own.Tk : 0) + 15) / 16;
    return std::max(2, (int)(std::sqrt((double)longest) / 3 + 0.5));
}

// Parts that the kernels on CUDA cores take a half's keys in.
int key_parts(const Problem& p, const Geom& g, int sms) { return p.tensor ? 1 : na2d_attn::simt_key_parts(g, sms); }

struct ForwardLayout {
    size_t q, o_prefix, lse_prefix, o_own, lse_own, scratch, scratch_bytes, own_scratch, own_scratch_bytes, table, part_o, part_lse, size;
};
ForwardLayout forward_layout(const Problem& p, int sms) {
    Layout l;
    ForwardLayout f{};
    const size_t rows = p.rows.all, values = rows * p.rows.C;
    const OnLine line = on_line(p);
    if (!line.prefix) {
        if (!p.follow[0]) f.q = l.take(values * esize_of(p));
        const int parts = key_parts(p, p.prefix, sms);
        f.o_prefix = l.take(parts * values * 4);
        f.lse_prefix = l.take(parts * rows * 4);
        if (p.tensor) f.scratch_bytes = na2d_attn::forward_floats(p.prefix, sms) * 4;
    }
    if (p.any_own && !line.own) {
        const int parts = key_parts(p, p.own, sms);
        f.o_own = l.take(parts * values * 4);
        f.lse_own = l.take(parts * rows * 4);
        if (p.tensor) f.own_scratch_bytes = na2d_attn::forward_floats(p.own, sms) * 4;
    }
    f.scratch = l.take(f.scratch_bytes);
    f.own_scratch = l.take(f.own_scratch_bytes);
    if (line.any()) {
        const size_t parts = (line.prefix ? line_rows(p.prefix, sms) : 0) + (line.own ? line_rows(p.own, sms) : 0);
        f.table = l.take((na2d_prefix::kTokenEntries + 2) * sizeof(int));
        f.part_o = l.take(parts * p.rows.C * 4);
        f.part_lse = l.take(parts * 4);
    }
    f.size = l.size;
    return f;
}
struct BackwardLayout {
    size_t rows[3], lse, delta_prefix, delta, dq_prefix, dq_own, scratch, scratch_bytes, prefix_sums, own_sums, size;
};
// d_prefix, d_own: whether that half's keys have gradients.
BackwardLayout backward_layout(const Problem& p, int sms, bool d_q, bool d_prefix, bool d_own) {
    Layout l;
    BackwardLayout f{};
    const size_t rows = p.rows.all, values = rows * p.rows.C;
    const bool f16 = p.dtype == NA2D_F16;
    for (int i = 0; i < 3; ++i)
        if (!p.follow[i]) f.rows[i] = l.take(values * esize_of(p));
    f.lse = l.take(rows * 4);
    f.delta_prefix = l.take(rows * 4);
    f.delta = l.take(rows * 4);
    if (d_q) {
        f.dq_prefix = l.take(key_parts(p, p.prefix, sms) * values * 4);
        if (p.any_own) f.dq_own = l.take(key_parts(p, p.own, sms) * values * 4);
    }
    auto sums = [&](const Geom& g) {                     // of the key half on CUDA cores
        return l.take(p.tensor ? 0 : 2 * (size_t)na2d_attn::simt_row_parts(g, sms) * g.units * g.Tk * g.C * 4);
    };
    if (d_prefix) f.prefix_sums = sums(p.prefix);
    if (p.any_own && d_own) f.own_sums = sums(p.own);
    if (p.tensor) {
        f.scratch_bytes = na2d_attn::backward_floats(p.prefix, sms, f16, d_q, d_prefix) * 4;
        if (p.any_own) f.scratch_bytes = std::max(f.scratch_bytes, na2d_attn::backward_floats(p.own, sms, f16, d_q, d_own) * 4);
    }
    f.scratch = l.take(f.scratch_bytes);
    f.size = l.size;
    return f;
}

// x as the prefixes' problem sees it: (S, N, A Tq, C).
Operand merged(const Problem& p, const Operand& x) {
    const Rows& g = p.rows;
    if (g.A == 1) return x;
    return Operand{x.ptr, g.A * x.b, x.n, g.Tq == 1 ? x.b : x.t};
}
Operand merged_copy(const Problem& p, void* at) {
    const Rows& g = p.rows;
    const long long row = g.C, head = (long long)g.A * g.Tq * row;
    return Operand{at, g.N * head, head, row};
}
// x as the entries' own problem sees it.
Operand own_rows(const Problem& p, const Operand& x) { return p.heads_as_rows ? Operand{x.ptr, x.b, p.prefix.G * x.n, x.n} : x; }
// A dense result in fp32.
Operand sums(const Geom& g, float* at) {
    const long long head = (long long)g.Tq * g.C;
    Operand x{at, g.N * head, head, g.C};
    x.wide = true;
    return x;
}

int place(int dtype, int device, void* stream, int* launched, na2d_attn::Place* at) {
    *at = na2d_attn::Place{dtype, device, (cudaStream_t)stream, nullptr, launched};
    return na2d_host::error_state(device, &at->errors);
}
int finish(int rc, int launched, const char* what) {
    na2d_host::count_launches(launched);
    return rc == NA2D_ERR_CUDA ? na2d_host::launch_fail(what) : rc;
}

int forward_of(const Problem& p, const na2d_attn::Place& at, const Geom& g, const Scratch& s, const Operand& q, const Operand& k, const Operand& v,
               const Operand& o, float* lse, na2d_attn::Parts* parts = nullptr) {
    return p.dtype == NA2D_BF16 ? na2d_attn::forward_bf16(at, g, s, q, k, v, o, lse, parts) : na2d_attn::forward_f16(at, g, s, q, k, v, o, lse, parts);
}
int backward_of(const Problem& p, const na2d_attn::Place& at, const Scratch& s, const na2d_attn::Backward* x, int count) {
    if (!p.tensor) return count ? na2d_attn::simt_backward(at, x, count) : NA2D_OK;
    for (int i = 0; i < count; ++i)
        if (int rc = p.dtype == NA2D_BF16 ? na2d_attn::backward_bf16(at, s, x[i]) : na2d_attn::backward_f16(at, s, x[i])) return rc;
    return NA2D_OK;
}

// Copies of those operands whose rows do not follow one another, and of lse.
int gather(const na2d_attn::Place& at, const Problem& p, const Operand* const* from, char* const* to, int tensors, const float* lse, float* lse_to) {
    Gather x{};
    const long long esize = (long long)esize_of(p);
    x.tensors = tensors;
    x.lse = lse;
    x.lse_to = lse_to;
    const long long row_bytes = p.rows.C * esize;
    bool by_16 = row_bytes % 16 == 0;
    for (int i = 0; i < tensors; ++i) {
        x.from[i] = from[i]->ptr;
        x.to[i] = to[i];
        x.b[i] = from[i]->b * esize;
        x.n[i] = from[i]->n * esize;
        x.t[i] = from[i]->t * esize;
        by_16 = by_16 && reinterpret_cast<uintptr_t>(from[i]->ptr) % 16 == 0 && x.b[i] % 16 == 0 && x.n[i] % 16 == 0 && x.t[i] % 16 == 0;
    }
    const int sides = tensors + (lse ? 1 : 0);
    if (!sides) return NA2D_OK;
    const int pieces = tensors ? (int)(row_bytes / (by_16 ? 16 : esize)) : 1;
    x.by_pieces = na2d_attn::Div(pieces);
    const dim3 grid(blocks_of(p.rows, pieces), (unsigned)sides);
    *at.launched += 1;
    const cudaError_t e = by_16        ? na2d_launch::launch(true, gather_rows_kernel<uint4>, grid, kThreads, 0, at.st, p.rows, x)
                          : esize == 4 ? na2d_launch::launch(true, gather_rows_kernel<uint32_t>, grid, kThreads, 0, at.st, p.rows, x)
                                       : na2d_launch::launch(true, gather_rows_kernel<uint16_t>, grid, kThreads, 0, at.st, p.rows, x);
    return e == cudaSuccess ? NA2D_OK : NA2D_ERR_CUDA;
}

template <typename DT, int N>
int join_outputs(const na2d_attn::Place& at, const Problem& p, const float* o_prefix, const float* lse_prefix, const float* o_own,
                 const float* lse_own, void* o, float* lse) {
    const int pieces = p.rows.C / N, sms = na2d_host::sm_count(at.device);
    *at.launched += 1;
    return na2d_launch::launch(true, join_outputs_kernel<DT, N>, blocks_of(p.rows, pieces), kThreads, 0, at.st, p.rows, na2d_attn::Div(pieces), o_prefix,
                               lse_prefix, o_own, lse_own, key_parts(p, p.prefix, sms), p.any_own ? key_parts(p, p.own, sms) : 0, static_cast<DT*>(o),
                               lse) == cudaSuccess
               ? NA2D_OK
               : NA2D_ERR_CUDA;
}
template <typename DT, int N>
int join_gradients(const na2d_attn::Place& at, const Problem& p, const float* prefix, const float* own, void* d_q) {
    const int pieces = p.rows.C / N, sms = na2d_host::sm_count(at.device);
    *at.launched += 1;
    return na2d_launch::launch(true, join_gradients_kernel<DT, N>, blocks_of(p.rows, pieces), kThreads, 0, at.st, p.rows, na2d_attn::Div(pieces), prefix,
                               own, key_parts(p, p.prefix, sms), p.any_own ? key_parts(p, p.own, sms) : 0, static_cast<DT*>(d_q)) == cudaSuccess
               ? NA2D_OK
               : NA2D_ERR_CUDA;
}
// f(element type, channels of a vector) for rows that are written at `to`
template <typename F>
int by_type(const Problem& p, const void* to, F&& f) {
    using One = std::integral_constant<int, 1>;
    using Four = std::integral_constant<int, 4>;
    const bool four = p.rows.C % 4 == 0 && reinterpret_cast<uintptr_t>(to) % (4 * esize_of(p)) == 0;
    if (p.dtype == NA2D_F32) return four ? f(float{}, Four{}) : f(float{}, One{});
    if (p.dtype == NA2D_BF16) return four ? f(__nv_bfloat16{}, Four{}) : f(__nv_bfloat16{}, One{});
    return four ? f(__half{}, Four{}) : f(__half{}, One{});
}

bool dense(const na2d_heads& x) { return x.stride_b == 0 && x.stride_n == 0 && x.stride_t == 0; }
bool enough(const na2d_prefix_attention_args* a, size_t bytes) {
    return a->workspace && reinterpret_cast<uintptr_t>(a->workspace) % 256 == 0 && a->workspace_bytes >= bytes;
}

}  // namespace

extern "C" {

int na2d_prefix_attention_forward(const na2d_prefix_attention_args* a) {
    if (!a || !a->q.ptr || !a->prefix_k.ptr || !a->prefix_v.ptr || !a->o.ptr || !a->lse) return NA2D_ERR_BAD_ARG;
    Problem p{};
    if (int rc = make_problem(a, &p)) return rc;
    if (p.any_own && (!a->k.ptr || !a->v.ptr)) return NA2D_ERR_BAD_ARG;
    if (!dense(a->o)) return NA2D_ERR_UNSUPPORTED;
    const ForwardLayout f = forward_layout(p, na2d_host::sm_count(a->device));
    if (!enough(a, f.size)) return NA2D_ERR_BAD_ARG;
    return na2d_host::on_device(a->device, [&]() -> int {
        int launched = 0;
        na2d_attn::Place at;
        if (int rc = place(a->dtype, a->device, a->stream, &launched, &at)) return rc;
        char* ws = static_cast<char*>(a->workspace);
        auto floats = [&](size_t where) { return reinterpret_cast<float*>(ws + where); };
        const Scratch scratch{floats(f.scratch), f.scratch_bytes / 4}, own_scratch{floats(f.own_scratch), f.own_scratch_bytes / 4};
        const OnLine line = on_line(p);
        auto run = [&]() -> int {
            na2d_attn::Parts prefix{};
            if (!line.prefix) {
                Operand q = p.follow[0] ? merged(p, p.q) : merged_copy(p, ws + f.q);
                if (!p.follow[0]) {
                    const Operand* from = &p.q;
                    char* to = ws + f.q;
                    if (int rc = gather(at, p, &from, &to, 1, nullptr, nullptr)) return rc;
                }
                if (!p.tensor) {
                    const na2d_attn::Forward x[2] = {{&p.prefix, q, p.pk, p.pv, sums(p.prefix, floats(f.o_prefix)), floats(f.lse_prefix)},
                                                     {&p.own, own_rows(p, p.q), p.k, p.v, sums(p.own, floats(f.o_own)), floats(f.lse_own)}};
                    if (int rc = na2d_attn::simt_forward(at, x, p.any_own ? 2 : 1)) return rc;
                } else if (int rc = forward_of(p, at, p.prefix, scratch, q, p.pk, p.pv, sums(p.prefix, floats(f.o_prefix)), floats(f.lse_prefix),
                                        line.any() ? &prefix : nullptr))
                    return rc;
            }
            if (p.tensor && p.any_own && !line.own)
                if (int rc = forward_of(p, at, p.own, own_scratch, p.q, p.k, p.v, sums(p.own, floats(f.o_own)), floats(f.lse_own))) return rc;
            if (line.any()) {
                na2d_prefix::Tokens x{};
                auto side = [&](int which, const Geom& g, const Operand& k, const Operand& v, int share, size_t first_row) {
                    x.side[which] = na2d_prefix::TokenSide{k, v, g.lengths, g.B, g.Tk, share, g.G * g.Tq, first_row};
                };
                const size_t rows = line.prefix ? line_rows(p.prefix, na2d_host::sm_count(a->device)) : 0;
                if (line.prefix) side(0, p.prefix, p.pk, p.pv, p.rows.A, 0);
                if (line.own) side(1, p.own, p.k, p.v, 1, rows);
                x.q = p.q;
                x.N = p.rows.N;
                x.Nk = p.prefix.Nk;
                x.G = p.prefix.G;
                x.Tq = p.rows.Tq;
                x.C = p.rows.C;
                x.causal = p.any_own && p.own.causal;
                x.sl2 = p.prefix.sl2;
                x.behind = launched > 0;
                x.least = least_steps(p);
                x.by_tq = na2d_attn::Div(p.rows.Tq);
                x.by_n = na2d_attn::Div(p.rows.N);
                x.by_g = na2d_attn::Div(p.prefix.G);
                x.table = reinterpret_cast<int*>(ws + f.table);
                x.part_o = floats(f.part_o);
                x.part_lse = floats(f.part_lse);
                const na2d_prefix::JoinPrefix by_prefix{prefix.o, prefix.lse, (size_t)p.rows.all, prefix.count, p.rows.A, na2d_attn::Div(p.rows.A)};
                return p.dtype == NA2D_BF16 ? na2d_prefix::tokens_bf16(at, x, by_prefix, a->o.ptr, a->lse, p.B)
                                            : na2d_prefix::tokens_f16(at, x, by_prefix, a->o.ptr, a->lse, p.B);
            }
            const float *o_own = p.any_own ? floats(f.o_own) : nullptr, *lse_own = p.any_own ? floats(f.lse_own) : nullptr;
            return by_type(p, a->o.ptr, [&](auto type, auto n) {
                return join_outputs<decltype(type), decltype(n)::value>(at, p, floats(f.o_prefix), floats(f.lse_prefix), o_own, lse_own, a->o.ptr, a->lse);
            });
        };
        return finish(run(), launched, "prefix attention forward launch");
    });
}

int na2d_prefix_attention_backward(const na2d_prefix_attention_args* a) {
    if (!a || !a->q.ptr || !a->prefix_k.ptr || !a->prefix_v.ptr || !a->o.ptr || !a->d_o.ptr || !a->lse) return NA2D_ERR_BAD_ARG;
    const bool d_prefix = a->d_prefix_k.ptr != nullptr, d_own = a->d_k.ptr != nullptr, d_q = a->d_q.ptr != nullptr;
    if (d_prefix != (a->d_prefix_v.ptr != nullptr) || d_own != (a->d_v.ptr != nullptr) || !(d_q || d_prefix || d_own)) return NA2D_ERR_BAD_ARG;
    Problem p{};
    if (int rc = make_problem(a, &p)) return rc;
    if (p.any_own ? !a->k.ptr || !a->v.ptr : d_own) return NA2D_ERR_BAD_ARG;
    for (const na2d_heads* x : {&a->d_q, &a->d_k, &a->d_v, &a->d_prefix_k, &a->d_prefix_v})
        if (!dense(*x)) return NA2D_ERR_UNSUPPORTED;
    const BackwardLayout f = backward_layout(p, na2d_host::sm_count(a->device), d_q, d_prefix, d_own);
    if (!enough(a, f.size)) return NA2D_ERR_BAD_ARG;
    return na2d_host::on_device(a->device, [&]() -> int {
        int launched = 0;
        na2d_attn::Place at;
        if (int rc = place(a->dtype, a->device, a->stream, &launched, &at)) return rc;
        char* ws = static_cast<char*>(a->workspace);
        auto floats = [&](size_t where) { return reinterpret_cast<float*>(ws + where); };
        const Scratch scratch{floats(f.scratch), f.scratch_bytes / 4};
        auto result = [&](void* ptr, int B, int T) {     // a dense gradient of keys
            const long long head = (long long)T * a->C;
            return Operand{ptr, a->Nk * head, head, a->C};
        };
        auto run = [&]() -> int {
            const float* lse = a->lse;
            na2d_attn::Backward x_of[2]{};
            int count = 0;
            if (d_q || d_prefix) {
                const Operand* given[3] = {&p.q, &p.o, &p.d_o};
                Operand x[3];
                const Operand* from[3];
                char* to[3];
                int copies = 0;
                for (int i = 0; i < 3; ++i) {
                    x[i] = p.follow[i] ? merged(p, *given[i]) : merged_copy(p, ws + f.rows[i]);
                    if (p.follow[i]) continue;
                    from[copies] = given[i];
                    to[copies++] = ws + f.rows[i];
                }
                const bool lse_apart = p.rows.A > 1 && p.rows.N > 1;
                if (int rc = gather(at, p, from, to, copies, lse_apart ? lse : nullptr, floats(f.lse))) return rc;
                na2d_attn::Backward& b = x_of[count++];
                b.g = &p.prefix;
                b.q = x[0];
                b.o = x[1];
                b.d_o = x[2];
                b.k = p.pk;
                b.v = p.pv;
                b.lse = lse_apart ? floats(f.lse) : lse;
                b.delta = floats(f.delta_prefix);
                if (d_q) b.d_q = sums(p.prefix, floats(f.dq_prefix));
                if (d_prefix) {
                    b.d_k = result(a->d_prefix_k.ptr, a->S, a->P);
                    b.d_v = result(a->d_prefix_v.ptr, a->S, a->P);
                    if (!p.tensor) b.key_sums = floats(f.prefix_sums);
                }
            }
            if (p.any_own && (d_q || d_own)) {
                na2d_attn::Backward& b = x_of[count++];
                b.g = &p.own;
                b.q = own_rows(p, p.q);
                b.o = own_rows(p, p.o);
                b.d_o = own_rows(p, p.d_o);
                b.k = p.k;
                b.v = p.v;
                b.lse = lse;
                b.delta = floats(f.delta);
                if (d_q) b.d_q = sums(p.own, floats(f.dq_own));
                if (d_own) {
                    b.d_k = result(a->d_k.ptr, a->B, a->Tk);
                    b.d_v = result(a->d_v.ptr, a->B, a->Tk);
                    if (!p.tensor) b.key_sums = floats(f.own_sums);
                }
            }
            if (int rc = backward_of(p, at, scratch, x_of, count)) return rc;
            if (!d_q) return NA2D_OK;
            return by_type(p, a->d_q.ptr, [&](auto type, auto n) {
                return join_gradients<decltype(type), decltype(n)::value>(at, p, floats(f.dq_prefix), p.any_own ? floats(f.dq_own) : nullptr, a->d_q.ptr);
            });
        };
        return finish(run(), launched, "prefix attention backward launch");
    });
}

size_t na2d_prefix_attention_workspace(const na2d_prefix_attention_args* a, int backward) {
    Problem p{};
    if (make_problem(a, &p) != NA2D_OK) return 0;
    const int sms = na2d_host::sm_count(a->device);
    return backward ? backward_layout(p, sms, a->d_q.ptr != nullptr, a->d_prefix_k.ptr != nullptr, a->d_k.ptr != nullptr).size
                    : forward_layout(p, sms).size;
}

}  // extern "C"
