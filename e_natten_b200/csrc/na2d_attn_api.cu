// C entry points of attention over all keys (include/na2d.h): argument checks, choice of kernels, parts and workspace.
#include <cstddef>

#include "na2d_attn_entry.h"
#include "na2d_host.h"

namespace {

using na2d_attn::Geom;
using na2d_attn::Operand;

struct Problem {
    Geom g;
    bool tensor = false;
    Operand q, k, v, o, d_o, d_q, d_k, d_v;
};

// What a tensor map needs of an operand: a base and strides on 16-byte boundaries, strides below 2^40 bytes.
bool tma_ready(const Operand& x) {
    if (reinterpret_cast<uintptr_t>(x.ptr) & 15u) return false;
    for (long long s : {x.b, x.n, x.t})
        if (s <= 0 || (s & 7) != 0 || s >= (1ll << 39)) return false;
    return true;
}

int make_problem(const na2d_attention_args* a, Problem* p) {
    if (!a || a->struct_size < sizeof(na2d_attention_args)) return NA2D_ERR_BAD_ARG;
    if (a->B <= 0 || a->N <= 0 || a->Nk <= 0 || a->Tq <= 0 || a->Tk <= 0 || a->C <= 0 || a->N % a->Nk != 0) return NA2D_ERR_BAD_ARG;
    if (a->dtype != NA2D_F32 && a->dtype != NA2D_BF16 && a->dtype != NA2D_F16) return NA2D_ERR_UNSUPPORTED;
    if (a->path != NA2D_PATH_AUTO && a->path != NA2D_PATH_SIMT && a->path != NA2D_PATH_TENSOR) return NA2D_ERR_BAD_ARG;
    if (!(a->scale > 0.f) || !(a->scale < 3.0e38f)) return NA2D_ERR_BAD_ARG;
    if (a->workspace && reinterpret_cast<uintptr_t>(a->workspace) % 16) return NA2D_ERR_BAD_ARG;
    // (tokens and chunks are counted in 32 bits, with room for a sum of two lengths and a tile; rows of all heads in 31)
    if (a->Tq > (1 << 29) || a->Tk > (1 << 29) || (long long)a->B * a->N > (1 << 24)) return NA2D_ERR_TOO_LARGE;
    Geom& g = p->g;
    g.B = a->B; g.N = a->N; g.Nk = a->Nk; g.Tq = a->Tq; g.Tk = a->Tk; g.C = a->C;
    g.causal = a->causal != 0;
    g.lengths = a->key_lengths;
    g.scale = a->scale;
    g.sl2 = a->scale * 1.4426950408889634f;
    na2d_attn::cut_rows(g);
    auto operand = [&](const na2d_heads& x, int heads, int T) {
        const na2d_host::HeadStrides s = na2d_host::head_strides(x, a->B, heads, T, a->C);
        return Operand{x.ptr, s.b, s.n, s.t};
    };
    p->q = operand(a->q, a->N, a->Tq);
    p->o = operand(a->o, a->N, a->Tq);
    p->d_o = operand(a->d_o, a->N, a->Tq);
    p->d_q = operand(a->d_q, a->N, a->Tq);
    p->k = operand(a->k, a->Nk, a->Tk);
    p->v = operand(a->v, a->Nk, a->Tk);
    p->d_k = operand(a->d_k, a->Nk, a->Tk);
    p->d_v = operand(a->d_v, a->Nk, a->Tk);
    // results are written as rows of a dense tensor
    for (const na2d_heads* x : {&a->o, &a->d_q, &a->d_k, &a->d_v})
        if (x->ptr && (x->stride_b || x->stride_n || x->stride_t)) {
            const bool rows = x == &a->o || x == &a->d_q;
            const na2d_host::HeadStrides d = na2d_host::head_strides(na2d_heads{}, a->B, rows ? a->N : a->Nk, rows ? a->Tq : a->Tk, a->C);
            const Operand& got = x == &a->o ? p->o : x == &a->d_q ? p->d_q : x == &a->d_k ? p->d_k : p->d_v;
            if (got.b != d.b || got.n != d.n || got.t != d.t) return NA2D_ERR_UNSUPPORTED;
        }
    bool fits = a->dtype != NA2D_F32 && a->C <= 128 && a->C % 8 == 0;
    for (const Operand* x : {&p->q, &p->k, &p->v, &p->o, &p->d_o, &p->d_q, &p->d_k, &p->d_v}) fits = fits && (!x->ptr || tma_ready(*x));
    if (a->path == NA2D_PATH_TENSOR && !fits) return NA2D_ERR_UNSUPPORTED;
    p->tensor = fits && a->path != NA2D_PATH_SIMT;
    if (!p->tensor && a->C > na2d_attn::kSimtMaxC) return NA2D_ERR_UNSUPPORTED;
    return NA2D_OK;
}

na2d_attn::Scratch scratch_of(const na2d_attention_args* a) {
    return na2d_attn::Scratch{static_cast<float*>(a->workspace), a->workspace ? a->workspace_bytes / sizeof(float) : 0};
}

int place(const na2d_attention_args* a, int* launched, na2d_attn::Place* at) {
    *at = na2d_attn::Place{a->dtype, a->device, (cudaStream_t)a->stream, nullptr, launched};
    return na2d_host::error_state(a->device, &at->errors);
}

int finish(int rc, int launched, const char* what) {
    na2d_host::count_launches(launched);
    return rc == NA2D_ERR_CUDA ? na2d_host::launch_fail(what) : rc;
}

}  // namespace

extern "C" {

int na2d_attention_forward(const na2d_attention_args* a) {
    if (!a || !a->q.ptr || !a->k.ptr || !a->v.ptr || !a->o.ptr || !a->lse) return NA2D_ERR_BAD_ARG;
    Problem p;
    if (int rc = make_problem(a, &p)) return rc;
    return na2d_host::on_device(a->device, [&]() -> int {
        int launched = 0;
        na2d_attn::Place at;
        if (int rc = place(a, &launched, &at)) return rc;
        int rc;
        if (!p.tensor) {
            rc = na2d_attn::simt_forward(at, p.g, p.q, p.k, p.v, p.o, a->lse);
        } else {
            const na2d_attn::Scratch scratch = scratch_of(a);
            rc = a->dtype == NA2D_BF16 ? na2d_attn::forward_bf16(at, p.g, scratch, p.q, p.k, p.v, p.o, a->lse)
                                       : na2d_attn::forward_f16(at, p.g, scratch, p.q, p.k, p.v, p.o, a->lse);
        }
        return finish(rc, launched, "attention forward launch");
    });
}

int na2d_attention_backward(const na2d_attention_args* a) {
    if (!a || !a->q.ptr || !a->k.ptr || !a->v.ptr || !a->o.ptr || !a->d_o.ptr || !a->lse || !a->delta) return NA2D_ERR_BAD_ARG;
    if ((a->d_k.ptr == nullptr) != (a->d_v.ptr == nullptr) || (!a->d_q.ptr && !a->d_k.ptr)) return NA2D_ERR_BAD_ARG;
    Problem p;
    if (int rc = make_problem(a, &p)) return rc;
    return na2d_host::on_device(a->device, [&]() -> int {
        int launched = 0;
        na2d_attn::Place at;
        if (int rc = place(a, &launched, &at)) return rc;
        const na2d_attn::Backward x{p.q, p.k, p.v, p.o, p.d_o, p.d_q, p.d_k, p.d_v, a->lse, a->delta};
        int rc;
        if (!p.tensor) {
            rc = na2d_attn::simt_backward(at, p.g, x);
        } else {
            const na2d_attn::Scratch scratch = scratch_of(a);
            rc = a->dtype == NA2D_BF16 ? na2d_attn::backward_bf16(at, p.g, scratch, x) : na2d_attn::backward_f16(at, p.g, scratch, x);
        }
        return finish(rc, launched, "attention backward launch");
    });
}

size_t na2d_attention_workspace(const na2d_attention_args* a, int backward) {
    Problem p;
    if (make_problem(a, &p) != NA2D_OK || !p.tensor) return 0;
    const int sms = na2d_tc::sm_count(a->device);
    return (backward ? na2d_attn::backward_floats(p.g, sms, a->dtype == NA2D_F16, a->d_q.ptr != nullptr, a->d_k.ptr != nullptr)
                     : na2d_attn::forward_floats(p.g, sms)) *
           sizeof(float);
}

}  // extern "C"
