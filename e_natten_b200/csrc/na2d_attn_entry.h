// Host entry points of the kernels of attention over all keys: on tensor cores, compiled once per 16-bit element type
// (na2d_attn_tc.cu with -DNA2D_TC_DT=1 for bf16 and 2 for fp16), and on CUDA cores (na2d_attn_simt.cu).
#pragma once

#include "na2d_attn.cuh"

namespace na2d_attn {

// Scratch (fp32) for results that are computed in parts, of which there are fewer with less than *_floats() of it, and for the bounds of
// fp16's backward.
struct Scratch {
    float* at;
    size_t floats;
};
size_t forward_floats(const Geom& g, int sms);
size_t backward_floats(const Geom& g, int sms, bool f16, bool d_q, bool d_k);

// What a tensor map needs of an operand: a base and strides on 16-byte boundaries, strides below 2^40 bytes.
inline bool tma_ready(const Operand& x) {
    if (reinterpret_cast<uintptr_t>(x.ptr) & 15u) return false;
    for (long long s : {x.b, x.n, x.t})
        if (s <= 0 || (s & 7) != 0 || s >= (1ll << 39)) return false;
    return true;
}

// How a wide result lies, where whoever asked for it joins the parts itself: `count` of them, each of the rows (B, N, Tq), one behind
// the other.
struct Parts {
    const float *o, *lse;
    int count;
};

// 16 bits, C a multiple of 8 up to 128, every operand on 16-byte boundaries; o, d_q, d_k and d_v dense.  o and d_q may be `wide`; of a wide o only
// rows with a finite lse are written, where rows are not in parts.
int forward_bf16(const Place& at, const Geom& g, const Scratch& scratch, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse,
                 Parts* parts = nullptr);
int forward_f16(const Place& at, const Geom& g, const Scratch& scratch, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse,
                Parts* parts = nullptr);

// d_q.ptr or d_k.ptr (with d_v.ptr) may be null: that half is left out.  Writes delta.
struct Backward {
    const Geom* g;
    Operand q, k, v, o, d_o, d_q, d_k, d_v;
    const float* lse;
    float* delta;
    float* key_sums = nullptr;          // CUDA cores: room for simt_row_parts dK and dV, fp32; null: the key half is not taken in parts
};
int backward_bf16(const Place& at, const Scratch& scratch, const Backward& x);
int backward_f16(const Place& at, const Scratch& scratch, const Backward& x);

// CUDA cores: any strides, C up to kSimtMaxC, fp32 and 16 bits.
// One problem, or two of one head dim whose results are alike, `wide` or not, in the same launches.
constexpr int kSimtMaxC = 256;
struct Forward {
    const Geom* g;
    Operand q, k, v, o;
    float* lse;
};
int simt_forward(const Place& at, const Forward* x, int count);
// Parts of the keys, whose wide o and lse, or wide d_q, lie one behind the other, and of the rows in the key half.
int simt_key_parts(const Geom& g, int sms);
int simt_row_parts(const Geom& g, int sms);
int simt_backward(const Place& at, const Backward* x, int count);

}  // namespace na2d_attn
