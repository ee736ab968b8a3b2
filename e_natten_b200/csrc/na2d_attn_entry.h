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

// 16 bits, C a multiple of 8 up to 128, every operand on 16-byte boundaries; o, d_q, d_k and d_v dense.
int forward_bf16(const Place& at, const Geom& g, const Scratch& scratch, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse);
int forward_f16(const Place& at, const Geom& g, const Scratch& scratch, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse);

// d_q.ptr or d_k.ptr (with d_v.ptr) may be null: that half is left out.  Writes delta.
struct Backward {
    Operand q, k, v, o, d_o, d_q, d_k, d_v;
    const float* lse;
    float* delta;
};
int backward_bf16(const Place& at, const Geom& g, const Scratch& scratch, const Backward& x);
int backward_f16(const Place& at, const Geom& g, const Scratch& scratch, const Backward& x);

// CUDA cores: any strides, C up to kSimtMaxC, fp32 and 16 bits.
constexpr int kSimtMaxC = 256;
int simt_forward(const Place& at, const Geom& g, const Operand& q, const Operand& k, const Operand& v, const Operand& o, float* lse);
int simt_backward(const Place& at, const Geom& g, const Backward& x);

}  // namespace na2d_attn
