// What the files of the extension module share whose calls are operators of the dispatcher: checks of arguments, layouts, the operators'
// handles.
#pragma once

#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAStream.h>

#include <limits>

#include "na2d_torch.h"

namespace na2d_torch {

// ---- checks and layouts ---------------------------------------------------------------------------------------------
inline int dtype_of(const Tensor& t) {
    return t.scalar_type() == at::kFloat ? NA2D_F32 : t.scalar_type() == at::kBFloat16 ? NA2D_BF16 : NA2D_F16;
}
// What t says of itself is in its memory.
inline void check_plain(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(!t.is_neg() && !t._is_zerotensor(), name, ": a lazily negated or zero tensor is not supported");
}
inline void check_map(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.is_cuda() && t.layout() == at::kStrided, name, ": e_natten_b200 runs on CUDA tensors only (there is no CPU path)");
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name, ": dtype ",
                      t.scalar_type(), " not supported (float32, bfloat16, float16)");
    check_plain(t, name);
}
inline void check_like(const Tensor& t, const Tensor& first, const char* name, const char* first_name) {
    check_map(t, name);
    TORCH_CHECK_VALUE(t.device() == first.device() && t.scalar_type() == first.scalar_type(), name, " must be on ", first_name,
                      "'s device, of its dtype");
}
inline int extent(int64_t n, const char* what) {
    TORCH_CHECK_VALUE(n <= std::numeric_limits<int>::max(), what, " of ", n, " is too large");
    return (int)n;
}
inline void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
inline void check_once(const char* name) {
    TORCH_CHECK(!at::GradMode::is_enabled(), name, " is not differentiable twice");
}
// (an absent tensor goes to an autograd function as none: it has no edge of the graph then)
inline MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }
inline bool wants_grad(std::initializer_list<Tensor> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : tensors)
        if (t.defined() && (t.requires_grad() || t._fw_grad(0).defined())) return true;
    return false;
}
inline Tensor scratch(size_t bytes, const Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// ---- operators of the dispatcher ------------------------------------------------------------------------------------
// Whether any of them is more than its memory; whether a call on these tensors goes through the dispatcher.
inline bool any_special(std::initializer_list<Tensor> tensors) {
    for (const Tensor& t : tensors)
        if (t.defined() && !ordinary(t) && !t.is_neg() && !t._is_zerotensor()) return true;      // (those two are refused)
    return false;
}
inline bool goes_through(std::initializer_list<Tensor> tensors) { return looked_into() || any_special(tensors); }
// The operator of that name, on arguments of F.
template <typename F>
c10::TypedOperatorHandle<F> operator_of(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// ---- layouts --------------------------------------------------------------------------------------------------------
// (B, heads, T, C), of (B, heads, H, W, C) too: a view where the grid's rows follow one another.
inline Tensor tokens(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.dim() == 4 || t.dim() == 5, name, " must be (B, heads, T, C) or (B, heads, H, W, C); got ", t.sizes());
    TORCH_CHECK_VALUE(t.size(-1) > 0, name, " has no channels");
    return t.dim() == 5 ? t.flatten(2, 3) : t;
}
inline na2d_heads heads_of(const Tensor& t) {
    const auto s = t.strides();
    return {t.data_ptr(), at_least_one(s[0]), at_least_one(s[1]), at_least_one(s[2])};
}
inline na2d_heads dense_heads(const Tensor& t) { return {t.data_ptr(), 0, 0, 0}; }

}  // namespace na2d_torch
