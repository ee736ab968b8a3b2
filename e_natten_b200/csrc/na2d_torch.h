// What the files of the extension module share: layout tests and the exception of a status.
#pragma once

#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>

#include <optional>

#include "../../include/na2d.h"

namespace na2d_torch {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

// Whether the kernels can read t in place: contiguous channels, no broadcast dimension, and for 16-bit types (the
// tensor-core path's TMA tensor maps) a base and strides on 16-byte boundaries.
inline bool kernel_ready(const Tensor& t) {
    if (t.numel() == 0) return true;
    if (t.dim() == 0) return false;
    const auto sizes = t.sizes();
    const auto strides = t.strides();
    const int64_t last = t.dim() - 1;
    if (strides[last] != 1 && sizes[last] != 1) return false;
    const bool half = t.element_size() == 2;
    if (half && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
    for (int64_t i = 0; i < last; ++i) {
        if (sizes[i] <= 1) continue;
        if (strides[i] <= 0 || (half && strides[i] % 8)) return false;
    }
    return true;
}
inline Tensor in_place_or_copy(const Tensor& t) { return kernel_ready(t) ? t : t.contiguous(); }

// A dimension of extent 1 may report any stride; the library ignores it, but all-zero means dense.
inline int64_t at_least_one(int64_t stride) { return stride < 1 ? 1 : stride; }
// Raises what _lib.check raises for a status.
inline void check(int status) {
    if (status == NA2D_OK) return;
    pybind11::gil_scoped_acquire gil;
    pybind11::module_::import("e_natten_b200._lib").attr("check")(status);
}

// group_norm, rotary and attention (na2d_torch_block.cpp).
void add_block_operators(pybind11::module_& m);

}  // namespace na2d_torch
