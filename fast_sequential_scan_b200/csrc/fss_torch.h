// Shared by the C++ sources of the autograd functions.
#pragma once

#include <torch/extension.h>

#include "../../include/fss_b200.h"

namespace fss_torch {

using at::Tensor;

// unit channel stride, rows and batches that do not overlap
inline Tensor rowwise(const Tensor &t) {
    if (t.is_contiguous()) return t;
    const int64_t B = t.size(0), T = t.size(1), D = t.size(2);
    const bool ok = (D == 1 || t.stride(2) == 1) && (T == 1 || t.stride(1) >= D) && (B == 1 || t.stride(0) >= (T - 1) * t.stride(1) + D);
    return ok ? t : t.contiguous();
}
inline fss_view view(const Tensor &t) {
    const int64_t B = t.size(0), T = t.size(1), D = t.size(2);
    if (t.is_contiguous()) return {t.data_ptr(), std::max<int64_t>(T * D, 1), D};
    const int64_t st = T > 1 ? t.stride(1) : D;
    return {t.data_ptr(), B > 1 ? t.stride(0) : std::max<int64_t>(st * T, 1), st};
}
inline Tensor like(const Tensor &t) { return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)); }

// the entries of fss_torch_layers.cpp
void define_layers(py::module_ &m);

}  // namespace fss_torch
