// What the binding files share.
#pragma once

#include <torch/extension.h>

// The status word of the tensor's device, written by kernels whose bounded waits run out.
int* bgn_status_word(const at::Tensor& like);
at::Tensor kernel_status(int64_t device);  // the same as a tensor

void bgn_register_packed(pybind11::module& m);
