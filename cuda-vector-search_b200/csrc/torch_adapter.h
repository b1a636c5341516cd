// Registers the query adapter's operators (torch_adapter.cpp) with the binding.
#pragma once

#include <torch/extension.h>

namespace cvs_torch {

void bind_adapter(pybind11::module_& m);

}  // namespace cvs_torch
