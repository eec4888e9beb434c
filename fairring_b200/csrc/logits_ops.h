// torch-facing wrappers of the kernels that ask a language-model head's logits for probabilities.
#pragma once

#include <pybind11/pybind11.h>

namespace fairring {
void bindLogitsOps(pybind11::module_& m);
}  // namespace fairring
