// Shared pieces of the Python bindings.
#pragma once

#include <torch/extension.h>

namespace agb_python {

// One int32 status word per device; kernels write a non-zero code when a bounded wait
// ran out or an argument was rejected on the device.
torch::Tensor status_word(int device);

void bind_packed(pybind11::module& m);

}  // namespace agb_python
