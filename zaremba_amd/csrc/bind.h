// What the files of host entry points share.
#pragma once

#include <torch/extension.h>

#include <ATen/hip/HIPContext.h>
#include <hip/hip_runtime.h>

#define HIP_CHECK(expr)                                              \
  do {                                                               \
    hipError_t _e = (expr);                                          \
    TORCH_CHECK(_e == hipSuccess, "HIP error: ", hipGetErrorString(_e)); \
  } while (0)

namespace zamd {

inline hipStream_t current_stream() {
  return at::hip::getCurrentHIPStream().stream();
}

void bind_adamw(py::module_& m);
void bind_glr(py::module_& m);

}  // namespace zamd
