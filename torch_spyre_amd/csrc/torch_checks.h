// What the PyTorch kernels share: streams, the library's errors, and checks
// of tensors that a kernel reads or writes through their pointers.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cstdint>

#include "../../include/spyre_hip.h"

namespace spyre_torch {

inline void* stream_of(const at::Tensor& t) {
  return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

inline void check_rc(const char* fn, int rc) {
  if (rc != SPYRE_OK) {
    const char* msg = spyre_last_error();
    TORCH_CHECK(false, "[spyre_hip ", fn, " ", rc, "] ", msg ? msg : "");
  }
}

// t must be a CUDA tensor on `dev`: a kernel launched there reads or writes
// it through its pointer (a host pointer would fault there).
inline void require_on(const at::Tensor& t, const c10::Device& dev, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA (HIP) tensor; there is no CPU path");
  TORCH_CHECK_VALUE(t.device() == dev, name, " is on ", t.device(), "; the call runs on ", dev);
}

}  // namespace spyre_torch
