// What the PyTorch kernels share: streams, the library's errors, and checks
// of tensors that a kernel reads or writes through their pointers.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cstdint>
#include <limits>

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

constexpr int64_t kPage = 64;

inline int as_int(int64_t x, const char* name) {
  TORCH_CHECK_VALUE(x >= 0 && x <= std::numeric_limits<int>::max(), name, " ", x, " does not fit 31 bits");
  return static_cast<int>(x);
}

inline void check_table(const at::Tensor& t, int64_t B, const c10::Device& dev) {
  require_on(t, dev, "block_table");
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == B && (t.size(1) <= 1 || t.stride(1) == 1),
                    "block_table must be int32 [B, pages_per_seq] with unit column stride");
}

inline void check_lens(const at::Tensor& t, int64_t B, const c10::Device& dev, const char* name) {
  require_on(t, dev, name);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == B && t.is_contiguous(), name,
                    " must be contiguous int32 [B]");
}

// fp16 rows that the kernels read as 16-byte vectors: feature stride 1, other
// strides multiples of 8, 16-byte aligned; anything else is copied into that form.
inline at::Tensor rows_operand(const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA (HIP) tensor; there is no CPU path");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kHalf, name, " must be float16 (got ", t.scalar_type(), ")");
  TORCH_CHECK_VALUE(t.dim() == 4, name, " must be 4-D [B, T, H, D]");
  const auto st = t.strides();
  const bool ready = st[3] == 1 && st[0] % 8 == 0 && st[1] % 8 == 0 && st[2] % 8 == 0 &&
                     reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return ready ? t : t.clone(at::MemoryFormat::Contiguous);
}

}  // namespace spyre_torch
