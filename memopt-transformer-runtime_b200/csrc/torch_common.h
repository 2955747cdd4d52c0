// torch_common.h — helpers shared by the sources of the Python module.
#pragma once
#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "memopt_b200.h"

namespace memopt_torch {

inline void check(int st, const char* what) {
  if (st != MEMOPT_OK) {
    TORCH_CHECK(false, what, ": ", memopt_last_error(), " (", memopt_status_string(st), ")");
  }
}

inline void* cur_stream() { return reinterpret_cast<void*>(at::cuda::getCurrentCUDAStream().stream()); }

inline bool aligned16(const torch::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }

inline torch::Tensor aligned_contig(const torch::Tensor& t) {
  auto c = t.contiguous();
  if (c.numel() > 0 && !aligned16(c)) c = c.clone();
  return c;
}

}  // namespace memopt_torch

// Registers the packed-batch operators (memopt_C_packed.cpp) with the module.
void bind_packed(pybind11::module_& m);
