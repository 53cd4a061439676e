// Pieces of the torch binding that its source files share.
#pragma once

#include <torch/extension.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

namespace cmpext3_binding {

// dtype code of the C ABI, -1 for a type it does not take
int dtype_code(at::ScalarType t);

// Key-split workspace of one (device, stream): a byte tensor from torch's
// caching allocator (so torch.cuda.memory_allocated counts it), zero-filled
// when made -- its first 64 KiB are the counters every launch leaves at zero
// -- and kept for later calls on the stream, replaced by a larger one when a
// bigger plan arrives.  Calls on one stream run in order, so they can share
// it.  A stream under graph capture gets none and its launch runs unsplit: a
// captured launch would carry the buffer into replays that can run beside
// eager calls on the stream.
struct Workspace {
  void* ptr = nullptr;
  size_t bytes = 0;
};

bool capturing(hipStream_t stream);
Workspace workspace_for(const torch::Tensor& like, hipStream_t stream, size_t need);

// the paged cache's operators (paged_binding.cpp)
void register_paged(pybind11::module_& m);

}  // namespace cmpext3_binding
