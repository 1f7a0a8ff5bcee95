// What the binding files of the torch extension module share: argument checks, the current
// stream, scratch from torch's allocator, and the Plan object behind a ScatterData.
#pragma once

#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <vector>

#include "texb_scatter.h"

namespace texb_binding {

#define TEXB_CHECK_CUDA(x) TORCH_CHECK((x).device().is_cuda(), #x, " must be a CUDAtensor ")
#define TEXB_CHECK_CONTIGUOUS(x) TORCH_CHECK((x).is_contiguous(), #x, " must be contiguous ")
#define TEXB_CHECK_INPUT(x) \
  TEXB_CHECK_CUDA(x);       \
  TEXB_CHECK_CONTIGUOUS(x)
#define TEXB_CHECK_DTYPE(x, t) \
  TORCH_CHECK((x).scalar_type() == (t), #x, " must have dtype ", (t), ", got ", (x).scalar_type())

// Forward-mode derivatives are not computed: a tensor that carries one is refused, not read as a constant.
inline void check_no_tangent(const at::Tensor& t, const char* name) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), name, " carries a forward-mode derivative, which is not supported");
}

inline void check_status(int status, const char* what) {
  TORCH_CHECK(status == TEXB_OK, what, " failed with status ", status, ": ", texb_last_error());
}

inline void* stream_of(const at::Tensor& t) {
  return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

inline at::Tensor scratch(size_t bytes, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes > 0 ? bytes : 1)}, like.options().dtype(at::kByte));
}

struct Plan {
  at::Tensor sid;      // int32 [n]: segment id at each segment-sorted position
  at::Tensor perm;     // int32 [n]: feats row at that position; undefined when the ids arrived sorted
  at::Tensor offsets;  // int32 [m + 1]: TorchEx's preSum
  at::Tensor balance;  // int32 [K + 1]: cost-balanced cut points of the sorted rows
  int64_t num_total = 0, num_segments = 0;
  int64_t max_cnt = -1;    // rows of the largest segment, -1 while the host does not know it
  bool has_empty = true;   // false only once the host knows that every segment has rows
  bool settled = false;    // the host has synchronised with the stream since the arrays were built
  bool no_split = false;   // every cut of the balance table is a segment start (short segments only)
  struct Scratch {
    int64_t channels;
    int slot;  // 0: single calls; k: the k-th reduction of a sequence; -1: the two-output operator
    void* stream;
    at::Tensor buffer;
  };
  std::vector<Scratch> scratch_cache;  // one buffer per (channel count, operator kind, stream)

  int flags() const {
    return (has_empty || num_total == 0 ? TEXB_PLAN_HAS_EMPTY : 0) | (settled ? TEXB_PLAN_SETTLED : 0) |
           (no_split ? TEXB_PLAN_NO_SPLIT : 0);
  }
  const int32_t* perm_ptr() const { return perm.defined() ? perm.data_ptr<int>() : nullptr; }

  // Calls on one stream are ordered, so they can share a buffer; another stream gets its own.
  at::Tensor& workspace(int64_t channels, int slot, void* stream, size_t bytes) {
    for (auto& s : scratch_cache)
      if (s.channels == channels && s.slot == slot && s.stream == stream) {
        if (size_t(s.buffer.numel()) < bytes) s.buffer = scratch(bytes, sid);
        return s.buffer;
      }
    scratch_cache.push_back({channels, slot, stream, scratch(bytes, sid)});
    return scratch_cache.back().buffer;
  }
};

void register_token_ops(py::module& m);   // token_ops_binding.cpp
void register_attention(py::module& m);   // attention_binding.cpp

}  // namespace texb_binding
