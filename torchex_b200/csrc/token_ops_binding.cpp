// Binding of the table lookup with its gradient, and of gradient clipping, of the module `scatter_ext`:
// tensors in, the C ABI of include/texb_scatter.h underneath.  Each call checks its arguments,
// runs on its tensors' device and on torch's current stream, and takes outputs and scratch from
// torch's caching allocator.

#include "binding.h"

#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <algorithm>
#include <climits>
#include <memory>
#include <mutex>
#include <string>
#include <tuple>

namespace texb_binding {
namespace {

int dtype_code(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return TEXB_FLOAT32;
    case at::kBFloat16: return TEXB_BFLOAT16;
    case at::kHalf: return TEXB_FLOAT16;
    default: TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

at::Tensor checked_tokens(const at::Tensor& tokens) {
  TEXB_CHECK_CUDA(tokens);
  TORCH_CHECK(tokens.scalar_type() == at::kInt || tokens.scalar_type() == at::kLong, "tokens must be int32 or int64, got ",
              tokens.scalar_type());
  return tokens.contiguous();
}

at::Tensor embedding_forward(const at::Tensor& tokens_in, const at::Tensor& weight_in, double scale) {
  const at::Tensor tokens = checked_tokens(tokens_in);
  TORCH_CHECK(weight_in.device().is_cuda(), "weight must be a CUDAtensor ");
  TORCH_CHECK(weight_in.dim() == 2, "weight must be [vocab, dim]");
  check_no_tangent(weight_in, "weight");
  TORCH_CHECK(weight_in.size(1) >= 1 && weight_in.size(1) <= INT_MAX, "weight needs between one and 2^31 - 1 columns");
  TORCH_CHECK(weight_in.device() == tokens.device(), "tokens and weight live on different devices");
  const int dtype = dtype_code(weight_in, "weight");
  const c10::cuda::CUDAGuard guard(tokens.device());
  const at::Tensor weight = weight_in.contiguous();
  auto shape = tokens.sizes().vec();
  shape.push_back(weight.size(1));
  at::Tensor out = at::empty(shape, weight.options());
  check_status(texb_embedding_forward(tokens.data_ptr(), int(tokens.element_size()), tokens.numel(), weight.data_ptr(),
                                      dtype, weight.size(0), int(weight.size(1)), float(scale), out.data_ptr(),
                                      stream_of(tokens)),
               "texb_embedding_forward");
  return out;
}

at::Tensor embedding_backward(const at::Tensor& tokens_in, const at::Tensor& g_in, int64_t vocab, double scale,
                              int64_t padding_idx) {
  const at::Tensor tokens = checked_tokens(tokens_in);
  TORCH_CHECK(g_in.device() == tokens.device(), "tokens and the gradient live on different devices");
  TORCH_CHECK(g_in.dim() == tokens.dim() + 1 && g_in.sizes().slice(0, tokens.dim()) == tokens.sizes(),
              "the gradient must have the shape of tokens and one more axis");
  check_no_tangent(g_in, "the gradient");
  const int dtype = dtype_code(g_in, "the gradient");
  const c10::cuda::CUDAGuard guard(tokens.device());
  const at::Tensor g = g_in.contiguous();
  const int64_t n = tokens.numel(), dim = g.size(-1);
  TORCH_CHECK(dim >= 1 && dim <= INT_MAX, "the gradient needs between one and 2^31 - 1 columns");
  at::Tensor out = at::empty({vocab, dim}, g.options());
  const at::Tensor ws = scratch(texb_embedding_backward_workspace_bytes(n, vocab, int(dim)), tokens);
  check_status(texb_embedding_backward(tokens.data_ptr(), int(tokens.element_size()), n, g.data_ptr(), dtype, vocab,
                                       int(dim), float(scale), padding_idx, out.data_ptr(), ws.data_ptr(),
                                       size_t(ws.numel()), stream_of(tokens)),
               "texb_embedding_backward");
  return out;
}

// The autograd node of the lookup.  A node of its own, set up by hand: a training step on a small batch costs
// more host time than its kernels take, and the general wrappers (Python's above all) would add to that.
struct EmbeddingBackward : torch::autograd::Node {
  torch::autograd::SavedVariable tokens;
  int64_t vocab = 0, padding_idx = -1;
  double scale = 1.0;

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    TORCH_CHECK(!at::GradMode::is_enabled(), "embedding is differentiable once (create_graph is not supported)");
    if (!grads[0].defined()) return {at::Tensor()};
    at::Tensor t;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      t = tokens.unpack();
    }
    return {embedding_backward(t, grads[0], vocab, scale, padding_idx)};
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    tokens.reset_data();
  }
  std::string name() const override { return "EmbeddingBackward"; }
};

at::Tensor embedding(const at::Tensor& tokens, const at::Tensor& weight, double scale, int64_t padding_idx) {
  if (!at::GradMode::is_enabled() || !weight.requires_grad()) return embedding_forward(tokens, weight, scale);
  at::Tensor out;
  {
    const at::NoGradGuard no_grad;
    out = embedding_forward(tokens, weight, scale);
  }
  auto node = std::shared_ptr<EmbeddingBackward>(new EmbeddingBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(weight));
  node->tokens = torch::autograd::SavedVariable(tokens, /*is_output=*/false);
  node->vocab = weight.size(0);
  node->scale = scale;
  node->padding_idx = padding_idx;
  torch::autograd::set_history(out, node);
  return out;
}

// ---- gradient clipping -----------------------------------------------------------------

struct Tensors {  // the host arrays of the C ABI
  std::vector<const void*> in;
  std::vector<int64_t> sizes;
  std::vector<int> dtypes;
};

Tensors gather(const std::vector<at::Tensor>& grads) {
  Tensors r;
  for (const at::Tensor& g : grads) {
    check_no_tangent(g, "a gradient");
    TORCH_CHECK(g.layout() == at::kStrided, "gradients must be dense tensors, got a sparse one");
    TORCH_CHECK(g.device().is_cuda(), "gradients must be CUDAtensors ");
    TORCH_CHECK(g.device() == grads[0].device(), "gradients live on different devices");
    TORCH_CHECK(g.is_non_overlapping_and_dense(), "gradients must fill their memory without gaps or overlaps");
    r.in.push_back(g.data_ptr());
    r.sizes.push_back(g.numel());
    r.dtypes.push_back(dtype_code(g, "gradients"));
  }
  return r;
}

// The norm and the scaled tensors have no gradient: where one would be recorded, the call is refused, so that a
// penalty on the norm does not silently lose its own.
void check_no_gradient(const std::vector<at::Tensor>& tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor& t : tensors)
    TORCH_CHECK(!t.requires_grad(), "grad_norm and clip_grads are not differentiable: detach the tensors, or call them under torch.no_grad()");
}

at::Tensor grad_norm(const std::vector<at::Tensor>& grads) {
  TORCH_CHECK(!grads.empty() && grads.size() <= size_t(INT_MAX), "grad_norm needs at least one tensor");
  check_no_gradient(grads);
  const Tensors t = gather(grads);
  const c10::cuda::CUDAGuard guard(grads[0].device());
  at::Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  const at::Tensor ws = scratch(texb_grad_norm_workspace_bytes(int(grads.size())), norm);
  check_status(texb_grad_norm(int(grads.size()), t.in.data(), t.sizes.data(), t.dtypes.data(), norm.data_ptr<float>(),
                              ws.data_ptr(), size_t(ws.numel()), stream_of(norm)),
               "texb_grad_norm");
  return norm;
}

// Outputs may not overlap each other, nor an input other than their own.
void check_apart(const Tensors& t, const std::vector<at::Tensor>& grads, const std::vector<at::Tensor>& outs) {
  struct Range { uintptr_t begin, end; size_t index; };
  std::vector<Range> ranges;
  for (size_t i = 0; i < outs.size(); ++i) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(outs[i].data_ptr());
    if (outs[i].numel() > 0) ranges.push_back({p, p + outs[i].nbytes(), i});
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  for (size_t i = 1; i < ranges.size(); ++i)
    TORCH_CHECK(ranges[i - 1].end <= ranges[i].begin, "tensors ", ranges[i - 1].index, " and ", ranges[i].index,
                " would be written to overlapping memory (the same gradient twice?)");
  for (size_t i = 0; i < grads.size(); ++i) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(t.in[i]), e = p + grads[i].nbytes();
    if (p == e) continue;
    auto at = std::partition_point(ranges.begin(), ranges.end(), [&](const Range& r) { return r.end <= p; });
    for (; at != ranges.end() && at->begin < e; ++at)
      TORCH_CHECK(at->index == i && at->begin == p, "output ", at->index, " overlaps gradient ", i);
  }
}

std::tuple<std::vector<at::Tensor>, at::Tensor> clip_grads(const std::vector<at::Tensor>& grads, double max_norm,
                                                           c10::optional<std::vector<at::Tensor>> given) {
  TORCH_CHECK(!grads.empty() && grads.size() <= size_t(INT_MAX), "clip_grads needs at least one tensor");
  TORCH_CHECK(max_norm >= 0, "max_norm must not be negative, got ", max_norm);
  check_no_gradient(grads);
  const Tensors t = gather(grads);
  const c10::cuda::CUDAGuard guard(grads[0].device());
  std::vector<at::Tensor> outs;
  if (given.has_value()) {
    outs = std::move(*given);
    check_no_gradient(outs);
    TORCH_CHECK(outs.size() == grads.size(), "out has ", outs.size(), " tensors for ", grads.size(), " gradients");
    for (size_t i = 0; i < outs.size(); ++i) {
      const at::Tensor &o = outs[i], &g = grads[i];
      check_no_tangent(o, "an output");
      TORCH_CHECK(o.device() == g.device(), "out[", i, "] lives on another device than its gradient");
      TORCH_CHECK(o.sizes() == g.sizes(), "out[", i, "] has another shape than its gradient");
      TORCH_CHECK(o.layout() == at::kStrided && ((o.is_contiguous() && g.is_contiguous()) || o.strides() == g.strides()),
                  "out[", i, "] has other strides than its gradient");
      TORCH_CHECK(o.scalar_type() == g.scalar_type() || o.scalar_type() == at::kFloat,
                  "out[", i, "] must have the dtype of its gradient or float32");
    }
    check_apart(t, grads, outs);
  } else {
    for (const at::Tensor& g : grads) outs.push_back(at::empty_like(g));
  }
  std::vector<void*> out;
  std::vector<int> out_dtypes;
  for (const at::Tensor& o : outs) {
    out.push_back(o.data_ptr());
    out_dtypes.push_back(dtype_code(o, "out"));
  }
  at::Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  const at::Tensor ws = scratch(texb_grad_norm_workspace_bytes(int(grads.size())), norm);
  check_status(texb_clip_grads(int(grads.size()), t.in.data(), t.sizes.data(), t.dtypes.data(), out.data(),
                               out_dtypes.data(), float(max_norm), norm.data_ptr<float>(), ws.data_ptr(),
                               size_t(ws.numel()), stream_of(norm)),
               "texb_clip_grads");
  if (given.has_value())
    for (const at::Tensor& o : outs)
      if (!o.is_inference()) torch::autograd::impl::bump_version(o);
  return {outs, norm};
}

}  // namespace

void register_token_ops(py::module& m) {
  m.def("embedding", &embedding, py::arg("tokens"), py::arg("weight"), py::arg("scale"), py::arg("padding_idx"));
  m.def("embedding_backward", &embedding_backward, py::arg("tokens"), py::arg("g"), py::arg("vocab"), py::arg("scale"),
        py::arg("padding_idx"));
  m.def("grad_norm", &grad_norm, py::arg("grads"));
  m.def("clip_grads", &clip_grads, py::arg("grads"), py::arg("max_norm"), py::arg("out") = c10::nullopt);
}

}  // namespace texb_binding
