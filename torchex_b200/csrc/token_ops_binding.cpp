// Binding of the token operators (table lookup and its gradient) of the module `scatter_ext`:
// tensors in, the C ABI of include/texb_scatter.h underneath.  Each call checks its arguments,
// runs on its tensors' device and on torch's current stream, and takes outputs and scratch from
// torch's caching allocator.

#include "binding.h"

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
  TORCH_CHECK(weight_in.size(1) >= 1, "weight needs at least one column");
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
  const int dtype = dtype_code(g_in, "the gradient");
  const c10::cuda::CUDAGuard guard(tokens.device());
  const at::Tensor g = g_in.contiguous();
  const int64_t n = tokens.numel(), dim = g.size(-1);
  TORCH_CHECK(dim >= 1, "the gradient needs at least one column");
  at::Tensor out = at::empty({vocab, dim}, g.options());
  const at::Tensor ws = scratch(texb_embedding_backward_workspace_bytes(n, vocab, int(dim)), tokens);
  check_status(texb_embedding_backward(tokens.data_ptr(), int(tokens.element_size()), n, g.data_ptr(), dtype, vocab,
                                       int(dim), float(scale), padding_idx, out.data_ptr(), ws.data_ptr(),
                                       size_t(ws.numel()), stream_of(tokens)),
               "texb_embedding_backward");
  return out;
}

// The autograd node of the lookup.  Compiled: a node written in Python costs more host time per step
// than the kernels of a small batch take.
struct EmbeddingNode : torch::autograd::Function<EmbeddingNode> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& tokens, const at::Tensor& weight,
                            double scale, int64_t padding_idx) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = weight.dim() == 2 ? weight.size(0) : int64_t(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding_idx"] = padding_idx;
    return embedding_forward(tokens, weight, scale);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "embedding is differentiable once (create_graph is not supported)");
    const auto saved = ctx->get_saved_variables();
    return {at::Tensor(),
            embedding_backward(saved[0], g[0], ctx->saved_data["vocab"].toInt(), ctx->saved_data["scale"].toDouble(),
                               ctx->saved_data["padding_idx"].toInt()),
            at::Tensor(), at::Tensor()};
  }
};

at::Tensor embedding(const at::Tensor& tokens, const at::Tensor& weight, double scale, int64_t padding_idx) {
  if (at::GradMode::is_enabled() && weight.requires_grad()) return EmbeddingNode::apply(tokens, weight, scale, padding_idx);
  return embedding_forward(tokens, weight, scale);
}

}  // namespace

void register_token_ops(py::module& m) {
  m.def("embedding", &embedding, py::arg("tokens"), py::arg("weight"), py::arg("scale"), py::arg("padding_idx"));
  m.def("embedding_backward", &embedding_backward, py::arg("tokens"), py::arg("g"), py::arg("vocab"), py::arg("scale"),
        py::arg("padding_idx"));
}

}  // namespace texb_binding
