// Binding of the attention within segments: tensors and a Plan in, texb_attention_forward /
// texb_attention_backward underneath, as a compiled autograd node.

#include "binding.h"

#include <cmath>
#include <tuple>

namespace texb_binding {
namespace {

constexpr int64_t kMaxDim = 128;

// Rows that the kernels can read where they are: contiguous along the head dimension, every row of every
// head on a 16-byte boundary (a slice of a fused projection qualifies).  Others are copied.
at::Tensor readable_rows(const at::Tensor& t) {
  const bool fine = t.stride(2) == 1 && (t.size(0) == 1 || t.stride(0) % 8 == 0) && (t.size(1) == 1 || t.stride(1) % 8 == 0);
  const at::Tensor r = fine ? t : t.contiguous();
  return reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0 ? r : r.clone(at::MemoryFormat::Contiguous);
}

// Strides of the rows and heads; torch leaves that of an axis of size one open.
void strides_of(const at::Tensor& t, int64_t* to) {
  to[0] = t.size(0) == 1 ? t.size(1) * t.size(2) : t.stride(0);
  to[1] = t.size(1) == 1 ? t.size(2) : t.stride(1);
}

struct Options {
  double scale = 1.0, softcap = 0.0;
  bool causal = false;
  int64_t num_segments = 0, max_count = -1;
};

texb_attention_problem problem_of(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& sid,
                                  const at::Tensor& perm, const at::Tensor& offsets, const at::Tensor& slopes, const Options& o) {
  texb_attention_problem p = {};
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  strides_of(q, p.q_strides);
  strides_of(k, p.k_strides);
  strides_of(v, p.v_strides);
  p.dtype = q.scalar_type() == at::kBFloat16 ? TEXB_BFLOAT16 : TEXB_FLOAT16;
  p.sid = sid.data_ptr<int>();
  p.perm = perm.defined() ? perm.data_ptr<int>() : nullptr;
  p.offsets = offsets.data_ptr<int>();
  p.n = q.size(0);
  p.num_segments = o.num_segments;
  p.max_count = o.max_count;
  p.heads = int(q.size(1));
  p.kv_heads = int(k.size(1));
  p.dim = int(q.size(2));
  p.scale = float(o.scale);
  p.softcap = float(o.softcap);
  p.slopes = slopes.defined() ? slopes.data_ptr<float>() : nullptr;
  p.causal = o.causal ? 1 : 0;
  return p;
}

void check_rows(const at::Tensor& t, const char* name, const at::Tensor& sid, const at::Tensor& q) {
  TORCH_CHECK(t.device().is_cuda(), name, " must be a CUDAtensor ");
  TORCH_CHECK(t.dim() == 3, name, " must be [num_total, heads, dim]");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name, " must be bfloat16 or float16, got ",
              t.scalar_type());
  TORCH_CHECK(t.scalar_type() == q.scalar_type(), name, " has another dtype than q");
  TORCH_CHECK(t.device() == sid.device(), name, " and ScatterData live on different devices");
  TORCH_CHECK(t.size(0) == sid.numel(), name, " has ", t.size(0), " rows but ScatterData was built for ", sid.numel());
  TORCH_CHECK(t.size(2) == q.size(2), name, " has another head dimension than q");
  check_no_tangent(t, name);
}

// out and, where a gradient will be wanted, what rounding took from it and the log-sums of the rows
std::tuple<at::Tensor, at::Tensor, at::Tensor> forward(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                          const at::Tensor& sid, const at::Tensor& perm, const at::Tensor& offsets,
                                          const at::Tensor& slopes, const Options& o, bool want_lse) {
  const c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor q = readable_rows(q_in), k = readable_rows(k_in), v = readable_rows(v_in);
  at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous)), low, lse;
  texb_attention_problem p = problem_of(q, k, v, sid, perm, offsets, slopes, o);
  if (want_lse) {
    low = at::empty_like(out);
    lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
  }
  p.out = out.data_ptr();
  p.out_low = want_lse ? low.data_ptr() : nullptr;
  p.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  const at::Tensor ws = scratch(texb_attention_workspace_bytes(p.n, p.heads, p.kv_heads, 0), q);
  check_status(texb_attention_forward(&p, ws.data_ptr(), size_t(ws.numel()), stream_of(q)), "texb_attention_forward");
  return {out, low, lse};
}

struct AttentionNode : torch::autograd::Function<AttentionNode> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& sid, const c10::optional<at::Tensor>& perm_given, const at::Tensor& offsets,
                            const c10::optional<at::Tensor>& slopes_given, double scale, double softcap, bool causal,
                            int64_t num_segments, int64_t max_count) {
    const at::Tensor perm = perm_given.value_or(at::Tensor()), slopes = slopes_given.value_or(at::Tensor());
    const Options o = {scale, softcap, causal, num_segments, max_count};
    const auto [out, low, lse] = texb_binding::forward(q, k, v, sid, perm, offsets, slopes, o, true);
    ctx->save_for_backward({q, k, v, sid, perm, offsets, slopes, out, low, lse});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["softcap"] = softcap;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["num_segments"] = num_segments;
    ctx->saved_data["max_count"] = max_count;
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "segment_attention is differentiable once (create_graph is not supported)");
    check_no_tangent(grads[0], "the gradient");
    const auto s = ctx->get_saved_variables();
    const Options o = {ctx->saved_data["scale"].toDouble(), ctx->saved_data["softcap"].toDouble(), ctx->saved_data["causal"].toBool(),
                       ctx->saved_data["num_segments"].toInt(), ctx->saved_data["max_count"].toInt()};
    const c10::cuda::CUDAGuard guard(s[0].device());
    const at::Tensor q = readable_rows(s[0]), k = readable_rows(s[1]), v = readable_rows(s[2]), g = readable_rows(grads[0]);
    const at::Tensor out = s[7].contiguous(), low = s[8], lse = s[9];
    const bool want_q = ctx->needs_input_grad(0), want_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    at::Tensor gq, gk, gv;
    if (want_q) gq = at::empty(q.sizes(), q.options());
    if (want_kv) {
      gk = at::empty(k.sizes(), k.options());
      gv = at::empty(v.sizes(), v.options());
    }
    texb_attention_problem p = problem_of(q, k, v, s[3], s[4], s[5], s[6], o);
    p.out = out.data_ptr();
    p.out_low = low.data_ptr();
    p.lse = lse.data_ptr<float>();
    p.g = g.data_ptr();
    strides_of(g, p.g_strides);
    p.g_q = want_q ? gq.data_ptr() : nullptr;
    p.g_k = want_kv ? gk.data_ptr() : nullptr;
    p.g_v = want_kv ? gv.data_ptr() : nullptr;
    const at::Tensor ws = scratch(texb_attention_workspace_bytes(p.n, p.heads, p.kv_heads, 1), q);
    check_status(texb_attention_backward(&p, ws.data_ptr(), size_t(ws.numel()), stream_of(q)), "texb_attention_backward");
    torch::autograd::variable_list r(12);
    r[0] = gq;
    r[1] = gk;
    r[2] = gv;
    return r;
  }
};

c10::optional<at::Tensor> given(const at::Tensor& t) { return t.defined() ? c10::make_optional(t) : c10::nullopt; }

at::Tensor segment_attention(const Plan& plan, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scale,
                             bool causal, double softcap, c10::optional<at::Tensor> slopes_given) {
  check_rows(q, "q", plan.sid, q);
  check_rows(k, "k", plan.sid, q);
  check_rows(v, "v", plan.sid, q);
  TORCH_CHECK(q.size(1) + k.size(1) <= 65535, "too many heads");
  TORCH_CHECK(k.size(1) == v.size(1), "k and v have different numbers of heads");
  TORCH_CHECK(q.size(1) >= 1 && k.size(1) >= 1 && q.size(1) % k.size(1) == 0, q.size(1), " query heads do not share ", k.size(1),
              " key / value heads evenly");
  TORCH_CHECK(q.size(2) >= 8 && q.size(2) <= kMaxDim && q.size(2) % 8 == 0, "the head dimension must be a multiple of 8 up to ",
              kMaxDim, ", got ", q.size(2));
  TORCH_CHECK(softcap >= 0 && std::isfinite(softcap), "softcap must be finite and not negative, got ", softcap);
  TORCH_CHECK(softcap == 0 || float(softcap) > 0.f, "softcap ", softcap, " is out of the range of float32");
  TORCH_CHECK(std::isfinite(scale), "scale must be finite, got ", scale);
  at::Tensor slopes;
  if (slopes_given.has_value() && slopes_given->defined()) {
    TORCH_CHECK(slopes_given->dim() == 1 && slopes_given->size(0) == q.size(1), "slopes must hold one value per query head");
    TORCH_CHECK(slopes_given->device() == q.device(), "slopes and q live on different devices");
    TORCH_CHECK(!slopes_given->requires_grad() || !at::GradMode::is_enabled(), "slopes take no gradient: pass slopes.detach()");
    TEXB_CHECK_DTYPE((*slopes_given), at::kFloat);
    check_no_tangent(*slopes_given, "slopes");
    slopes = slopes_given->contiguous();
  }
  const Options o = {scale, softcap, causal, plan.num_segments, plan.max_cnt};
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return AttentionNode::apply(q, k, v, plan.sid, given(plan.perm), plan.offsets, given(slopes), scale, softcap, causal,
                                plan.num_segments, plan.max_cnt);
  return std::get<0>(forward(q, k, v, plan.sid, plan.perm, plan.offsets, slopes, o, false));
}

}  // namespace

void register_attention(py::module& m) {
  m.def("segment_attention", &segment_attention, py::arg("plan"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("scale"),
        py::arg("causal") = false, py::arg("softcap") = 0.0, py::arg("slopes") = c10::nullopt);
}

}  // namespace texb_binding
