// Gradients of the embedding lookup and of document attention as nodes of
// torch's graph in C++.
//
// A training step runs these once a layer, next to kernels of 10 to 100 us;
// a node written in Python adds about 60 us of host time to a forward and
// backward pass (the interpreter lock changes hands between threads), one in
// C++ about 20.
//
// The gradients have no gradient of their own: asking for a graph of them
// (create_graph) raises, and so does an input with a forward-mode tangent.  Saved inputs are checked for changes in place.
#include <torch/extension.h>
#include <limits>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/utils.h>

namespace dlx {

at::Tensor embed_sum_fwd_impl(at::TensorList ids, at::TensorList tables,
                              at::ArrayRef<double> scales);
std::vector<at::Tensor> embed_sum_bwd_impl(const at::Tensor& dy,
                                           at::TensorList ids,
                                           at::IntArrayRef rows,
                                           at::ArrayRef<double> scales);
void embed_check_grad(int64_t n, int64_t width, at::IntArrayRef rows);
std::tuple<at::Tensor, at::Tensor, at::Tensor> doc_attn_fwd_impl(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const at::Tensor& cu, const c10::optional<at::Tensor>& slopes,
    double scale, bool need_grad);
void doc_attn_bwd_impl(const at::Tensor& dout, const at::Tensor& q,
                       const at::Tensor& k, const at::Tensor& v,
                       const at::Tensor& o, const at::Tensor& lse,
                       const at::Tensor& low, const at::Tensor& cu,
                       const c10::optional<at::Tensor>& slopes, double scale,
                       at::Tensor dq, at::Tensor dk, at::Tensor dv);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using torch::autograd::tensor_list;

void refuse_graph(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name,
              ": its gradient has no gradient (create_graph)");
}

// A tangent that no formula here takes on would be lost without a word.
void refuse_tangent(const char* name, const at::Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), name,
                              ": no forward-mode gradient");
}

// What functional.embedding_sum checks elsewhere, for 4 us less of host time
void check_lookup(at::TensorList ids, at::TensorList tables,
                  at::ArrayRef<double> scales) {
  const size_t n = tables.size();
  TORCH_CHECK_VALUE(n >= 1 && n <= 4, "embedding_sum: 1 to 4 tables, got ", n);
  TORCH_CHECK_VALUE(ids.size() == n && scales.size() == n,
                    "embedding_sum: as many ids and scales as tables");
  const at::Tensor& w0 = tables[0];
  for (size_t j = 0; j < n; ++j) {
    const at::Tensor &i = ids[j], &w = tables[j];
    TORCH_CHECK_VALUE(
        i.scalar_type() == at::kInt || i.scalar_type() == at::kLong,
        "embedding_sum: ids are int32 or int64, got ", i.scalar_type());
    TORCH_CHECK_VALUE(i.sizes() == ids[0].sizes(),
                      "embedding_sum: the ids differ in shape");
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == w0.size(1) &&
                          w.scalar_type() == w0.scalar_type(),
                      "embedding_sum: tables are [rows, width], of one width "
                      "and type");
    TORCH_CHECK_VALUE(i.device() == w0.device() && w.device() == w0.device(),
                      "embedding_sum: ids and tables are on different devices");
    refuse_tangent("embedding_sum", w);
  }
}

// The same for document attention; borders as contiguous int32 (what lies
// outside is cut off like what lies outside the tokens), slopes as fp32.
std::pair<at::Tensor, c10::optional<at::Tensor>> attention_args(
    const char* name, const at::Tensor& q, int64_t heads, int64_t kv_heads,
    const at::Tensor& cu, const c10::optional<at::Tensor>& slopes,
    double scale) {
  TORCH_CHECK_VALUE(cu.dim() == 1 && cu.numel() >= 1 &&
                        (cu.scalar_type() == at::kInt ||
                         cu.scalar_type() == at::kLong),
                    name, ": cu_seqlens is a vector of int32 or int64");
  TORCH_CHECK_VALUE(kv_heads >= 1 && heads % kv_heads == 0, name,
                    ": query heads have to be a multiple of key heads, got ",
                    heads, " and ", kv_heads);
  TORCH_CHECK_VALUE(cu.device() == q.device(), name,
                    ": cu_seqlens is on another device");
  TORCH_CHECK_VALUE(scale >= 1e-30 && scale <= 1e30, name,
                    ": scale has to lie between 1e-30 and 1e30");
  at::AutoDispatchBelowADInplaceOrView below;
  c10::optional<at::Tensor> s;
  if (slopes) {
    TORCH_CHECK_VALUE(!slopes->requires_grad(), name,
                      ": slopes are constants, they get no gradient");
    TORCH_CHECK_VALUE(slopes->dim() == 1 && slopes->size(0) == heads &&
                          slopes->device() == q.device(),
                      name, ": slopes has one number a query head, on the same "
                      "device");
    refuse_tangent(name, *slopes);
    s = slopes->to(at::kFloat).contiguous();
  }
  if (cu.scalar_type() == at::kInt && cu.is_contiguous()) return {cu, s};
  return {cu.clamp(-1, std::numeric_limits<int>::max())
              .to(at::kInt).contiguous(), s};
}

at::Tensor lookup(at::TensorList ids, at::TensorList tables,
                  at::ArrayRef<double> scales) {
  auto y = embed_sum_fwd_impl(ids, tables, scales);
  auto shape = ids[0].sizes().vec();
  shape.push_back(tables[0].size(1));
  return y.view(shape);
}

// A Node of its own spares what Function keeps by name: 3000 tokens forward
// and backward 74 -> 72 us of host time, 16 tokens 70 -> 65.
struct EmbeddingSumBackward : Node {
  std::vector<SavedVariable> ids;
  std::vector<int64_t> rows;
  std::vector<double> scales;

  std::string name() const override { return "EmbeddingSumBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto& i : ids) i.reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    refuse_graph("embedding_sum");
    variable_list out(ids.size());
    const at::Tensor dy = grads[0];
    std::vector<at::Tensor> want;
    std::vector<int64_t> want_rows;
    std::vector<double> want_scales;
    for (size_t i = 0; i < ids.size(); ++i)
      if (task_should_compute_output(i)) {
        want.push_back(ids[i].unpack());
        want_rows.push_back(rows[i]);
        want_scales.push_back(scales[i]);
      }
    if (want.empty() || !dy.defined()) return out;
    // -1 in place of the tokens would be ambiguous for rows of no width
    const auto got =
        embed_sum_bwd_impl(dy.reshape({want[0].numel(), dy.size(-1)}), want,
                           want_rows, want_scales);
    for (size_t i = 0, k = 0; i < ids.size(); ++i)
      if (task_should_compute_output(i)) out[i] = got[k++];
    return out;
  }
};

struct DocAttention : Function<DocAttention> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q,
                            const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& cu,
                            const c10::optional<at::Tensor>& slopes,
                            double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [o, lse, low] = doc_attn_fwd_impl(q, k, v, cu, slopes, scale, true);
    ctx->save_for_backward(
        {q, k, v, o, lse, low, cu, slopes ? *slopes : at::Tensor()});
    ctx->saved_data["scale"] = scale;
    return o;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    refuse_graph("document_attention");
    tensor_list out(6);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    for (int i = 0; i < 3; ++i) out[i] = at::empty(s[i].sizes(), s[i].options());
    c10::optional<at::Tensor> slopes;
    if (s[7].defined()) slopes = s[7];
    doc_attn_bwd_impl(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6],
                      slopes, ctx->saved_data["scale"].toDouble(), out[0],
                      out[1], out[2]);
    return out;
  }
};

// The same on one projection's output [tokens, 3, heads, dim]: the gradient
// is written in its layout.
struct DocAttentionQKV : Function<DocAttentionQKV> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& qkv,
                            const at::Tensor& cu,
                            const c10::optional<at::Tensor>& slopes,
                            double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [o, lse, low] =
        doc_attn_fwd_impl(qkv.select(1, 0), qkv.select(1, 1), qkv.select(1, 2),
                          cu, slopes, scale, true);
    ctx->save_for_backward(
        {qkv, o, lse, low, cu, slopes ? *slopes : at::Tensor()});
    ctx->saved_data["scale"] = scale;
    return o;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    refuse_graph("document_attention_qkv");
    tensor_list out(4);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const auto& qkv = s[0];
    out[0] = at::empty(qkv.sizes(), qkv.options());
    c10::optional<at::Tensor> slopes;
    if (s[5].defined()) slopes = s[5];
    doc_attn_bwd_impl(grads[0], qkv.select(1, 0), qkv.select(1, 1),
                      qkv.select(1, 2), s[1], s[2], s[3], s[4], slopes,
                      ctx->saved_data["scale"].toDouble(), out[0].select(1, 0),
                      out[0].select(1, 1), out[0].select(1, 2));
    return out;
  }
};

bool wants_grad(at::TensorList ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto& t : ts)
    if (t.requires_grad()) return true;
  return false;
}

}  // namespace

// ids of one shape, tables [rows, width] -> [*shape, width]
at::Tensor embedding_sum(at::TensorList ids, at::TensorList tables,
                         at::ArrayRef<double> scales) {
  check_lookup(ids, tables, scales);
  std::shared_ptr<EmbeddingSumBackward> node;
  if (wants_grad(tables)) {
    std::vector<int64_t> wanted;
    for (const auto& w : tables)
      if (w.requires_grad()) wanted.push_back(w.size(0));
    embed_check_grad(ids[0].numel(), tables[0].size(1), wanted);
    node.reset(new EmbeddingSumBackward, torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(tables));
    for (const auto& i : ids) node->ids.emplace_back(i, false);
    for (const auto& w : tables) node->rows.push_back(w.size(0));
    node->scales = scales.vec();
  }
  at::Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    y = lookup(ids, tables, scales);
  }
  if (node) torch::autograd::set_history(y, node);
  return y;
}

at::Tensor doc_attention(const at::Tensor& q, const at::Tensor& k,
                         const at::Tensor& v, const at::Tensor& cu_in,
                         const c10::optional<at::Tensor>& slopes_in,
                         double scale) {
  TORCH_CHECK_VALUE(
      q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() &&
          k.size(0) == q.size(0) && k.size(2) == q.size(2),
      "document_attention: q is [tokens, heads, dim], k and v [tokens, "
      "kv_heads, dim], got ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type() &&
                        q.scalar_type() == v.scalar_type(),
                    "document_attention: q, k and v differ in type");
  const auto [cu, slopes] =
      attention_args("document_attention", q, q.size(1), k.size(1), cu_in,
                     slopes_in, scale);
  for (const auto* t : {&q, &k, &v}) refuse_tangent("document_attention", *t);
  if (wants_grad({q, k, v}))
    return DocAttention::apply(q, k, v, cu, slopes, scale);
  at::AutoDispatchBelowADInplaceOrView below;
  return std::get<0>(doc_attn_fwd_impl(q, k, v, cu, slopes, scale, false));
}

at::Tensor doc_attention_qkv(const at::Tensor& qkv, const at::Tensor& cu_in,
                             const c10::optional<at::Tensor>& slopes_in,
                             double scale) {
  TORCH_CHECK_VALUE(qkv.dim() == 4 && qkv.size(1) == 3,
                    "document_attention_qkv: [tokens, 3, heads, dim] expected, "
                    "got ", qkv.sizes());
  const auto [cu, slopes] =
      attention_args("document_attention_qkv", qkv, qkv.size(2), qkv.size(2),
                     cu_in, slopes_in, scale);
  refuse_tangent("document_attention_qkv", qkv);
  if (wants_grad({qkv})) return DocAttentionQKV::apply(qkv, cu, slopes, scale);
  at::AutoDispatchBelowADInplaceOrView below;
  return std::get<0>(doc_attn_fwd_impl(qkv.select(1, 0), qkv.select(1, 1),
                                       qkv.select(1, 2), cu, slopes, scale,
                                       false));
}

}  // namespace dlx
