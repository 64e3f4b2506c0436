// Differentiable operators of the torch layer: LayerNorm, embedding and varlen attention on packed ragged batches, each a
// C++ autograd function over the C ABI's forward pass (which keeps what the gradients need) and backward pass.  First
// derivatives only: differentiating a gradient raises.  Host validation, allocation through torch's caching allocator and
// launches on the current stream as in dispatch.cpp; nothing is kept between calls, so captured CUDA graphs share nothing.
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <unordered_set>
#include <vector>

#include "dispatch_common.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Passes a gradient computed with create_graph=True on to the graph, with an error in the place of its own derivative.
struct FirstOrderOnly : public torch::autograd::Function<FirstOrderOnly> {
  using Maybe = c10::optional<Tensor>;
  static Tensor forward(AutogradContext*, const Tensor& grad, const Maybe&, const Maybe&, const Maybe&, const Maybe&) { return grad.detach(); }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "nestedtensor_b200: the training operators have first derivatives only");
  }
};

c10::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt; }

// A leaf's gradient node belongs to the stream it was made on, and lives as long as any graph of that leaf.  In a capture, the engine
// would make that stream wait for the captured one; the default stream must not, and the process does not survive it.  The leaf may
// lie behind other nodes (views, projections): all that this pass will run from here on are looked at.
void refuse_capture_into_default_stream() {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  const auto* wanted = torch::autograd::get_current_graph_task_exec_info();  // (empty: every node)
  std::vector<torch::autograd::Node*> todo = {node.get()};
  std::unordered_set<torch::autograd::Node*> seen;
  while (!todo.empty()) {
    const auto* at = todo.back();
    todo.pop_back();
    for (const auto& edge : at->next_edges()) {
      if (!edge.is_valid() || !seen.insert(edge.function.get()).second) continue;
      if (wanted != nullptr && !wanted->empty()) {
        const auto it = wanted->find(edge.function.get());
        if (it == wanted->end() || !it->second.should_execute()) continue;
      }
      const auto stream = edge.function->stream();
      TORCH_CHECK(!stream || stream->device_type() != c10::DeviceType::CUDA || c10::cuda::CUDAStream(*stream).stream() != nullptr,
                  "nestedtensor_b200: a backward pass is being captured into a CUDA graph while an eager graph of the same leaves, made on the "
                  "default stream, is alive: drop it (its outputs, its loss) before the capture, or run it on another stream");
      todo.push_back(edge.function.get());
    }
  }
}

// Runs `compute` (the gradients) without recording it; with create_graph=True every result keeps its dependence on `deps`.
template <typename F>
variable_list first_order(const std::array<Tensor, 4>& deps, F&& compute) {
  refuse_capture_into_default_stream();
  const bool create_graph = at::GradMode::is_enabled();
  variable_list grads;
  {
    at::AutoGradMode no_grad(false);
    grads = compute();
  }
  if (create_graph)
    for (auto& g : grads)
      if (g.defined()) g = FirstOrderOnly::apply(g, maybe(deps[0]), maybe(deps[1]), maybe(deps[2]), maybe(deps[3]));
  return grads;
}

Tensor byte_workspace(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 16)}, like.options().dtype(at::kByte));
}

bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

void same_kind(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == like.scalar_type(), "nestedtensor_b200: ", name,
              " must be on the input's device and of its dtype");
}

// The rows of a ragged batch.  `sizes` holds the lengths in its first column; features >= 0: the rows are a packed matrix of that
// width, which the sizes of another nested tensor with the same lengths describe; -1: `sizes` are the tensor's own, and its
// trailing dimensions must be regular.
struct Rows {
  int64_t B, tokens, longest, features;  // features: elements of the last dimension (-1: no sequences to tell)
};

Rows make_rows(const Tensor& t, const Tensor& sizes, int64_t features, const char* name) {
  TORCH_CHECK(sizes.device().is_cpu() && sizes.scalar_type() == at::kLong && sizes.dim() == 2 && sizes.is_contiguous() &&
                  (sizes.size(1) >= 1 || sizes.size(0) == 0),
              "nestedtensor_b200: sizes must be a contiguous CPU int64 [B, tensor_dim] tensor");
  TORCH_CHECK(t.is_cuda(), "nestedtensor_b200: this operator needs a CUDA ", name, " (this build has no CPU implementation)");
  Rows r = {sizes.size(0), 0, 0, features};
  const int64_t* p = sizes.data_ptr<int64_t>();
  const int64_t td = sizes.size(1);
  int64_t numel = 0;
  for (int64_t b = 0; b < r.B; ++b) {
    const int64_t* s = p + b * td;
    TORCH_CHECK(s[0] >= 0, "nestedtensor_b200: negative size");
    r.tokens += s[0];
    r.longest = std::max(r.longest, s[0]);
    if (features < 0) {
      TORCH_CHECK(s[td - 1] == p[td - 1] || td == 1, name, "'s last dimension must be regular.");
      int64_t n = 1;
      for (int64_t j = 0; j < td; ++j) n *= s[j];
      numel += n;
    }
  }
  if (features < 0) {
    if (r.B > 0) r.features = td > 1 ? p[td - 1] : 1;
  } else {
    TORCH_CHECK(t.dim() >= 1 && t.size(0) == r.tokens, "nestedtensor_b200: ", name, " must have sum(L_i) rows");
    numel = t.numel();
  }
  TORCH_CHECK(t.numel() == numel, "nestedtensor_b200: buffer must have sum(numel) elements");
  return r;
}

// Elements per row of constituents (L_i, ...), where all rows have the same number and at least one; 0 otherwise.
int64_t row_elems(const Tensor& sizes) {
  TORCH_CHECK(sizes.device().is_cpu() && sizes.scalar_type() == at::kLong && sizes.dim() == 2 && sizes.is_contiguous(),
              "nestedtensor_b200: sizes must be a contiguous CPU int64 [B, tensor_dim] tensor");
  const int64_t B = sizes.size(0), td = sizes.size(1);
  const int64_t* p = sizes.data_ptr<int64_t>();
  int64_t width = 1;
  for (int64_t b = 0; b < B; ++b) {
    int64_t n = 1;
    for (int64_t j = 1; j < td; ++j) n *= p[b * td + j];
    if (b == 0) width = n;
    if (n != width || n < 1) return 0;
  }
  return width;
}

void check_meta(const Tensor& meta, int64_t row_elems, int64_t B, const Tensor& like) {
  TORCH_CHECK(meta.is_cuda() && meta.device() == like.device() && meta.scalar_type() == at::kLong && meta.is_contiguous() && meta.numel() >= B + 1,
              "nestedtensor_b200: meta must be a CUDA int64 tensor that begins with B+1 offsets, on the input's device");
  TORCH_CHECK(row_elems >= 1 || B == 0, "nestedtensor_b200: row_elems must be at least 1");
}

// ------------------------------------------------------------------ LayerNorm
struct LayerNormTrain : public torch::autograd::Function<LayerNormTrain> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& weight, const c10::optional<Tensor>& bias,
                        int64_t cols, double eps) {
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.numel() / cols;
    Tensor out = at::empty({rows, cols}, x.options());
    Tensor stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    Tensor w, b;
    if (weight) w = weight->contiguous(), b = bias->contiguous();
    float* st = stats.data_ptr<float>();
    check_rc(ntb200_layer_norm_train(x.data_ptr(), w.defined() ? w.data_ptr() : nullptr, b.defined() ? b.data_ptr() : nullptr, (float)eps,
                                     out.data_ptr(), st, st + rows, rows, cols, dtype_code(x.scalar_type()), cur_stream()),
             "ntb200_layer_norm_train");
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["wants_x"] = wants(x);
    ctx->saved_data["wants_w"] = weight && wants(*weight);
    ctx->saved_data["wants_b"] = bias && wants(*bias);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    return first_order({grads[0], x, w, Tensor()}, [&]() -> variable_list {
      c10::cuda::CUDAGuard guard(x.device());
      const Tensor g = grads[0].contiguous();
      const int64_t rows = g.size(0), cols = g.size(1);
      const bool wx = ctx->saved_data["wants_x"].toBool(), ww = ctx->saved_data["wants_w"].toBool(), wb = ctx->saved_data["wants_b"].toBool();
      Tensor gx, gw, gb;
      if (wx) gx = at::empty(x.sizes(), x.options());
      if (ww) gw = at::empty({cols}, x.options());
      if (wb) gb = at::empty({cols}, x.options());
      const size_t bytes = w.defined() ? ntb200_layer_norm_backward_workspace_bytes(rows, cols) : 0;
      Tensor ws = byte_workspace(bytes, x);
      const float* st = stats.data_ptr<float>();
      check_rc(ntb200_layer_norm_backward(g.data_ptr(), x.data_ptr(), st, st + rows, w.defined() ? w.data_ptr() : nullptr,
                                          wx ? gx.data_ptr() : nullptr, ww ? gw.data_ptr() : nullptr, wb ? gb.data_ptr() : nullptr, rows, cols,
                                          dtype_code(x.scalar_type()), ws.data_ptr(), bytes, cur_stream()),
               "ntb200_layer_norm_backward");
      return {gx, gw, gb, Tensor(), Tensor()};
    });
  }
};

// LayerNorm over the last dimension of the packed rows; x is the buffer of the record, in any contiguous shape.  [T, E].
Tensor layer_norm_train(const Tensor& x_, const Tensor& sizes, int64_t features, at::IntArrayRef normalized_shape,
                        const c10::optional<Tensor>& weight, const c10::optional<Tensor>& bias, double eps) {
  TORCH_CHECK(normalized_shape.size() == 1, "Currently only singleton tuples of integers supported for layer_norm.");
  const int64_t E = normalized_shape[0];
  TORCH_CHECK(E > 0, "nestedtensor_b200: layer_norm over an empty dimension");
  TORCH_CHECK(features >= 0 || sizes.size(0) == 0 || sizes.size(1) > 1 ||
                  (sizes.numel() > 0 && (sizes == sizes[0][0]).all().item<bool>()),
              "Cannot normalize across irregular dimension 1");
  const Rows r = make_rows(x_, sizes, features, "input");
  const int64_t last = features < 0 && r.B > 0 && sizes.size(1) == 1 ? r.longest : r.features;
  TORCH_CHECK(last < 0 || last == E, "Normalized shape [", E, "] does not match the size of the last dimension (", last, ") of input.");
  dtype_code(x_.scalar_type());
  const bool has_w = weight && weight->defined(), has_b = bias && bias->defined();
  TORCH_CHECK(has_w == has_b, "Either both weight and bias are used or not.");
  if (has_w) {
    same_kind(*weight, x_, "weight");
    same_kind(*bias, x_, "bias");
    TORCH_CHECK(weight->dim() == 1 && weight->size(0) == E, "nestedtensor_b200: weight must have ", E, " entries");
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == E, "nestedtensor_b200: bias must have ", E, " entries");
  }
  TORCH_CHECK(eps >= 0, "nestedtensor_b200: eps must not be negative");
  return LayerNormTrain::apply(x_.contiguous(), has_w ? weight : c10::nullopt, has_b ? bias : c10::nullopt, E, eps);
}

// ------------------------------------------------------------------ embedding
struct EmbeddingTrain : public torch::autograd::Function<EmbeddingTrain> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& index, int64_t padding_idx, double scale) {
    c10::cuda::CUDAGuard guard(weight.device());
    Tensor w = weight.contiguous();
    const int64_t T = index.numel(), V = w.size(0), E = w.size(1);
    Tensor out = at::empty({T, E}, w.options());
    if (scale == 1.0)  // rows copied bit for bit
      check_rc(ntb200_embedding(w.data_ptr(), index.data_ptr(), (int)index.element_size(), out.data_ptr(), T, V, E, (int)w.element_size(),
                                cur_stream()),
               "ntb200_embedding");
    else
      check_rc(ntb200_embedding_scaled(w.data_ptr(), index.data_ptr(), (int)index.element_size(), out.data_ptr(), T, V, E, (float)scale,
                                       dtype_code(w.scalar_type()), cur_stream()),
               "ntb200_embedding_scaled");
    ctx->save_for_backward({index});
    ctx->saved_data["padding_idx"] = padding_idx;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["vocab"] = V;
    maybe_check_device_errors("embedding");
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor index = ctx->get_saved_variables()[0];
    return first_order({grads[0], Tensor(), Tensor(), Tensor()}, [&]() -> variable_list {
      c10::cuda::CUDAGuard guard(index.device());
      const Tensor g = grads[0].contiguous();
      const int64_t T = g.size(0), E = g.size(1), V = ctx->saved_data["vocab"].toInt();
      Tensor gw = at::empty({V, E}, g.options());
      const size_t bytes = ntb200_embedding_backward_workspace_bytes(T, E);
      Tensor ws = byte_workspace(bytes, g);
      check_rc(ntb200_embedding_backward(g.data_ptr(), index.data_ptr(), (int)index.element_size(), gw.data_ptr(), T, V, E,
                                         ctx->saved_data["padding_idx"].toInt(), (float)ctx->saved_data["scale"].toDouble(),
                                         dtype_code(g.scalar_type()), ws.data_ptr(), bytes, cur_stream()),
               "ntb200_embedding_backward");
      return {gw, Tensor(), Tensor(), Tensor()};
    });
  }
};

// scale * weight[index] for the packed index buffer of 1-D sequences: [T, E]
Tensor embedding_train(const Tensor& weight, const Tensor& index, const Tensor& sizes, c10::optional<int64_t> padding_idx, double scale) {
  TORCH_CHECK(weight.is_cuda() && weight.dim() == 2, "nestedtensor_b200: embedding needs a 2-D CUDA weight");
  dtype_code(weight.scalar_type());
  TORCH_CHECK(index.is_cuda() && index.device() == weight.device() && index.dim() == 1 && index.is_contiguous(),
              "nestedtensor_b200: the index buffer must be 1-D contiguous on the weight's device");
  TORCH_CHECK(index.scalar_type() == at::kLong || index.scalar_type() == at::kInt,
              "Expected tensor for argument #1 'indices' to have one of the following scalar types: Long, Int");
  TORCH_CHECK(sizes.device().is_cpu() && sizes.scalar_type() == at::kLong && sizes.dim() == 2 && (sizes.size(1) == 1 || sizes.size(0) == 0),
              "nestedtensor_b200: embedding expects a nested tensor of 1-D index sequences");
  make_rows(index, sizes, -1, "index tensor");
  const int64_t V = weight.size(0);
  TORCH_CHECK(V > 0 || index.numel() == 0, "nestedtensor_b200: embedding needs a weight with at least one row");
  TORCH_CHECK(V < (1ll << 31) - 1 && index.numel() < (1ll << 31) - 1, "nestedtensor_b200: embedding supports fewer than 2^31 - 1 rows and tokens");
  int64_t pad = -1;
  if (padding_idx) {
    TORCH_CHECK(*padding_idx >= -V && *padding_idx < V, "padding_idx must be within num_embeddings");
    pad = *padding_idx < 0 ? *padding_idx + V : *padding_idx;
  }
  return EmbeddingTrain::apply(weight, index, pad, scale);
}

// ------------------------------------------------------------------ attention
struct AttentionShape {
  int64_t B, Tq, Tk, longest_q, longest_k, row_q, row_k, H, d;
  double scaling;
};

void attention_forward(const AttentionShape& s, const void* q, const void* k, const void* v, int64_t ldq, int64_t ldkv, const Tensor& meta_q,
                       const Tensor& meta_k, Tensor& out, Tensor& lse) {
  const int dt = dtype_code(out.scalar_type());
  const size_t bytes = ntb200_varlen_attention_train_workspace_bytes(s.B, s.Tq, (int)s.H, (int)s.d, dt);
  Tensor ws = byte_workspace(bytes, out);
  check_rc(ntb200_varlen_attention_train(q, ldq, k, ldkv, v, ldkv, out.data_ptr(), lse.data_ptr<float>(), meta_q.data_ptr<int64_t>(), s.row_q,
                                         meta_k.data_ptr<int64_t>(), s.row_k, s.B, s.Tq, s.Tk, (int)s.H, (int)s.d, s.longest_q,
                                         (float)s.scaling, dt, 0, ws.data_ptr(), bytes, cur_stream()),
           "ntb200_varlen_attention_train");
  maybe_check_device_errors("attention");
}

void attention_backward(const AttentionShape& s, const Tensor& grad, const void* q, const void* k, const void* v, int64_t ldq, int64_t ldkv,
                        const Tensor& out, const Tensor& lse, void* dq, void* dk, void* dv, const Tensor& meta_q, const Tensor& meta_k) {
  const int dt = dtype_code(out.scalar_type());
  const size_t bytes = ntb200_varlen_attention_backward_workspace_bytes(s.B, s.Tq, s.Tk, (int)s.H, (int)s.d, s.longest_q, s.longest_k, dt, 0);
  Tensor ws = byte_workspace(bytes, out);
  check_rc(ntb200_varlen_attention_backward(grad.data_ptr(), q, ldq, k, ldkv, v, ldkv, out.data_ptr(), lse.data_ptr<float>(), dq, ldq, dk, ldkv,
                                            dv, ldkv, meta_q.data_ptr<int64_t>(), s.row_q, meta_k.data_ptr<int64_t>(), s.row_k, s.B, s.Tq, s.Tk,
                                            (int)s.H, (int)s.d, s.longest_q, s.longest_k, (float)s.scaling, dt, 0, ws.data_ptr(), bytes,
                                            cur_stream()),
           "ntb200_varlen_attention_backward");
  maybe_check_device_errors("attention backward");
}

void save_shape(AutogradContext* ctx, const AttentionShape& s) {
  ctx->saved_data["shape"] = std::vector<int64_t>{s.B, s.Tq, s.Tk, s.longest_q, s.longest_k, s.row_q, s.row_k, s.H, s.d};
  ctx->saved_data["scaling"] = s.scaling;
}

AttentionShape load_shape(AutogradContext* ctx) {
  const auto v = ctx->saved_data["shape"].toIntVector();
  return {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], ctx->saved_data["scaling"].toDouble()};
}

// q | k | v of every token in one [T, 3E] matrix; the gradient has the same form
struct SelfAttentionTrain : public torch::autograd::Function<SelfAttentionTrain> {
  static const void* part(const Tensor& t, int64_t elems) { return static_cast<const char*>(t.data_ptr()) + elems * t.element_size(); }
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& meta, const AttentionShape& s) {
    c10::cuda::CUDAGuard guard(qkv.device());
    const int64_t E = s.H * s.d;
    Tensor out = at::empty({s.Tq, E}, qkv.options()), lse = at::empty({s.H, s.Tq}, qkv.options().dtype(at::kFloat));
    if (s.Tq > 0) attention_forward(s, qkv.data_ptr(), part(qkv, E), part(qkv, 2 * E), 3 * E, 3 * E, meta, meta, out, lse);
    ctx->save_for_backward({qkv, meta, out, lse});
    save_shape(ctx, s);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &qkv = saved[0], &meta = saved[1], &out = saved[2], &lse = saved[3];
    return first_order({grads[0], qkv, Tensor(), Tensor()}, [&]() -> variable_list {
      c10::cuda::CUDAGuard guard(qkv.device());
      const AttentionShape s = load_shape(ctx);
      const int64_t E = s.H * s.d;
      const Tensor g = grads[0].contiguous();
      Tensor dqkv = at::empty(qkv.sizes(), qkv.options());
      if (s.Tq > 0)
        attention_backward(s, g, qkv.data_ptr(), part(qkv, E), part(qkv, 2 * E), 3 * E, 3 * E, out, lse, dqkv.data_ptr(),
                           const_cast<void*>(part(dqkv, E)), const_cast<void*>(part(dqkv, 2 * E)), meta, meta);
      return {dqkv, Tensor(), Tensor()};
    });
  }
};

struct AttentionTrain : public torch::autograd::Function<AttentionTrain> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& meta_q, const Tensor& meta_k,
                        const AttentionShape& s) {
    c10::cuda::CUDAGuard guard(q.device());
    const int64_t E = s.H * s.d;
    Tensor out = at::empty({s.Tq, E}, q.options()), lse = at::empty({s.H, s.Tq}, q.options().dtype(at::kFloat));
    if (s.Tq > 0) attention_forward(s, q.data_ptr(), k.data_ptr(), v.data_ptr(), E, E, meta_q, meta_k, out, lse);
    ctx->save_for_backward({q, k, v, meta_q, meta_k, out, lse});
    save_shape(ctx, s);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &meta_q = saved[3], &meta_k = saved[4], &out = saved[5], &lse = saved[6];
    return first_order({grads[0], q, k, v}, [&]() -> variable_list {
      c10::cuda::CUDAGuard guard(q.device());
      const AttentionShape s = load_shape(ctx);
      const int64_t E = s.H * s.d;
      const Tensor g = grads[0].contiguous();
      Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
      if (s.Tq > 0 || s.Tk > 0)
        attention_backward(s, g, q.data_ptr(), k.data_ptr(), v.data_ptr(), E, E, out, lse, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), meta_q,
                           meta_k);
      return {dq, dk, dv, Tensor(), Tensor(), Tensor()};
    });
  }
};

int64_t check_heads(int64_t num_heads, int64_t E) {
  TORCH_CHECK(num_heads >= 1 && E >= num_heads && E % num_heads == 0, "embed_dim must be divisible by num_heads");
  TORCH_CHECK(E / num_heads <= 256, "nestedtensor_b200: head_dim must be in [1, 256]");
  return E / num_heads;
}

double scaling_or_default(c10::optional<double> scaling, int64_t d) {
  if (!scaling) return 1.0 / std::sqrt((double)d);
  TORCH_CHECK(std::isfinite((float)*scaling * 1.4426950408889634f), "nestedtensor_b200: scaling must be finite in 32 bits, got ", *scaling);
  return *scaling;
}

// Self-attention of packed q|k|v rows: qkv is the buffer of (L_i, 3E) constituents in any contiguous shape; [T, E].
Tensor self_attention_train(const Tensor& qkv, const Tensor& sizes, int64_t features, const Tensor& meta, int64_t row_elems, int64_t num_heads,
                            c10::optional<double> scaling) {
  dtype_code(qkv.scalar_type());
  const Rows r = make_rows(qkv, sizes, features, "nested tensor");
  check_meta(meta, row_elems, r.B, qkv);
  const int64_t F = r.features < 0 ? 3 * num_heads : r.features;
  TORCH_CHECK(F % 3 == 0 && qkv.numel() == r.tokens * F, "nestedtensor_b200: self_attention expects (L_i, 3 * embed_dim) constituents");
  const int64_t d = check_heads(num_heads, F / 3);
  const AttentionShape s = {r.B, r.tokens, r.tokens, r.longest, r.longest, row_elems, row_elems, num_heads, d, scaling_or_default(scaling, d)};
  return SelfAttentionTrain::apply(qkv.contiguous(), meta, s);
}

// Attention of the queries of sequence b over the keys and values of sequence b: buffers of (L_i, E) constituents; [Tq, E].
Tensor attention_train(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_sizes, int64_t q_features, const Tensor& q_meta,
                       int64_t q_row_elems, const Tensor& k_sizes, int64_t k_features, const Tensor& k_meta, int64_t k_row_elems,
                       int64_t num_heads, c10::optional<double> scaling) {
  dtype_code(q.scalar_type());
  const Rows rq = make_rows(q, q_sizes, q_features, "query");
  same_kind(k, q, "key");
  same_kind(v, q, "value");
  const Rows rk = make_rows(k, k_sizes, k_features, "key");
  check_meta(q_meta, q_row_elems, rq.B, q);
  check_meta(k_meta, k_row_elems, rk.B, q);
  TORCH_CHECK(rq.B == rk.B, "nestedtensor_b200: query and key must hold the same number of sequences");
  const int64_t E = rq.features < 0 ? num_heads : rq.features;
  TORCH_CHECK((rk.features < 0 || rk.features == E) && q.numel() == rq.tokens * E && k.numel() == rk.tokens * E && v.numel() == k.numel(),
              "nestedtensor_b200: query, key and value need the same last dimension and constituents of (L_i, embed_dim)");
  const int64_t d = check_heads(num_heads, E);
  const AttentionShape s = {rq.B, rq.tokens, rk.tokens, rq.longest, rk.longest, q_row_elems, k_row_elems, num_heads, d,
                            scaling_or_default(scaling, d)};
  return AttentionTrain::apply(q.contiguous(), k.contiguous(), v.contiguous(), q_meta, k_meta, s);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(nestedtensor, m) {
  m.def(
      "layer_norm_train(Tensor x, Tensor sizes, int features, int[] normalized_shape, Tensor? weight, Tensor? bias, float eps) -> Tensor",
      &layer_norm_train);
  m.def("row_elems(Tensor sizes) -> int", &row_elems);
  m.def("embedding_train(Tensor weight, Tensor index, Tensor sizes, int? padding_idx, float scale) -> Tensor", &embedding_train);
  m.def(
      "self_attention_train(Tensor qkv, Tensor sizes, int features, Tensor meta, int row_elems, int num_heads, float? scaling) -> Tensor",
      &self_attention_train);
  m.def(
      "attention_train(Tensor q, Tensor k, Tensor v, Tensor q_sizes, int q_features, Tensor q_meta, int q_row_elems, Tensor k_sizes, "
      "int k_features, Tensor k_meta, int k_row_elems, int num_heads, float? scaling) -> Tensor",
      &attention_train);
}
