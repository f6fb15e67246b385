// Torch-facing launchers of the language-model operators: embedding
// (kernels/embedding.hip), cross entropy (kernels/cross_entropy.hip) and the
// gradient norm (kernels/grad_norm.hip). They run on the tensors' device, on
// its current torch stream; scratch comes from torch's allocator per call.
//
// Each one that gives new tensors is an operator of torch's dispatcher
// (axon::...), its backward pass too. What records calls there (torch.jit.trace,
// make_fx, a profiler) or transforms them (vmap, torch.func) then sees the
// operator and its inputs; in a call that goes past the dispatcher it sees only
// how the output is allocated, and a trace of that returns memory that nothing
// wrote. The dispatcher costs a call about 0.1 us (a lookup 4.2 us).
#include <torch/extension.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/library.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <algorithm>
#include <mutex>

#include "kernels/grad_norm.h"
#include "kernels/kernels.h"

namespace axon {
namespace {

using Guard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

hipStream_t stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device())
      .stream();
}

int code_of(const at::Tensor& t) { return static_cast<int>(t.scalar_type()); }

bool float_type(at::ScalarType t) {
  return t == at::kFloat || t == at::kHalf || t == at::kBFloat16;
}

void check_launch() {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, "axon: kernel launch failed: ",
              hipGetErrorString(e));
}

// A gradient that must not be differentiated again: an error where that is
// tried, under torch's graph as under its function transforms.
template <typename... Inputs>
at::Tensor once(at::Tensor grad, const char* what, const Inputs&... inputs) {
  if (!torch::autograd::compute_requires_grad(inputs...)) return grad;
  auto node = std::shared_ptr<torch::autograd::Error>(
      new torch::autograd::Error(
          std::string(what) + ": the gradient is not differentiable again",
          torch::autograd::collect_next_edges(inputs...)),
      torch::autograd::deleteNode);
  torch::autograd::set_history(grad, node);
  return grad;
}

// Forward-mode tangents would be lost without a word.
void check_no_tangent(const at::Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), what,
                              ": no forward-mode derivative");
}

// What reads and writes the parameters' .grad is no function of its arguments.
void check_untraced(const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      !torch::jit::tracer::isTracing() &&
          !c10::impl::TorchDispatchModeTLS::get_mode(
               c10::impl::TorchDispatchModeKey::PROXY)
               .has_value(),
      what, ": cannot be traced");
}

// An operator of the dispatcher, by its name.
template <typename Signature>
c10::TypedOperatorHandle<Signature> op_of(const char* name) {
  return c10::Dispatcher::singleton()
      .findSchemaOrThrow(name, "")
      .typed<Signature>();
}

// The nodes below are written against torch's graph itself: a Python
// autograd.Function costs about 20 us for each pass through it, more than
// the kernels of a small batch.

// ------------------------------------------------------------- embedding

void check_embedding(const at::Tensor& ids, at::ScalarType type, int64_t vocab,
                     int64_t dim) {
  TORCH_CHECK_TYPE(ids.scalar_type() == at::kLong ||
                       ids.scalar_type() == at::kInt,
                   "embedding: ids must be int32 or int64, got ",
                   ids.scalar_type());
  TORCH_CHECK_TYPE(float_type(type),
                   "embedding: weight must be float, half or bfloat16");
  // A launch takes fewer than 2^32 threads, 64 for each token.
  TORCH_CHECK_VALUE(vocab < (int64_t{1} << 31) && dim < (int64_t{1} << 22) &&
                        ids.numel() < (int64_t{1} << 26),
                    "embedding: fewer than 2^31 rows, of fewer than 2^22 "
                    "values, and fewer than 2^26 ids");
}

at::Tensor embedding_kernel(const at::Tensor& ids_in,
                            const at::Tensor& weight_in, double scale,
                            c10::optional<int64_t> padding_idx) {
  TORCH_CHECK_VALUE(weight_in.dim() == 2, "embedding: weight must be [V, D], "
                    "got ", weight_in.sizes());
  const int64_t vocab = weight_in.size(0), dim = weight_in.size(1);
  TORCH_CHECK_VALUE(!padding_idx.has_value() ||
                        (*padding_idx >= -vocab && *padding_idx < vocab),
                    "embedding: padding_idx ", padding_idx.value_or(0),
                    " outside the ", vocab, " rows");
  TORCH_CHECK_VALUE(weight_in.is_cuda() && ids_in.device() == weight_in.device(),
                    "embedding: ids on ", ids_in.device(), ", weight on ",
                    weight_in.device());
  check_embedding(ids_in, weight_in.scalar_type(), vocab, dim);
  const Guard guard(weight_in.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const at::Tensor weight = dim > 1 && weight_in.stride(1) != 1
                                ? weight_in.contiguous()
                                : weight_in;
  const at::Tensor ids = ids_in.contiguous();
  auto shape = ids.sizes().vec();
  shape.push_back(dim);
  at::Tensor y = at::empty(shape, weight.options());
  if (y.numel()) {
    launch_embed_fwd(code_of(weight), ids.scalar_type() == at::kLong,
                     ids.data_ptr(), weight.data_ptr(), y.data_ptr(),
                     ids.numel(), vocab, dim, weight.stride(0),
                     static_cast<float>(scale), stream_of(weight));
    check_launch();
  }
  return y;
}

// padding: the row without a gradient, or -1.
at::Tensor embedding_backward_kernel(const at::Tensor& ids_in,
                                     const at::Tensor& dy_in, int64_t vocab,
                                     int64_t padding, double scale) {
  TORCH_CHECK_VALUE(dy_in.is_cuda() && ids_in.device() == dy_in.device() &&
                        dy_in.dim() == ids_in.dim() + 1 && vocab >= 0 &&
                        dy_in.sizes().slice(0, ids_in.dim()) == ids_in.sizes(),
                    "embedding: ids ", ids_in.sizes(), " and gradient ",
                    dy_in.sizes());
  const int64_t n = ids_in.numel(), dim = dy_in.size(-1);
  check_embedding(ids_in, dy_in.scalar_type(), vocab, dim);
  const Guard guard(dy_in.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const at::Tensor dy = dy_in.contiguous(), ids = ids_in.contiguous();
  // Whole units of 16 bytes, as the kernels fill it.
  const int64_t unit = 16 / static_cast<int64_t>(dy.element_size());
  at::Tensor dw =
      at::empty({(vocab * dim + unit - 1) / unit * unit}, dy.options());
  if (dw.numel() == 0) return dw.view({vocab, dim});
  dw = dw.as_strided({vocab, dim}, {dim, 1});
  // Keys, twice, and partial sums.
  const int64_t parts =
      embed_part_floats(n, dim, static_cast<int>(dy.element_size()));
  at::Tensor scratch =
      at::empty({4 * n + parts}, dy.options().dtype(at::kFloat));
  float* const part = scratch.data_ptr<float>() + 4 * n;
  launch_embed_bwd(code_of(dy), ids.scalar_type() == at::kLong, ids.data_ptr(),
                   dy.data_ptr(), dw.data_ptr(),
                   reinterpret_cast<uint64_t*>(scratch.data_ptr()), part, n,
                   vocab, dim, padding, static_cast<float>(scale),
                   stream_of(dy));
  check_launch();
  return dw;
}

at::Tensor embedding_backward(const at::Tensor& ids, const at::Tensor& dy,
                              int64_t vocab, int64_t padding, double scale) {
  static const auto op = op_of<decltype(embedding_backward_kernel)>(
      "axon::embedding_backward");
  return op.call(ids, dy, vocab, padding, scale);
}

at::Tensor embedding_backward_autograd(const at::Tensor& ids,
                                       const at::Tensor& dy, int64_t vocab,
                                       int64_t padding, double scale) {
  check_no_tangent(dy, "embedding");
  at::Tensor dw;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    dw = embedding_backward(ids, dy, vocab, padding, scale);
  }
  return once(dw, "embedding", dy);
}

struct EmbeddingBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable ids;
  int64_t vocab = 0, padding = -1;
  double scale = 1.0;

  torch::autograd::variable_list apply(
      torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const at::Tensor i = ids.unpack(shared_from_this());
    if (!grads[0].defined()) return {at::Tensor()};
    return {embedding_backward(i, grads[0], vocab, padding, scale)};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    ids.reset_data();
  }
  std::string name() const override { return "AxonEmbeddingBackward"; }
};

at::Tensor embedding(const at::Tensor& ids, const at::Tensor& weight,
                     double scale, c10::optional<int64_t> padding_idx) {
  static const auto op = op_of<decltype(embedding_kernel)>("axon::embedding");
  return op.call(ids, weight, scale, padding_idx);
}

at::Tensor embedding_autograd(const at::Tensor& ids, const at::Tensor& weight,
                              double scale,
                              c10::optional<int64_t> padding_idx) {
  check_no_tangent(weight, "embedding");
  at::Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    y = embedding(ids, weight, scale, padding_idx);
  }
  if (!torch::autograd::compute_requires_grad(weight)) return y;
  auto node = std::shared_ptr<EmbeddingBackward>(new EmbeddingBackward(),
                                                 torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(weight));
  node->ids = torch::autograd::SavedVariable(ids, false);
  node->vocab = weight.size(0);
  const int64_t row = padding_idx.value_or(-1);
  node->padding = padding_idx.has_value() && row < 0 ? row + node->vocab : row;
  node->scale = scale;
  torch::autograd::set_history(y, node);
  return y;
}

// --------------------------------------------------------- cross entropy

struct LogitRows {
  int64_t n, vocab, inner, stride_outer, stride_inner;
};

// Logits [V], [N, V] or [B, S, V] with a dense last dimension; the others may
// have any strides.
LogitRows logit_rows(const at::Tensor& x, const at::Tensor& target) {
  LogitRows r;
  r.vocab = x.size(-1);
  r.n = target.numel();
  r.inner = x.dim() == 1 ? 1 : std::max<int64_t>(1, x.size(-2));
  r.stride_inner = x.dim() == 1 ? 0 : x.stride(-2);
  r.stride_outer = x.dim() == 3 ? x.stride(0) : 0;
  return r;
}

void check_cross_entropy(const at::Tensor& logits, const at::Tensor& target,
                         double eps, int64_t reduction) {
  TORCH_CHECK_VALUE(reduction >= 0 && reduction <= 2,
                    "cross_entropy: reduction ", reduction);
  TORCH_CHECK_VALUE(eps >= 0.0 && eps <= 1.0,
                    "cross_entropy: label_smoothing outside [0, 1]: ", eps);
  TORCH_CHECK_TYPE(target.scalar_type() == at::kLong ||
                       target.scalar_type() == at::kInt,
                   "cross_entropy: target must hold class numbers (int32 or "
                   "int64), got ", target.scalar_type());
  TORCH_CHECK_VALUE(
      logits.dim() >= 1 && logits.size(-1) > 0 &&
          target.sizes() == logits.sizes().slice(0, logits.dim() - 1),
      "cross_entropy: logits ", logits.sizes(), " and target ",
      target.sizes(), ": one label for each row of classes");
  TORCH_CHECK_VALUE(logits.is_cuda() && target.device() == logits.device(),
                    "cross_entropy: target on ", target.device(),
                    ", logits on ", logits.device());
  TORCH_CHECK_TYPE(float_type(logits.scalar_type()),
                   "cross_entropy: logits must be float, half or bfloat16");
  // Places within a row are counted in 32 bits.
  TORCH_CHECK_VALUE(logits.size(-1) < (int64_t{1} << 30),
                    "cross_entropy: fewer than 2^30 classes");
  const int64_t most = ce_max_rows(code_of(logits), logits.size(-1));
  TORCH_CHECK_VALUE(target.numel() <= most, "cross_entropy: at most ", most,
                    " rows of ", logits.size(-1), " classes");
}

// The logits and labels as the kernels take them.
std::pair<at::Tensor, at::Tensor> dense_rows(const at::Tensor& logits,
                                             const at::Tensor& target) {
  at::Tensor x = logits, t = target;
  if (x.size(-1) > 1 && x.stride(-1) != 1) x = x.contiguous();
  if (x.dim() > 3) {
    x = x.flatten(0, -3);
    t = t.flatten(0, -2);
  }
  if (t.scalar_type() != at::kLong) t = t.to(at::kLong);
  return {x, t.contiguous()};
}

// Scratch of the forward pass, in floats (whole doubles).
int64_t scratch_floats(const at::Tensor& x, const LogitRows& r) {
  return (ce_scratch_bytes(code_of(x), r.n, r.vocab) + 7) / 8 * 2;
}

// The loss, and what the backward pass takes: behind the scratch, a row's
// (m, 1/S), and the factor at its end. reduction: 0 none, 1 mean, 2 sum.
std::tuple<at::Tensor, at::Tensor> cross_entropy_kernel(
    const at::Tensor& logits, const at::Tensor& target, int64_t ignore,
    double eps, int64_t reduction) {
  check_cross_entropy(logits, target, eps, reduction);
  const Guard guard(logits.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const auto [x, t] = dense_rows(logits, target);
  const LogitRows r = logit_rows(x, t);
  const auto fopt = x.options().dtype(at::kFloat);
  // The loss, which its user may change in place, is memory of its own.
  at::Tensor loss = reduction == 0 ? at::empty(target.sizes(), fopt)
                                   : at::empty({}, fopt);
  const int64_t scratch = scratch_floats(x, r);
  at::Tensor work = at::empty({scratch + 2 * r.n + 1}, fopt);
  float* const kept = work.data_ptr<float>() + scratch;
  launch_ce_fwd(code_of(x), x.data_ptr(), r.inner, r.stride_outer,
                r.stride_inner, t.data_ptr<int64_t>(), ignore, r.n, r.vocab,
                static_cast<float>(eps), static_cast<int>(reduction),
                work.data_ptr(), kept, loss.data_ptr<float>(), kept + 2 * r.n,
                stream_of(x));
  check_launch();
  return {loss, work};
}

at::Tensor cross_entropy_backward_kernel(
    const at::Tensor& grad, const at::Tensor& logits, const at::Tensor& target,
    const at::Tensor& kept, int64_t ignore, double eps, int64_t reduction) {
  check_cross_entropy(logits, target, eps, reduction);
  const Guard guard(logits.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const auto [x, t] = dense_rows(logits, target);
  const LogitRows r = logit_rows(x, t);
  const at::Tensor g = grad.contiguous();
  const int64_t scratch = scratch_floats(x, r);
  for (const at::Tensor* f : {&g, &kept})
    TORCH_CHECK(f->device() == x.device() && f->scalar_type() == at::kFloat,
                "cross_entropy: the loss's gradient");
  TORCH_CHECK(g.numel() == (reduction == 0 ? r.n : 1) &&
                  kept.is_contiguous() &&
                  kept.numel() == scratch + 2 * r.n + 1,
              "cross_entropy: the loss's gradient");
  at::Tensor dx = at::empty(logits.sizes(), x.options());
  if (r.n > 0) {
    const float* const k = kept.data_ptr<float>() + scratch;
    launch_ce_bwd(code_of(x), x.data_ptr(), r.inner, r.stride_outer,
                  r.stride_inner, t.data_ptr<int64_t>(), ignore, r.n, r.vocab,
                  static_cast<float>(eps), k, g.data_ptr<float>(),
                  reduction == 0 ? 1 : 0,
                  reduction == 0 ? nullptr : k + 2 * r.n, dx.data_ptr(),
                  stream_of(x));
    check_launch();
  }
  return dx;
}

at::Tensor cross_entropy_backward(const at::Tensor& grad,
                                  const at::Tensor& logits,
                                  const at::Tensor& target,
                                  const at::Tensor& kept, int64_t ignore,
                                  double eps, int64_t reduction) {
  static const auto op = op_of<decltype(cross_entropy_backward_kernel)>(
      "axon::cross_entropy_backward");
  return op.call(grad, logits, target, kept, ignore, eps, reduction);
}

at::Tensor cross_entropy_backward_autograd(
    const at::Tensor& grad, const at::Tensor& logits, const at::Tensor& target,
    const at::Tensor& kept, int64_t ignore, double eps, int64_t reduction) {
  for (const at::Tensor* t : {&grad, &logits})
    check_no_tangent(*t, "cross_entropy");
  at::Tensor dx;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    dx = cross_entropy_backward(grad, logits, target, kept, ignore, eps,
                                reduction);
  }
  return once(dx, "cross_entropy", grad, logits);
}

struct CrossEntropyBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable logits, target;
  at::Tensor kept;  // of this file alone
  int64_t ignore = 0;
  double eps = 0.0;
  int64_t reduction = 1;

  torch::autograd::variable_list apply(
      torch::autograd::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const at::Tensor x = logits.unpack(), t = target.unpack();
    if (!grads[0].defined()) return {at::Tensor()};
    return {cross_entropy_backward(grads[0], x, t, kept, ignore, eps,
                                   reduction)};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    logits.reset_data();
    target.reset_data();
    kept.reset();
  }
  std::string name() const override { return "AxonCrossEntropyBackward"; }
};

std::tuple<at::Tensor, at::Tensor> call_cross_entropy(
    const at::Tensor& logits, const at::Tensor& target, int64_t ignore,
    double eps, int64_t reduction) {
  static const auto op =
      op_of<decltype(cross_entropy_kernel)>("axon::cross_entropy");
  return op.call(logits, target, ignore, eps, reduction);
}

std::tuple<at::Tensor, at::Tensor> cross_entropy_autograd(
    const at::Tensor& logits, const at::Tensor& target, int64_t ignore,
    double eps, int64_t reduction) {
  check_no_tangent(logits, "cross_entropy");
  if (!torch::autograd::compute_requires_grad(logits)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_cross_entropy(logits, target, ignore, eps, reduction);
  }
  check_cross_entropy(logits, target, eps, reduction);
  // With the caller's autograd: the gradient goes back through these, and the
  // backward pass has them as the kernels take them.
  const auto [x, t] = dense_rows(logits, target);
  at::Tensor loss, kept;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    std::tie(loss, kept) = call_cross_entropy(x, t, ignore, eps, reduction);
  }
  auto node = std::shared_ptr<CrossEntropyBackward>(
      new CrossEntropyBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x));
  node->logits = torch::autograd::SavedVariable(x, false);
  node->target = torch::autograd::SavedVariable(t, false);
  node->kept = kept;
  node->ignore = ignore;
  node->eps = eps;
  node->reduction = reduction;
  torch::autograd::set_history(loss, node);
  if (reduction == 0 && logits.dim() > 3) loss = loss.view(target.sizes());
  return {loss, kept};
}

at::Tensor cross_entropy(const at::Tensor& logits, const at::Tensor& target,
                         int64_t ignore, double eps,
                         const std::string& reduction_name) {
  const int reduction = reduction_name == "none"   ? 0
                        : reduction_name == "mean" ? 1
                        : reduction_name == "sum"  ? 2
                                                   : -1;
  TORCH_CHECK_VALUE(reduction >= 0, "cross_entropy: reduction '",
                    reduction_name, "', expected 'none', 'mean' or 'sum'");
  return std::get<0>(
      call_cross_entropy(logits, target, ignore, eps, reduction));
}

// ---------------------------------------------------------- gradient norm

// The tensors as one list for the kernels: each buffer once (a tensor given
// twice counts once and is scaled once), and dense (a strided one goes
// through a dense copy).
struct Grads {
  std::vector<at::Tensor> dense;
  std::vector<std::pair<at::Tensor, size_t>> strided;  // original, its copy
};

Grads collect(at::TensorList ts, bool written) {
  Grads g;
  TORCH_CHECK_VALUE(!ts.empty(), "grad norm: no tensors");
  for (const at::Tensor& t : ts)
    TORCH_CHECK_VALUE(t.is_cuda() && t.layout() == at::kStrided &&
                          float_type(t.scalar_type()) && t.device() == ts[0].device(),
                      "grad norm: tensors must be dense float/half/bfloat16 "
                      "on one GPU");
  // By address: equal tensors are neighbours then (of those that start at one
  // place, few as they are, each is compared with each).
  std::vector<std::pair<const char*, size_t>> order;
  order.reserve(ts.size());
  for (size_t i = 0; i < ts.size(); ++i)
    if (ts[i].numel())
      order.emplace_back(static_cast<const char*>(ts[i].data_ptr()), i);
  std::sort(order.begin(), order.end());
  std::vector<char> skip(ts.size(), 0);
  const char* dense_end = nullptr;
  for (size_t k = 0, same = 0; k < order.size(); ++k) {
    const at::Tensor& t = ts[order[k].second];
    if (order[k].first != order[same].first) same = k;
    for (size_t j = same; j < k && !skip[order[k].second]; ++j) {
      const at::Tensor& o = ts[order[j].second];
      skip[order[k].second] = o.sizes() == t.sizes() &&
                              o.strides() == t.strides() &&
                              o.scalar_type() == t.scalar_type();
    }
    if (skip[order[k].second] || !written) continue;
    if (!t.is_non_overlapping_and_dense()) {
      at::assert_no_internal_overlap(t);
      continue;
    }
    // Two blocks would scale the same value. (A strided tensor's copy holds
    // the values from before; writing it back gives the same ones.)
    TORCH_CHECK_VALUE(order[k].first >= dense_end,
                      "grad norm: gradients share memory in part");
    dense_end = order[k].first + t.nbytes();
  }
  g.dense.reserve(ts.size());
  for (size_t i = 0; i < ts.size(); ++i) {
    const at::Tensor& t = ts[i];
    if (!t.numel() || skip[i]) continue;
    if (t.is_non_overlapping_and_dense()) {
      g.dense.push_back(t);
    } else {
      g.strided.emplace_back(t, g.dense.size());
      g.dense.push_back(t.contiguous());
    }
  }
  return g;
}

struct Table {
  GradTable t;
  int dtype;
};

// Tables that cover all tensors, one type each.
std::vector<Table> tables_of(const std::vector<at::Tensor>& ts) {
  std::vector<Table> tables;
  for (auto type : {at::kFloat, at::kHalf, at::kBFloat16}) {
    GradTable* t = nullptr;
    for (const at::Tensor& x : ts) {
      if (x.scalar_type() != type) continue;
      const int64_t chunks = (x.numel() + kGradChunk - 1) / kGradChunk;
      TORCH_CHECK(chunks < (int64_t{1} << 30), "grad norm: tensor too large");
      if (!t || t->count == kGradTensors ||
          t->first[t->count] + chunks >= (int64_t{1} << 30)) {
        tables.emplace_back();
        tables.back().dtype = static_cast<int>(type);
        t = &tables.back().t;
        t->count = 0;
        t->first[0] = 0;
      }
      t->ptr[t->count] = x.data_ptr();
      t->n[t->count] = x.numel();
      t->first[t->count + 1] = t->first[t->count] + static_cast<int32_t>(chunks);
      ++t->count;
    }
  }
  return tables;
}

// Strided tensors get their scaled copies; autograd learns that the others
// were written to.
void write_back(const Grads& g) {
  size_t next = 0;
  for (size_t i = 0; i < g.dense.size(); ++i) {
    if (next < g.strided.size() && g.strided[next].second == i)
      g.strided[next++].first.copy_(g.dense[i]);
    else if (!g.dense[i].is_inference())
      g.dense[i].unsafeGetTensorImpl()->bump_version();
  }
}

// (norm, factor) as fp32[2], and the tensors scaled by the factor if `clip`;
// type 0 is the maximum.
at::Tensor norm_of(at::TensorList ts, int64_t type, double max_norm,
                   bool clip) {
  TORCH_CHECK(type >= 0 && type <= 2, "grad norm: type");
  const Grads g = collect(ts, clip);
  const Guard guard(ts[0].device());
  const auto opt = ts[0].options();
  const std::vector<Table> tables = tables_of(g.dense);
  int blocks = 0;
  for (const Table& t : tables) blocks += grad_norm_blocks(t.t);
  at::Tensor out = at::empty({2}, opt.dtype(at::kFloat));
  at::Tensor partial = at::empty({blocks}, opt.dtype(at::kDouble));
  const hipStream_t stream = stream_of(ts[0]);
  const int kind = static_cast<int>(type);
  const float bound = static_cast<float>(max_norm);
  double* const sums = partial.data_ptr<double>();
  float* const result = out.data_ptr<float>();
  int at = 0;
  for (const Table& t : tables) {
    launch_grad_partial(t.t, t.dtype, kind, sums + at, stream);
    at += grad_norm_blocks(t.t);
  }
  const bool folds = clip && blocks > 0 && grad_clip_folds(blocks);
  if (!folds) launch_grad_finish(sums, blocks, kind, bound, result, stream);
  if (clip) {
    // What the norm read last comes first.
    for (auto t = tables.rbegin(); t != tables.rend(); ++t) {
      if (folds)
        launch_grad_clip(t->t, t->dtype, kind, sums, blocks, bound, result,
                         stream);
      else
        launch_grad_scale(t->t, t->dtype, result + 1, stream);
    }
    write_back(g);
  }
  check_launch();
  return out;
}

at::Tensor grad_norm_kernel(at::TensorList ts, int64_t type,
                            double max_norm) {
  at::AutoDispatchBelowADInplaceOrView below;
  return norm_of(ts, type, max_norm, false);
}

at::Tensor grad_norm(const std::vector<at::Tensor>& ts, int64_t type,
                     double max_norm) {
  static const auto op = op_of<decltype(grad_norm_kernel)>("axon::grad_norm");
  return op.call(ts, type, max_norm);
}

// The gradients of lists of parameters, read here rather than in Python:
// that takes longer than the kernels where there are hundreds of small ones.
// False where one is not a float/half/bfloat16 tensor on the first one's GPU.
bool param_grads(const pybind11::list& lists, std::vector<at::Tensor>& grads) {
  for (const auto& list : lists) {
    if (!PyList_Check(list.ptr())) return false;
    const Py_ssize_t n = PyList_GET_SIZE(list.ptr());
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PyList_GET_ITEM(list.ptr(), i);
      if (!THPVariable_Check(o)) return false;
      const at::Tensor& g = THPVariable_Unpack(o).grad();
      if (!g.defined()) continue;
      if (!g.is_cuda() || g.layout() != at::kStrided || !float_type(g.scalar_type()) ||
          (!grads.empty() && g.device() != grads[0].device()))
        return false;
      grads.push_back(g);
    }
  }
  return true;
}

// For lists of parameters: (norm, factor) as fp32[2], None where none has a
// gradient, False where the general path has to take them.
pybind11::object param_grad_norm(const pybind11::list& lists, int64_t type,
                                 double max_norm, bool clip) {
  std::vector<at::Tensor> grads;
  if (!param_grads(lists, grads)) return pybind11::bool_(false);
  if (grads.empty()) return pybind11::none();
  check_untraced("gradient clipping");
  return pybind11::cast(norm_of(grads, type, max_norm, clip));
}

void grad_scale_(const std::vector<at::Tensor>& ts, const at::Tensor& factor) {
  check_untraced("gradient clipping");
  const Grads g = collect(ts, true);
  TORCH_CHECK(factor.device() == ts[0].device() && factor.numel() == 1 &&
                  factor.scalar_type() == at::kFloat,
              "grad scale: the factor must be one float on the tensors' GPU");
  const Guard guard(ts[0].device());
  for (const Table& t : tables_of(g.dense))
    launch_grad_scale(t.t, t.dtype, factor.data_ptr<float>(),
                      stream_of(ts[0]));
  write_back(g);
  check_launch();
}

TORCH_LIBRARY(axon, m) {
  m.def("embedding(Tensor ids, Tensor weight, float scale, int? padding_idx) "
        "-> Tensor");
  m.def("embedding_backward(Tensor ids, Tensor grad, int vocab, int padding, "
        "float scale) -> Tensor");
  m.def("cross_entropy(Tensor logits, Tensor target, int ignore_index, "
        "float label_smoothing, int reduction) -> (Tensor, Tensor)");
  m.def("cross_entropy_backward(Tensor grad, Tensor logits, Tensor target, "
        "Tensor kept, int ignore_index, float label_smoothing, int reduction) "
        "-> Tensor");
  m.def("grad_norm(Tensor[] tensors, int norm_type, float max_norm) -> Tensor");
}

TORCH_LIBRARY_IMPL(axon, CUDA, m) {
  m.impl("embedding", &embedding_kernel);
  m.impl("embedding_backward", &embedding_backward_kernel);
  m.impl("cross_entropy", &cross_entropy_kernel);
  m.impl("cross_entropy_backward", &cross_entropy_backward_kernel);
  m.impl("grad_norm", &grad_norm_kernel);
}

TORCH_LIBRARY_IMPL(axon, AutogradCUDA, m) {
  m.impl("embedding", &embedding_autograd);
  m.impl("cross_entropy", &cross_entropy_autograd);
  m.impl("embedding_backward", &embedding_backward_autograd);
  m.impl("cross_entropy_backward", &cross_entropy_backward_autograd);
  // Its callers compute it without gradients.
  m.impl("grad_norm", torch::CppFunction::makeFallthrough());
}

}  // namespace

void register_lm(pybind11::module_& m) {
  m.def("embedding", &embedding, py::arg("ids"), py::arg("weight"),
        py::arg("scale"), py::arg("padding_idx"));
  m.def("cross_entropy", &cross_entropy, py::arg("logits"), py::arg("target"),
        py::arg("ignore_index"), py::arg("label_smoothing"),
        py::arg("reduction"));
  m.def("grad_norm", &grad_norm, py::arg("tensors"), py::arg("type"),
        py::arg("max_norm"));
  m.def("param_grad_norm", &param_grad_norm, py::arg("lists"),
        py::arg("type"), py::arg("max_norm"), py::arg("clip"));
  m.def("grad_scale_", &grad_scale_, py::arg("tensors"), py::arg("factor"));
}

}  // namespace axon
