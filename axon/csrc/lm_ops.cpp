// Torch-facing launchers of the language-model operators: embedding
// (kernels/embedding.hip), cross entropy (kernels/cross_entropy.hip) and the
// gradient norm (kernels/grad_norm.hip). They run on the tensors' device, on
// its current torch stream; scratch comes from torch's allocator per call.
#include <torch/extension.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <algorithm>
#include <unordered_map>

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

bool float_type(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf ||
         t.scalar_type() == at::kBFloat16;
}

void check_launch() {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, "axon: kernel launch failed: ",
              hipGetErrorString(e));
}

// ------------------------------------------------------------- embedding

void check_ids(const at::Tensor& ids, const at::Tensor& other) {
  TORCH_CHECK(ids.is_cuda() && ids.device() == other.device(),
              "embedding: ids and weight must be on the same GPU");
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt,
              "embedding: ids must be int32 or int64");
  TORCH_CHECK(ids.is_contiguous() && ids.numel() < (int64_t{1} << 31),
              "embedding: ids must be contiguous, fewer than 2^31");
}

at::Tensor embed_fwd(const at::Tensor& ids, const at::Tensor& w, double scale) {
  check_ids(ids, w);
  TORCH_CHECK(w.dim() == 2 && float_type(w) &&
                  (w.size(1) <= 1 || w.stride(1) == 1) &&
                  w.size(1) < (int64_t{1} << 22),
              "embedding: weight must be [V, D] float/half/bfloat16 with "
              "dense rows of fewer than 2^22 values");
  auto shape = ids.sizes().vec();
  shape.push_back(w.size(1));
  const Guard guard(w.device());
  at::Tensor y = at::empty(shape, w.options());
  if (y.numel() == 0) return y;
  launch_embed_fwd(code_of(w), ids.scalar_type() == at::kLong, ids.data_ptr(),
                   w.data_ptr(), y.data_ptr(), ids.numel(), w.size(0),
                   w.size(1), w.stride(0), static_cast<float>(scale),
                   stream_of(w));
  check_launch();
  return y;
}

at::Tensor embed_bwd(const at::Tensor& ids, const at::Tensor& dy_in,
                     int64_t vocab, int64_t padding, double scale) {
  check_ids(ids, dy_in);
  TORCH_CHECK(float_type(dy_in) && dy_in.dim() >= 1 &&
                  dy_in.sizes().slice(0, dy_in.dim() - 1) == ids.sizes(),
              "embedding: gradient must be ids' shape x D");
  TORCH_CHECK(vocab >= 0 && vocab < (int64_t{1} << 31),
              "embedding: fewer than 2^31 rows");
  const Guard guard(dy_in.device());
  const at::Tensor dy = dy_in.contiguous();
  const int64_t n = ids.numel(), dim = dy.size(-1);
  at::Tensor dw = at::empty({vocab, dim}, dy.options());
  if (dw.numel() == 0) return dw;
  at::Tensor keys = at::empty({2 * n}, ids.options().dtype(at::kLong));
  at::Tensor part =
      at::empty({embed_part_floats(n, dim, static_cast<int>(dy.element_size()))},
                dy.options().dtype(at::kFloat));
  launch_embed_bwd(code_of(dy), ids.scalar_type() == at::kLong, ids.data_ptr(),
                   dy.data_ptr(), dw.data_ptr(),
                   reinterpret_cast<uint64_t*>(keys.data_ptr()),
                   part.data_ptr<float>(), n, vocab, dim, padding,
                   static_cast<float>(scale), stream_of(dy));
  check_launch();
  return dw;
}

// --------------------------------------------------------- cross entropy

struct LogitRows {
  int64_t n, vocab, inner, stride_outer, stride_inner;
};

// Logits [V], [N, V] or [B, S, V] with a dense last dimension; the others may
// have any strides.
LogitRows logit_rows(const at::Tensor& x, const at::Tensor& target) {
  TORCH_CHECK(x.is_cuda() && target.is_cuda() && x.device() == target.device(),
              "cross_entropy: logits and target must be on the same GPU");
  TORCH_CHECK(float_type(x) && x.dim() >= 1 && x.dim() <= 3 &&
                  x.size(-1) > 0 && (x.size(-1) == 1 || x.stride(-1) == 1),
              "cross_entropy: logits must be [V], [N, V] or [B, S, V] "
              "float/half/bfloat16 with a dense last dimension");
  TORCH_CHECK(target.scalar_type() == at::kLong && target.is_contiguous() &&
                  target.sizes() == x.sizes().slice(0, x.dim() - 1),
              "cross_entropy: target must be contiguous int64 of the logits' "
              "shape without the last dimension");
  LogitRows r;
  r.vocab = x.size(-1);
  r.n = target.numel();
  r.inner = x.dim() == 1 ? 1 : std::max<int64_t>(1, x.size(-2));
  r.stride_inner = x.dim() == 1 ? 0 : x.stride(-2);
  r.stride_outer = x.dim() == 3 ? x.stride(0) : 0;
  TORCH_CHECK(r.n < (int64_t{1} << 31) / 4, "cross_entropy: too many rows");
  return r;
}

// Returns (loss, kept, factor): a 0-dim loss, or one of target's shape for
// reduction 0; what the backward pass takes.
std::vector<at::Tensor> ce_fwd(const at::Tensor& x, const at::Tensor& target,
                               int64_t ignore, double eps, int64_t reduction) {
  const LogitRows r = logit_rows(x, target);
  TORCH_CHECK(reduction >= 0 && reduction <= 2, "cross_entropy: reduction");
  const Guard guard(x.device());
  const auto fopt = x.options().dtype(at::kFloat);
  at::Tensor kept = at::empty({2 * r.n}, fopt);
  at::Tensor factor = at::empty({1}, fopt);
  at::Tensor loss = reduction == 0 ? at::empty(target.sizes(), fopt)
                                   : at::empty({}, fopt);
  at::Tensor scratch = at::empty({ce_scratch_bytes(r.n, r.vocab)},
                                 x.options().dtype(at::kByte));
  launch_ce_fwd(code_of(x), x.data_ptr(), r.inner, r.stride_outer,
                r.stride_inner, target.data_ptr<int64_t>(), ignore, r.n,
                r.vocab, static_cast<float>(eps), static_cast<int>(reduction),
                scratch.data_ptr(), kept.data_ptr<float>(),
                loss.data_ptr<float>(), factor.data_ptr<float>(),
                stream_of(x));
  check_launch();
  return {loss, kept, factor};
}

at::Tensor ce_bwd(const at::Tensor& x, const at::Tensor& target,
                  int64_t ignore, double eps, int64_t reduction,
                  const at::Tensor& kept, const at::Tensor& factor,
                  const at::Tensor& gout_in) {
  const LogitRows r = logit_rows(x, target);
  TORCH_CHECK(gout_in.is_cuda() && gout_in.scalar_type() == at::kFloat &&
                  gout_in.numel() == (reduction == 0 ? r.n : 1),
              "cross_entropy: the loss's gradient");
  const Guard guard(x.device());
  const at::Tensor gout = gout_in.contiguous();
  at::Tensor dx = at::empty(x.sizes(), x.options());
  if (r.n == 0) return dx;
  launch_ce_bwd(code_of(x), x.data_ptr(), r.inner, r.stride_outer,
                r.stride_inner, target.data_ptr<int64_t>(), ignore, r.n,
                r.vocab, static_cast<float>(eps), kept.data_ptr<float>(),
                gout.data_ptr<float>(), reduction == 0 ? 1 : 0,
                reduction == 0 ? nullptr : factor.data_ptr<float>(),
                dx.data_ptr(), stream_of(x));
  check_launch();
  return dx;
}

// ---------------------------------------------------------- gradient norm

// The tensors as one list for the kernels: each buffer once (a tensor given
// twice counts once and is scaled once), and dense (a strided one goes
// through a dense copy).
struct Grads {
  std::vector<at::Tensor> dense;
  std::vector<std::pair<at::Tensor, size_t>> strided;  // original, its copy
};

Grads collect(const std::vector<at::Tensor>& ts, bool written) {
  Grads g;
  TORCH_CHECK_VALUE(!ts.empty(), "grad norm: no tensors");
  struct Span {
    const char *begin, *end;
  };
  std::vector<Span> spans;  // of the dense tensors
  std::unordered_multimap<const void*, size_t> seen;
  for (size_t i = 0; i < ts.size(); ++i) {
    const at::Tensor& t = ts[i];
    TORCH_CHECK_VALUE(t.is_cuda() && t.layout() == at::kStrided &&
                          float_type(t) && t.device() == ts[0].device(),
                      "grad norm: tensors must be dense float/half/bfloat16 "
                      "on one GPU");
    if (t.numel() == 0) continue;
    const auto alike = seen.equal_range(t.data_ptr());
    if (std::any_of(alike.first, alike.second, [&](const auto& e) {
          const at::Tensor& o = ts[e.second];
          return o.sizes() == t.sizes() && o.strides() == t.strides() &&
                 o.scalar_type() == t.scalar_type();
        }))
      continue;
    seen.emplace(t.data_ptr(), i);
    if (t.is_non_overlapping_and_dense()) {
      const char* p = static_cast<const char*>(t.data_ptr());
      spans.push_back({p, p + t.nbytes()});
      g.dense.push_back(t);
    } else {
      if (written) at::assert_no_internal_overlap(t);
      g.strided.emplace_back(t, g.dense.size());
      g.dense.push_back(t.contiguous());
    }
  }
  if (written) {
    // Two blocks would scale the same value. (A strided tensor's copy holds
    // the values from before; writing it back gives the same ones.)
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) {
      return a.begin < b.begin;
    });
    for (size_t i = 1; i < spans.size(); ++i)
      TORCH_CHECK_VALUE(spans[i].begin >= spans[i - 1].end,
                        "grad norm: gradients share memory in part");
  }
  return g;
}

// Calls f(table, dtype) for tables that cover all tensors, one type each.
template <typename F>
void for_tables(const std::vector<at::Tensor>& ts, F f) {
  for (auto type : {at::kFloat, at::kHalf, at::kBFloat16}) {
    GradTable t;
    t.count = 0;
    t.first[0] = 0;
    auto done = [&] {
      if (t.count) f(t, static_cast<int>(type));
      t.count = 0;
    };
    for (const at::Tensor& x : ts) {
      if (x.scalar_type() != type) continue;
      const int64_t chunks = (x.numel() + kGradChunk - 1) / kGradChunk;
      TORCH_CHECK(chunks < (int64_t{1} << 30), "grad norm: tensor too large");
      if (t.count == kGradTensors ||
          (t.count && t.first[t.count] + chunks >= (int64_t{1} << 30)))
        done();
      t.ptr[t.count] = x.data_ptr();
      t.n[t.count] = x.numel();
      t.first[t.count + 1] =
          t.first[t.count] + static_cast<int32_t>(chunks);
      ++t.count;
    }
    done();
  }
}

at::Tensor norm_of(const Grads& g, const at::Tensor& like, int64_t type,
                   double max_norm) {
  const auto opt = like.options();
  at::Tensor out = at::empty({2}, opt.dtype(at::kFloat));
  int blocks = 0;
  for_tables(g.dense, [&](const GradTable& t, int) {
    blocks += grad_norm_blocks(t);
  });
  at::Tensor partial = at::empty({blocks}, opt.dtype(at::kDouble));
  const hipStream_t stream = stream_of(like);
  int at = 0;
  for_tables(g.dense, [&](const GradTable& t, int dtype) {
    launch_grad_partial(t, dtype, static_cast<int>(type),
                        partial.data_ptr<double>() + at, stream);
    at += grad_norm_blocks(t);
  });
  launch_grad_finish(partial.data_ptr<double>(), blocks,
                     static_cast<int>(type), static_cast<float>(max_norm),
                     out.data_ptr<float>(), stream);
  check_launch();
  return out;
}

void scale_by(const Grads& g, const at::Tensor& like, const float* factor) {
  const hipStream_t stream = stream_of(like);
  for_tables(g.dense, [&](const GradTable& t, int dtype) {
    launch_grad_scale(t, dtype, factor, stream);
  });
  check_launch();
  for (auto& s : g.strided) s.first.copy_(g.dense[s.second]);
}

// (norm, factor) as fp32[2]; type 0 is the maximum.
at::Tensor grad_norm(const std::vector<at::Tensor>& ts, int64_t type,
                     double max_norm) {
  TORCH_CHECK(type >= 0 && type <= 2, "grad norm: type");
  const Grads g = collect(ts, false);
  const Guard guard(ts[0].device());
  return norm_of(g, ts[0], type, max_norm);
}

at::Tensor grad_clip_(const std::vector<at::Tensor>& ts, int64_t type,
                      double max_norm) {
  TORCH_CHECK(type >= 0 && type <= 2, "grad norm: type");
  const Grads g = collect(ts, true);
  const Guard guard(ts[0].device());
  at::Tensor out = norm_of(g, ts[0], type, max_norm);
  scale_by(g, ts[0], out.data_ptr<float>() + 1);
  return out;
}

void grad_scale_(const std::vector<at::Tensor>& ts, const at::Tensor& factor) {
  const Grads g = collect(ts, true);
  TORCH_CHECK(factor.device() == ts[0].device() && factor.numel() == 1 &&
                  factor.scalar_type() == at::kFloat,
              "grad scale: the factor must be one float on the tensors' GPU");
  const Guard guard(ts[0].device());
  scale_by(g, ts[0], factor.data_ptr<float>());
}

}  // namespace

void register_lm(pybind11::module_& m) {
  m.def("embed_fwd", &embed_fwd, py::arg("ids"), py::arg("weight"),
        py::arg("scale"));
  m.def("embed_bwd", &embed_bwd, py::arg("ids"), py::arg("dy"),
        py::arg("vocab"), py::arg("padding"), py::arg("scale"));
  m.def("ce_fwd", &ce_fwd, py::arg("logits"), py::arg("target"),
        py::arg("ignore_index"), py::arg("label_smoothing"),
        py::arg("reduction"));
  m.def("ce_bwd", &ce_bwd, py::arg("logits"), py::arg("target"),
        py::arg("ignore_index"), py::arg("label_smoothing"),
        py::arg("reduction"), py::arg("kept"), py::arg("factor"),
        py::arg("grad_loss"));
  m.def("grad_norm", &grad_norm, py::arg("tensors"), py::arg("type"),
        py::arg("max_norm"));
  m.def("grad_scale_", &grad_scale_, py::arg("tensors"), py::arg("factor"));
  m.def("grad_clip_", &grad_clip_, py::arg("tensors"), py::arg("type"),
        py::arg("max_norm"));
}

}  // namespace axon
