// Torch-facing launchers for the fused optimizer kernels (K6): build
// multi-tensor chunk descriptors, stage them through pinned memory, launch
// on the current torch stream. One kernel launch per parameter group.
#include <torch/extension.h>

#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>

#include "kernels/optimizers.h"

namespace axon {
namespace {

int64_t pick_chunk_elems(int64_t total) {
  // Target ~4096 chunks so 256 CUs stay filled; clamp to [16K, 256K].
  int64_t c = total / 4096;
  int64_t v = 16384;
  while (v < c && v < (1 << 18)) v <<= 1;
  return v;
}

struct ChunkPlan {
  at::Tensor host;  // pinned byte buffer of OptChunk[]
  at::Tensor dev;
  int nchunks = 0;
};

void check_type(const at::Tensor& p) {
  TORCH_CHECK(p.scalar_type() == at::kFloat || p.scalar_type() == at::kHalf ||
                  p.scalar_type() == at::kBFloat16,
              "fused optimizer: float/half/bfloat16 parameters only");
}

ChunkPlan build_chunks(const std::vector<at::Tensor>& ps,
                       const std::vector<at::Tensor>& gs,
                       const std::vector<at::Tensor>& ms,
                       const std::vector<at::Tensor>& vs, bool with_m,
                       bool with_v, float* u_base /* fp32 scratch or null */) {
  check_type(ps[0]);
  int64_t total = 0;
  for (auto& p : ps) total += p.numel();
  int64_t ce = pick_chunk_elems(total);
  std::vector<OptChunk> chunks;
  chunks.reserve(ps.size() + total / ce);
  int64_t uoff = 0;
  TORCH_CHECK(gs.size() == ps.size() && ms.size() == (with_m ? ps.size() : 0) &&
                  vs.size() == (with_v ? ps.size() : 0),
              "fused optimizer: as many grads and states as params");
  for (size_t t = 0; t < ps.size(); ++t) {
    auto& p = ps[t];
    // Elementwise over dense storage: any non-overlapping-and-dense layout
    // (incl. channels_last) works as long as param/grad/state agree on
    // strides — same storage index = same logical element on all of them.
    // All of one type, which the kernels read and write them as.
    TORCH_CHECK(p.scalar_type() == ps[0].scalar_type() &&
                    p.device() == ps[0].device(),
                "fused optimizer: params of one type on one device");
    TORCH_CHECK(p.is_non_overlapping_and_dense() &&
                    gs[t].is_non_overlapping_and_dense(),
                "fused optimizer requires dense params/grads");
    for (auto* l : {&gs, &ms, &vs}) {
      if (l->empty()) continue;
      const at::Tensor& o = (*l)[t];
      TORCH_CHECK(o.sizes() == p.sizes() &&
                      o.scalar_type() == p.scalar_type() &&
                      o.device() == p.device(),
                  "fused optimizer: grad and state must have the param's "
                  "shape, type and device");
      TORCH_CHECK(p.numel() <= 1 || o.strides() == p.strides(),
                  "fused optimizer: grad and state layout must match param "
                  "layout");
    }
    size_t esize = p.element_size();
    char* pp = static_cast<char*>(p.data_ptr());
    char* gg = static_cast<char*>(gs[t].data_ptr());
    char* mm = ms.empty() ? nullptr : static_cast<char*>(ms[t].data_ptr());
    char* vv = vs.empty() ? nullptr : static_cast<char*>(vs[t].data_ptr());
    int64_t n = p.numel();
    for (int64_t off = 0; off < n; off += ce) {
      OptChunk c;
      c.p = pp + off * esize;
      c.g = gg + off * esize;
      c.m = mm ? mm + off * esize : nullptr;
      c.v = vv ? vv + off * esize : nullptr;
      c.u = u_base ? u_base + uoff + off : nullptr;
      c.n = std::min<int64_t>(ce, n - off);
      c.tidx = static_cast<int64_t>(t);
      chunks.push_back(c);
    }
    uoff += n;
  }
  ChunkPlan plan;
  plan.nchunks = static_cast<int>(chunks.size());
  int64_t bytes = static_cast<int64_t>(chunks.size() * sizeof(OptChunk));
  plan.host = at::empty({bytes}, at::TensorOptions()
                                     .dtype(at::kByte)
                                     .pinned_memory(true));
  std::memcpy(plan.host.data_ptr(), chunks.data(), bytes);
  plan.dev = at::empty({bytes}, at::TensorOptions()
                                    .dtype(at::kByte)
                                    .device(ps[0].device()));
  plan.dev.copy_(plan.host, /*non_blocking=*/true);
  return plan;
}

int dtype_code(const at::Tensor& t) {
  return static_cast<int>(t.scalar_type());
}

hipStream_t cur_stream(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(
             static_cast<c10::DeviceIndex>(t.get_device()))
      .stream();
}

// The clipping factor that the step multiplies the gradients by, or null.
const float* scale_ptr(const c10::optional<at::Tensor>& t,
                       const at::Tensor& like) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK(t->device() == like.device() && t->scalar_type() == at::kFloat &&
                  t->numel() == 1,
              "fused optimizer: grad_scale must be one float on the "
              "parameters' device");
  return t->data_ptr<float>();
}

void fused_sgd(std::vector<at::Tensor> ps, std::vector<at::Tensor> gs,
               std::vector<at::Tensor> ms, double lr, double momentum,
               double dampening, double wd, bool nesterov, bool maximize,
               c10::optional<at::Tensor> grad_scale) {
  if (ps.empty()) return;
  auto plan = build_chunks(ps, gs, momentum != 0 ? ms : std::vector<at::Tensor>{},
                           {}, momentum != 0, false, nullptr);
  // momentum==0 passes ms pointers as null via empty list; kernel ignores m.
  if (momentum != 0) {
    TORCH_CHECK(ms.size() == ps.size(), "momentum buffers missing");
  }
  launch_fused_sgd(reinterpret_cast<const OptChunk*>(plan.dev.data_ptr()),
                   plan.nchunks, dtype_code(ps[0]), static_cast<float>(lr),
                   static_cast<float>(momentum), static_cast<float>(dampening),
                   static_cast<float>(wd), nesterov, maximize,
                   scale_ptr(grad_scale, ps[0]), cur_stream(ps[0]));
}

void fused_adam(std::vector<at::Tensor> ps, std::vector<at::Tensor> gs,
                std::vector<at::Tensor> ms, std::vector<at::Tensor> vs,
                double lr, double beta1, double beta2, double eps, double wd,
                int64_t step, bool adamw,
                c10::optional<at::Tensor> grad_scale) {
  if (ps.empty()) return;
  auto plan = build_chunks(ps, gs, ms, vs, true, true, nullptr);
  float bc1 = 1.0f - std::pow(static_cast<float>(beta1), static_cast<float>(step));
  float bc2_sqrt =
      std::sqrt(1.0f - std::pow(static_cast<float>(beta2), static_cast<float>(step)));
  launch_fused_adam(reinterpret_cast<const OptChunk*>(plan.dev.data_ptr()),
                    plan.nchunks, dtype_code(ps[0]), static_cast<float>(lr),
                    static_cast<float>(beta1), static_cast<float>(beta2),
                    static_cast<float>(eps), static_cast<float>(wd), bc1,
                    bc2_sqrt, adamw, scale_ptr(grad_scale, ps[0]),
                    cur_stream(ps[0]));
}

void fused_lamb(std::vector<at::Tensor> ps, std::vector<at::Tensor> gs,
                std::vector<at::Tensor> ms, std::vector<at::Tensor> vs,
                double lr, double beta1, double beta2, double eps, double wd,
                int64_t step, c10::optional<at::Tensor> grad_scale) {
  if (ps.empty()) return;
  int64_t total = 0;
  for (auto& p : ps) total += p.numel();
  at::Tensor u = at::empty({total}, ps[0].options().dtype(at::kFloat));
  at::Tensor norms = at::zeros({2 * static_cast<int64_t>(ps.size())},
                               ps[0].options().dtype(at::kFloat));
  auto plan = build_chunks(ps, gs, ms, vs, true, true, static_cast<float*>(u.data_ptr()));
  float bc1 = 1.0f - std::pow(static_cast<float>(beta1), static_cast<float>(step));
  float bc2_sqrt =
      std::sqrt(1.0f - std::pow(static_cast<float>(beta2), static_cast<float>(step)));
  auto* descs = reinterpret_cast<const OptChunk*>(plan.dev.data_ptr());
  auto stream = cur_stream(ps[0]);
  launch_fused_lamb_phase1(descs, plan.nchunks, dtype_code(ps[0]),
                           static_cast<float>(beta1), static_cast<float>(beta2),
                           static_cast<float>(eps), static_cast<float>(wd), bc1,
                           bc2_sqrt, static_cast<float*>(norms.data_ptr()),
                           scale_ptr(grad_scale, ps[0]), stream);
  launch_fused_lamb_phase2(descs, plan.nchunks, dtype_code(ps[0]),
                           static_cast<float>(lr),
                           static_cast<const float*>(norms.data_ptr()), stream);
}

// ---------------------------------------------------------------- one group
//
// The work of a whole parameter group in one call: with hundreds of small
// parameters the step is a matter of the time that the host takes for each.

struct AdamLists {
  std::vector<at::Tensor> ps, gs, ms, vs, steps;
};

// Reads the group's tensors into `l`; false where the general path has to
// look at them first: state that is missing or of another layout or type, a
// step count that is not one float on the CPU, anything not on one GPU.
bool read_adam_group(PyObject* params, PyObject* state, AdamLists& l) {
  static PyObject* const k_step = PyUnicode_InternFromString("step");
  static PyObject* const k_m = PyUnicode_InternFromString("exp_avg");
  static PyObject* const k_v = PyUnicode_InternFromString("exp_avg_sq");
  if (!PyList_Check(params) || !PyDict_Check(state)) return false;
  const Py_ssize_t n = PyList_GET_SIZE(params);
  for (auto* v : {&l.ps, &l.gs, &l.ms, &l.vs, &l.steps}) v->reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(params, i);
    if (!THPVariable_Check(o)) return false;
    const at::Tensor& p = THPVariable_Unpack(o);
    const at::Tensor& g = p.grad();
    if (!g.defined()) continue;
    PyObject* st = PyDict_GetItemWithError(state, o);
    if (!st && PyErr_Occurred()) throw pybind11::error_already_set();
    if (!st || !PyDict_Check(st)) return false;
    PyObject* so = PyDict_GetItem(st, k_step);
    PyObject* mo = PyDict_GetItem(st, k_m);
    PyObject* vo = PyDict_GetItem(st, k_v);
    if (!so || !mo || !vo || !THPVariable_Check(so) ||
        !THPVariable_Check(mo) || !THPVariable_Check(vo))
      return false;
    const at::Tensor &step = THPVariable_Unpack(so),
                     &m = THPVariable_Unpack(mo), &v = THPVariable_Unpack(vo);
    if (!step.is_cpu() || step.scalar_type() != at::kFloat ||
        step.numel() != 1 || !p.is_cuda() ||
        (!l.ps.empty() && p.device() != l.ps[0].device()) ||
        !p.is_non_overlapping_and_dense())
      return false;
    for (const at::Tensor* t : {&g, &m, &v})
      if (t->device() != p.device() || t->scalar_type() != p.scalar_type() ||
          t->layout() != at::kStrided || t->sizes() != p.sizes() ||
          (p.numel() > 1 && t->strides() != p.strides()))
        return false;
    l.ps.push_back(p);
    l.gs.push_back(g);
    l.ms.push_back(m);
    l.vs.push_back(v);
    l.steps.push_back(step);
  }
  return true;
}

// kind: 0 Adam, 1 AdamW, 2 LAMB. Returns false, with nothing changed, where
// read_adam_group does.
bool fused_adam_group(pybind11::object params, pybind11::object state,
                      int64_t kind, double lr, double beta1, double beta2,
                      double eps, double wd,
                      c10::optional<at::Tensor> grad_scale) {
  AdamLists l;
  if (!read_adam_group(params.ptr(), state.ptr(), l)) return false;
  // The factor is where the first gradient of all groups is.
  if (grad_scale.has_value() && !l.ps.empty()) {
    grad_scale = grad_scale->to(l.ps[0].device());
    scale_ptr(grad_scale, l.ps[0]);  // refused before a step is counted
  }
  // One launch for each type and step count, in the order of the parameters.
  std::vector<std::pair<at::ScalarType, float>> keys;
  std::vector<AdamLists> parts;
  for (size_t i = 0; i < l.ps.size(); ++i) {
    float& step = *l.steps[i].data_ptr<float>();
    step += 1.0f;
    const std::pair<at::ScalarType, float> key(l.ps[i].scalar_type(), step);
    const size_t at = std::find(keys.begin(), keys.end(), key) - keys.begin();
    if (at == keys.size()) {
      keys.push_back(key);
      parts.emplace_back();
    }
    AdamLists& part = parts[at];
    part.ps.push_back(std::move(l.ps[i]));
    part.gs.push_back(std::move(l.gs[i]));
    part.ms.push_back(std::move(l.ms[i]));
    part.vs.push_back(std::move(l.vs[i]));
  }
  for (size_t k = 0; k < parts.size(); ++k) {
    AdamLists& part = parts[k];
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(
        part.ps[0].device());
    const int64_t step = static_cast<int64_t>(keys[k].second);
    if (kind == 2)
      fused_lamb(std::move(part.ps), std::move(part.gs), std::move(part.ms),
                 std::move(part.vs), lr, beta1, beta2, eps, wd, step,
                 grad_scale);
    else
      fused_adam(std::move(part.ps), std::move(part.gs), std::move(part.ms),
                 std::move(part.vs), lr, beta1, beta2, eps, wd, step,
                 kind == 1, grad_scale);
  }
  return true;
}

// Refuses a step over lists of parameters, before any of it is done, if the
// kernels do not take one of those on a GPU that have a gradient.
void check_fused_step(const pybind11::list& lists) {
  for (const auto& list : lists) {
    const pybind11::list params(  // the same one, if it is a list
        pybind11::reinterpret_borrow<pybind11::object>(list));
    for (size_t i = 0; i < params.size(); ++i) {
      PyObject* o = PyList_GET_ITEM(params.ptr(), i);
      if (!THPVariable_Check(o)) continue;
      const at::Tensor& p = THPVariable_Unpack(o);
      if (p.is_cuda() && p.grad().defined()) check_type(p);
    }
  }
}

}  // namespace

void register_optim(pybind11::module_& m) {
  m.def("check_fused_step", &check_fused_step, pybind11::arg("lists"));
  m.def("fused_adam_group", &fused_adam_group, pybind11::arg("params"),
        pybind11::arg("state"), pybind11::arg("kind"), pybind11::arg("lr"),
        pybind11::arg("beta1"), pybind11::arg("beta2"), pybind11::arg("eps"),
        pybind11::arg("weight_decay"),
        pybind11::arg("grad_scale") = pybind11::none());
  m.def("fused_sgd", &fused_sgd, pybind11::arg("params"), pybind11::arg("grads"),
        pybind11::arg("momentum_buffers"), pybind11::arg("lr"),
        pybind11::arg("momentum"), pybind11::arg("dampening"),
        pybind11::arg("weight_decay"), pybind11::arg("nesterov"),
        pybind11::arg("maximize"),
        pybind11::arg("grad_scale") = pybind11::none());
  m.def("fused_adam", &fused_adam, pybind11::arg("params"), pybind11::arg("grads"),
        pybind11::arg("exp_avgs"), pybind11::arg("exp_avg_sqs"),
        pybind11::arg("lr"), pybind11::arg("beta1"), pybind11::arg("beta2"),
        pybind11::arg("eps"), pybind11::arg("weight_decay"), pybind11::arg("step"),
        pybind11::arg("adamw"),
        pybind11::arg("grad_scale") = pybind11::none());
  m.def("fused_lamb", &fused_lamb, pybind11::arg("params"), pybind11::arg("grads"),
        pybind11::arg("exp_avgs"), pybind11::arg("exp_avg_sqs"),
        pybind11::arg("lr"), pybind11::arg("beta1"), pybind11::arg("beta2"),
        pybind11::arg("eps"), pybind11::arg("weight_decay"), pybind11::arg("step"),
        pybind11::arg("grad_scale") = pybind11::none());
}

}  // namespace axon
