// The operators whose smallest calls are bound by the host, as a Python module: argument checks, buffers,
// the launch through the C ABI and the autograd nodes in C++.  Written in Python, a lookup of 512 ids with
// its gradient took 89 us and a preference step over 8 rows 108, of which the two thread switches of
// torch's autograd engine are 36 and the kernels 15: the interpreter's work comes right behind the switches,
// when it is at its slowest.  Here they take 44 and 56, and an AdamW step over 40 tensors 22 instead of 54.
// (Run in the calling thread, torch.autograd.set_multithreading_enabled(False), the lookup takes 22.)
//
// The C ABI's functions are handed over as addresses (bind), so that this module uses the library that
// the rest of the package has loaded.  Host code only.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <mutex>

#include "../../include/recommend_amd.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

// ---- the C ABI
#define RK_EACH(F)                                                                                                   \
  F(rk_last_error) F(rk_embedding_fwd) F(rk_embedding_bwd_ws_bytes) F(rk_embedding_bwd) F(rk_list_logps_ws_bytes)    \
  F(rk_list_logps_fwd) F(rk_preference_fwd) F(rk_list_logps_bwd) F(rk_adamw_ws_bytes) F(rk_adamw_step)
struct Abi {
#define RK_MEMBER(name) decltype(&::name) name = nullptr;
  RK_EACH(RK_MEMBER)
} abi;
PyObject *rk_error = nullptr;   // the package's RkError

void bind(const py::dict &addresses, const py::object &error) {
#define RK_BIND(name) abi.name = reinterpret_cast<decltype(&::name)>(addresses[#name].cast<uintptr_t>());
  RK_EACH(RK_BIND)
  rk_error = error.inc_ref().ptr();
}

[[noreturn]] void raise_rk(int code, const std::string &what) {
  py::gil_scoped_acquire gil;
  py::object e = py::reinterpret_borrow<py::object>(rk_error)(code, what);
  PyErr_SetObject(rk_error, e.ptr());
  throw py::error_already_set();
}

// a failed call: RkError where Python called, a RuntimeError out of the autograd engine
void check(int rc) {
  if (rc != RK_OK) raise_rk(rc, abi.rk_last_error());
}
void check_in_backward(int rc) {
  TORCH_CHECK(rc == RK_OK, "librecommend_amd error ", rc, ": ", abi.rk_last_error());
}

void *stream_of(const at::Device &d) { return (void *)c10::hip::getCurrentHIPStream(d.index()).stream(); }

int32_t elem_of(at::ScalarType t, const char *what) {
  switch (t) {
    case at::kFloat: return RK_F32;
    case at::kBFloat16: return RK_BF16;
    case at::kHalf: return RK_F16;
    default:
      raise_rk(RK_ERR_UNSUPPORTED, std::string(what) + ": float32, bfloat16 or float16, not " + c10::toString(t));
  }
}

void need_device(const Tensor &t) {
  if (!t.is_cuda())
    raise_rk(RK_ERR_NODEV, "recommend_amd device ops need tensors on a HIP device; there is no CPU fallback");
}
void need_same_device(const Tensor &a, const Tensor &b) {
  need_device(a);
  need_device(b);
  TORCH_CHECK_VALUE(a.device() == b.device(), "tensors on several devices: ", a.device(), " and ", b.device());
}

constexpr int64_t kMaxInt = (1ll << 31) - (1 << 24);   // sizes are int32 at the C boundary

Tensor scratch(size_t bytes, const Tensor &like) {
  return at::empty({(int64_t)((bytes + 7) / 8)}, like.options().dtype(at::kDouble));
}

bool records(const Tensor &t) { return at::GradMode::is_enabled() && t.requires_grad(); }

void no_tangent(const char *what, const Tensor &t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), what, " has no forward-mode derivative");
}

// Gradients for a graph of the gradient (create_graph): they depend on what this node does not differentiate,
// so differentiating them raises.
variable_list only_once(const char *what, variable_list grads) {
  for (auto &g : grads)
    if (g.defined()) {
      auto node = std::make_shared<torch::autograd::DelayedError>(
          std::string(what) + " is differentiable once: it has no second derivative", 1);
      g = (*node)({g.detach().requires_grad_(true)})[0];
    }
  return grads;
}

// Whether a leaf's gradient would be handed to the default stream: its accumulator remembers the stream that it was made
// on, and lives as long as some graph over the leaf does.  A stream that records cannot hand anything to the default one.
bool waits_on_default(torch::autograd::Node *accumulator) {
  const auto s = accumulator ? accumulator->stream() : std::nullopt;
  return s && s->id() == c10::hip::getDefaultHIPStream(s->device_index()).id();   // (torch calls its device type CUDA)
}

void recordable(const char *what, const torch::autograd::Edge &edge) {
  torch::autograd::Node *next = edge.function.get();
  if (!dynamic_cast<torch::autograd::AccumulateGrad *>(next) || !waits_on_default(next)) return;
  TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None, what,
              ": a backward pass over this leaf cannot be recorded while a graph from the default stream is alive: delete the "
              "outputs of earlier passes first");
}

// ---- embedding lookup
struct LookupBackward : public Node {
  SavedVariable ids_;
  int64_t rows = 0, D = 0, padding = -1;
  float scale = 1.0f;
  int32_t kind = 0;

  std::string name() const override { return "EmbeddingLookupBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    ids_.reset_data();
  }

  Tensor gradient(const Tensor &grad, const Tensor &ids_in) {
    const Tensor g = grad.contiguous(), ids = ids_in.contiguous();
    c10::DeviceGuard guard(g.device());
    const int64_t n = ids.numel();
    // (a hook on saved tensors may have put something else in their place)
    TORCH_CHECK(n * D == g.numel() && ids.device() == g.device() &&
                    (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt),
                "embedding_lookup: the saved ids are not those of the forward pass");
    Tensor dw = at::empty({rows, D}, g.options());
    const Tensor ws = scratch(abi.rk_embedding_bwd_ws_bytes(n, (int32_t)rows, (int32_t)D, kind), g);
    check_in_backward(abi.rk_embedding_bwd(g.data_ptr(), kind, ids.data_ptr(), (int32_t)ids.element_size(), n, (int32_t)rows,
                                           (int32_t)D, scale, padding, dw.data_ptr(), ws.data_ptr(), ws.nbytes(),
                                           stream_of(g.device())));
    return dw;
  }

  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const Tensor &grad = grads[0];
    if (!grad.defined() || !task_should_compute_output(0)) return {Tensor()};
    no_tangent("embedding_lookup", grad);
    recordable("embedding_lookup", next_edge(0));
    const Tensor ids = ids_.unpack();
    // (linear in the upstream gradient: its derivative matters only where that has one)
    const bool graph = at::GradMode::is_enabled() && grad.requires_grad();
    at::AutoGradMode off(false);
    Tensor dw = gradient(grad.detach(), ids);
    if (!graph) return {dw};
    at::AutoGradMode on(true);
    return only_once("embedding_lookup", {dw});
  }
};

Tensor embedding_lookup(const Tensor &weight, const Tensor &ids_in, double scale, std::optional<int64_t> padding_idx) {
  no_tangent("embedding_lookup", weight);
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) >= 1, "embedding_lookup: the table is [rows, D], got ", weight.sizes());
  const int32_t kind = elem_of(weight.scalar_type(), "embedding_lookup");
  const int64_t rows = weight.size(0), D = weight.size(1);
  TORCH_CHECK_VALUE(rows < kMaxInt && D < kMaxInt, "embedding_lookup: a table of ", weight.sizes(),
                    " has more than 2^31 rows or columns");
  TORCH_CHECK_VALUE(ids_in.scalar_type() == at::kLong || ids_in.scalar_type() == at::kInt,
                    "embedding_lookup: ids are int32 or int64, not ", c10::toString(ids_in.scalar_type()));
  int64_t padding = -1;
  if (padding_idx) {
    TORCH_CHECK_VALUE(*padding_idx >= -rows && *padding_idx < rows, "embedding_lookup: padding_idx ", *padding_idx,
                      " outside the table of ", rows, " rows");
    padding = *padding_idx < 0 ? *padding_idx + rows : *padding_idx;
  }
  need_same_device(weight, ids_in);
  c10::DeviceGuard guard(weight.device());
  const bool record = records(weight);
  Tensor out, ids;
  {
    at::AutoGradMode off(false);
    ids = ids_in.contiguous();
    const Tensor w = weight.stride(1) == 1 && weight.stride(0) >= D ? weight : weight.contiguous();
    auto shape = ids.sizes().vec();
    shape.push_back(D);
    out = at::empty(shape, w.options());
    check(abi.rk_embedding_fwd(w.data_ptr(), rows > 1 ? w.stride(0) : D, (int32_t)rows, (int32_t)D, kind, ids.data_ptr(),
                               (int32_t)ids.element_size(), ids.numel(), (float)scale, out.data_ptr(),
                               stream_of(w.device())));
  }
  if (record) {
    auto node = std::shared_ptr<LookupBackward>(new LookupBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(weight));
    node->ids_ = SavedVariable(ids, false);
    node->rows = rows;
    node->D = D;
    node->padding = padding;
    node->scale = (float)scale;
    node->kind = kind;
    torch::autograd::set_history(out, node);
  }
  return out;
}

// ---- log-probabilities of lists, preference loss
struct Geometry {
  int32_t kind, S, T, V;
  int64_t stride_s, stride_t;
};

Geometry geometry_of(const Tensor &scores, int32_t kind) {
  const bool places = scores.dim() == 3;
  return {kind, (int32_t)scores.size(0), places ? (int32_t)scores.size(1) : 1, (int32_t)scores.size(-1), scores.stride(0),
          places ? scores.stride(1) : 0};
}

// rows whose scores lie side by side
Tensor rows_in_order(const Tensor &scores) {
  return scores.stride(-1) == 1 || scores.size(-1) == 1 ? scores : scores.contiguous();
}

struct ListBackward : public Node {
  SavedVariable scores_, items_;
  std::vector<int64_t> shape_;
  at::ScalarType type_ = at::kFloat;
  Tensor keep;                        // (max, log sum) of the rows, used places and slopes of the lists
  int64_t ignore = 0;
  int32_t average = 0, kind = 0;
  bool pairs = false;

  std::string name() const override { return pairs ? "PreferenceLossBackward" : "ListLogpsBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    scores_.reset_data();
    items_.reset_data();
    keep.reset();
  }

  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const char *what = pairs ? "preference_loss" : "list_logps";
    for (const Tensor &g : grads)
      if (g.defined()) no_tangent(what, g);
    const Tensor g_logps = grads[0].defined() ? grads[0].detach() : Tensor();
    const Tensor g_loss = grads.size() > 1 && grads[1].defined() ? grads[1].detach() : Tensor();
    if ((!g_logps.defined() && !g_loss.defined()) || !task_should_compute_output(0)) return {Tensor()};
    recordable(what, next_edge(0));
    Tensor scores = scores_.unpack(), items = items_.unpack();
    const bool graph = at::GradMode::is_enabled();
    at::AutoGradMode off(false);
    c10::DeviceGuard guard(scores.device());
    // (a hook on saved tensors, one that keeps them on the host for example, gives back other strides)
    scores = rows_in_order(scores);
    items = items.contiguous();
    const Geometry geo = geometry_of(scores, kind);
    TORCH_CHECK(scores.sizes() == shape_ && scores.scalar_type() == type_ && items.scalar_type() == at::kLong &&
                    items.numel() == (int64_t)geo.S * geo.T && items.device() == scores.device() &&
                    (geo.S == 0 || keep.device() == scores.device()),
                what, ": the saved tensors are not those of the forward pass");
    Tensor dx = at::empty(scores.sizes(), scores.options().memory_format(at::MemoryFormat::Contiguous));
    if (geo.S > 0) {
      const Tensor gp = g_logps.defined() ? g_logps.to(at::kFloat).contiguous() : Tensor();
      const Tensor gl = g_loss.defined() ? g_loss.to(at::kFloat).contiguous() : Tensor();
      const float *stat = keep.data_ptr<float>(), *used = stat + 2 * items.numel();
      check_in_backward(abi.rk_list_logps_bwd(scores.data_ptr(), geo.kind, geo.S, geo.T, geo.V, geo.stride_s, geo.stride_t,
                                              items.data_ptr<int64_t>(), geo.T, ignore, average, stat, (const int32_t *)used,
                                              gl.defined() ? gl.data_ptr<float>() : nullptr, pairs ? used + geo.S : nullptr,
                                              gp.defined() ? gp.data_ptr<float>() : nullptr, dx.data_ptr(),
                                              stream_of(scores.device())));
    }
    if (!graph) return {dx};
    at::AutoGradMode on(true);
    return only_once(what, {dx});
  }
};

// the loss where ref is given (undefined otherwise), and the lists' log-probabilities
std::pair<Tensor, Tensor> lists(const char *what, const Tensor &scores_in, const Tensor &items_in, const Tensor &ref_in,
                                int64_t ignore, bool average, double beta, double smoothing, int32_t form) {
  no_tangent(what, scores_in);
  const int32_t kind = elem_of(scores_in.scalar_type(), what);
  TORCH_CHECK_VALUE(items_in.scalar_type() == at::kLong || items_in.scalar_type() == at::kInt, what,
                    ": items are int32 or int64, not ", c10::toString(items_in.scalar_type()));
  const auto sizes = scores_in.sizes();
  TORCH_CHECK_VALUE((sizes.size() == 2 || sizes.size() == 3) && sizes.slice(0, sizes.size() - 1) == items_in.sizes(), what,
                    ": scores [lists, places, catalogue] and items [lists, places] (or without places), got ", sizes, " and ",
                    items_in.sizes());
  for (size_t k = 1; k < sizes.size(); ++k)
    TORCH_CHECK_VALUE(sizes[k] > 0, what, ": no places or no catalogue in ", sizes);
  for (const int64_t n : sizes)
    TORCH_CHECK_VALUE(n < kMaxInt, what, ": more than 2^31 lists, places or items in ", sizes);
  need_same_device(scores_in, items_in);
  c10::DeviceGuard guard(scores_in.device());
  const bool record = records(scores_in);
  // (recorded: the gradient of a copy finds its way back)
  const Tensor scores = rows_in_order(scores_in);
  const Geometry geo = geometry_of(scores, kind);
  Tensor items, keep, logps, loss;
  {
    at::AutoGradMode off(false);
    items = items_in.to(at::kLong).contiguous();
    const auto f32 = scores.options().dtype(at::kFloat);
    logps = at::empty({geo.S}, f32);
    if (geo.S > 0) {
      const int64_t rows = items.numel();
      int64_t n_keep = 2 * rows + 2 * (int64_t)geo.S;
      n_keep += n_keep % 2;
      const size_t ws_bytes = abi.rk_list_logps_ws_bytes(geo.S, geo.T, geo.V);
      keep = at::empty({n_keep + (int64_t)((ws_bytes + 3) / 4)}, f32);   // behind it: the call's workspace
      float *stat = keep.data_ptr<float>(), *used = stat + 2 * rows, *ws = stat + n_keep;
      if (!ref_in.defined()) {
        check(abi.rk_list_logps_fwd(scores.data_ptr(), geo.kind, geo.S, geo.T, geo.V, geo.stride_s, geo.stride_t,
                                    items.data_ptr<int64_t>(), geo.T, ignore, average, stat, logps.data_ptr<float>(),
                                    (int32_t *)used, ws, ws_bytes, stream_of(scores.device())));
      } else {
        const Tensor ref = ref_in.to(at::kFloat).contiguous();
        loss = at::empty({}, f32);
        check(abi.rk_preference_fwd(scores.data_ptr(), geo.kind, geo.S, geo.T, geo.V, geo.stride_s, geo.stride_t,
                                    items.data_ptr<int64_t>(), geo.T, ignore, average, ref.data_ptr<float>(), (float)beta,
                                    (float)smoothing, form, stat, logps.data_ptr<float>(), (int32_t *)used, used + geo.S,
                                    loss.data_ptr<float>(), ws, ws_bytes, stream_of(scores.device())));
      }
    }
  }
  if (record) {
    auto node = std::shared_ptr<ListBackward>(new ListBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(scores));
    node->scores_ = SavedVariable(scores, false);
    node->items_ = SavedVariable(items, false);
    node->keep = keep;
    node->shape_ = scores.sizes().vec();
    node->type_ = scores.scalar_type();
    node->kind = kind;
    node->ignore = ignore;
    node->average = average;
    node->pairs = loss.defined();
    torch::autograd::set_history(logps, node);
    if (loss.defined()) torch::autograd::set_history(loss, node);
  }
  return {loss, logps};
}

Tensor list_logps(const Tensor &scores, const Tensor &items, int64_t ignore, bool average) {
  return lists("list_logps", scores, items, Tensor(), ignore, average, 0.0, 0.0, 0).second;
}

std::pair<Tensor, Tensor> preference_loss(const Tensor &scores, const Tensor &items, const Tensor &ref, double beta,
                                          double smoothing, const std::string &form, int64_t ignore, bool average) {
  const int32_t kind = form == "sigmoid" ? RK_PREF_SIGMOID
                       : form == "hinge" ? RK_PREF_HINGE
                       : form == "squared" ? RK_PREF_SQUARED : -1;
  TORCH_CHECK_VALUE(kind >= 0, "preference_loss: kind is one of 'hinge', 'sigmoid', 'squared', not '", form, "'");
  TORCH_CHECK_VALUE(beta > 0, "preference_loss: beta must be positive");
  TORCH_CHECK_VALUE(smoothing >= 0 && smoothing <= 1, "preference_loss: label_smoothing outside [0, 1]");
  TORCH_CHECK_VALUE(smoothing == 0 || kind == RK_PREF_SIGMOID, "preference_loss: label smoothing is part of the sigmoid form only");
  const int64_t S = scores.dim() > 0 ? scores.size(0) : 0;
  TORCH_CHECK_VALUE(S >= 2 && S % 2 == 0, "preference_loss: pairs of lists are needed, got ", S, " lists");
  TORCH_CHECK_VALUE(ref.dim() == 1 && ref.size(0) == S, "preference_loss: one reference log-probability per list, got ",
                    ref.sizes(), " for ", S);
  TORCH_CHECK_VALUE(ref.is_floating_point(), "preference_loss: reference log-probabilities are floating point");
  TORCH_CHECK_VALUE(!records(ref), "preference_loss: the reference log-probabilities get no gradient: detach them, or "
                    "compute them under torch.no_grad()");
  no_tangent("preference_loss (of ref_logps)", ref);
  if (scores.is_cuda()) need_same_device(scores, ref);
  return lists("preference_loss", scores, items, ref, ignore, average, beta, smoothing, kind);
}

// ---- AdamW
int32_t adamw_elem(at::ScalarType t) {
  return t == at::kFloat ? RK_F32 : t == at::kBFloat16 ? RK_BF16 : t == at::kHalf ? RK_F16 : -1;
}

Tensor tensor_at(PyObject *dict, PyObject *key) {
  PyObject *o = PyDict_GetItemWithError(dict, key);
  return o && THPVariable_Check(o) ? THPVariable_Unpack(o) : Tensor();
}

struct Keys {
  PyObject *params = PyUnicode_InternFromString("params"), *m = PyUnicode_InternFromString("exp_avg"),
           *v = PyUnicode_InternFromString("exp_avg_sq"), *m8 = PyUnicode_InternFromString("exp_avg8"),
           *v8 = PyUnicode_InternFromString("exp_avg_sq8"), *ms = PyUnicode_InternFromString("exp_avg8_scale"),
           *vs = PyUnicode_InternFromString("exp_avg_sq8_scale");
};
const Keys &keys() {
  static const Keys k;
  return k;
}

bool has_moments(PyObject *st) {
  return st && (PyDict_GetItemWithError(st, keys().m) || PyDict_GetItemWithError(st, keys().m8));
}

// Moments of zero for the parameters that have a gradient and none yet; those of at least min_8bit elements as
// codes.  All are cleared by the launches of one call: the first step over 40 tensors takes 125 us with it (8-bit:
// 247), where clearing their moments one by one from Python took 552 (1129) by itself.
void make_moments(const py::list &groups, const py::dict &state, int64_t min_8bit, const at::Device &dev) {
  const Keys &k = keys();
  c10::DeviceGuard guard(dev);
  at::AutoGradMode off(false);
  std::vector<Tensor> made[2];   // of floats, of codes
  auto make = [&](py::object &st, PyObject *key, at::IntArrayRef sizes, bool codes) {
    const Tensor t = at::empty(sizes, at::TensorOptions(dev).dtype(codes ? at::kByte : at::kFloat));
    made[codes].push_back(t);
    const py::object o = py::cast(codes ? t.view(at::kFloat8_e4m3fn) : t);
    if (PyObject_SetItem(st.ptr(), key, o.ptr())) throw py::error_already_set();
  };
  for (const py::handle &gh : groups)
    for (const py::handle &ph : py::list(py::reinterpret_borrow<py::dict>(gh)["params"])) {
      const Tensor &p = THPVariable_Unpack(ph.ptr());
      if (!p.grad().defined() || p.numel() == 0 || p.device() != dev ||
          has_moments(PyDict_GetItemWithError(state.ptr(), ph.ptr())))
        continue;
      py::object st = py::reinterpret_steal<py::object>(PyObject_GetItem(state.ptr(), ph.ptr()));   // (makes an entry)
      if (!st) throw py::error_already_set();
      if (p.numel() < min_8bit) {
        make(st, k.m, p.sizes(), false);
        make(st, k.v, p.sizes(), false);
      } else {
        const int64_t blocks = (p.numel() + RK_ADAMW_BLOCK - 1) / RK_ADAMW_BLOCK;
        make(st, k.m8, {blocks * RK_ADAMW_BLOCK}, true);
        make(st, k.ms, {blocks}, false);
        make(st, k.v8, {blocks * RK_ADAMW_BLOCK}, true);
        make(st, k.vs, {blocks}, false);
      }
    }
  for (const auto &list : made)
    if (!list.empty()) at::_foreach_zero_(list);
}

// One step over the parameters of `groups` that have a gradient.  new_state() is called before moments are made,
// refuse(p, grad) raises for what the kernels do not take.  Returns 0, or the workspace bytes that it needs.
int64_t adamw_step(const py::list &groups, const py::dict &state, int64_t min_8bit, const py::object &new_state,
                   const py::object &refuse, const Tensor &step, const Tensor &lr, double max_norm, const Tensor &norm,
                   const Tensor &ws) {
  const Keys &k = keys();
  const at::Device dev = step.device();
  std::vector<rk_adamw_tensor> table;
  std::vector<rk_adamw_group> constants;
  table.reserve(64);
  int32_t group_index = 0;
  for (const py::handle &gh : groups) {
    const py::dict group = py::reinterpret_borrow<py::dict>(gh);
    const py::tuple betas(group["betas"]);
    constants.push_back({betas[0].cast<double>(), betas[1].cast<double>(), group["eps"].cast<double>(),
                         group["weight_decay"].cast<double>()});
    const py::list params(py::reinterpret_borrow<py::object>(PyDict_GetItemWithError(group.ptr(), k.params)));
    for (const py::handle &ph : params) {
      const Tensor &p = THPVariable_Unpack(ph.ptr());
      const Tensor &g = p.grad();
      if (!g.defined() || p.numel() == 0) continue;
      const int32_t pd = adamw_elem(p.scalar_type()), gd = adamw_elem(g.scalar_type());
      if (pd < 0 || (gd != pd && gd != RK_F32) || g.layout() != at::kStrided || !p.is_contiguous() || !g.is_contiguous() ||
          p.device() != dev || g.device() != dev)
        refuse(ph, py::cast(g));
      PyObject *st = PyDict_GetItemWithError(state.ptr(), ph.ptr());
      if (!has_moments(st)) {
        new_state();
        make_moments(groups, state, min_8bit, dev);
        st = PyDict_GetItemWithError(state.ptr(), ph.ptr());
      }
      const bool q8 = PyDict_GetItemWithError(st, k.m8) != nullptr;
      const Tensor m = tensor_at(st, q8 ? k.m8 : k.m), v = tensor_at(st, q8 ? k.v8 : k.v);
      const int64_t n = p.numel(), blocks = (n + RK_ADAMW_BLOCK - 1) / RK_ADAMW_BLOCK;
      Tensor ms, vs;
      if (q8) {
        ms = tensor_at(st, k.ms);
        vs = tensor_at(st, k.vs);
      }
      // (state that was put there by hand has to have the sizes that the kernels rely on)
      auto good = [&](const Tensor &t, int64_t size, at::ScalarType type) {
        return t.defined() && t.device() == dev && t.is_contiguous() && t.numel() == size && t.scalar_type() == type;
      };
      const bool fits = q8 ? good(m, blocks * RK_ADAMW_BLOCK, at::kFloat8_e4m3fn) && good(v, blocks * RK_ADAMW_BLOCK, at::kFloat8_e4m3fn) &&
                                 good(ms, blocks, at::kFloat) && good(vs, blocks, at::kFloat)
                           : good(m, n, at::kFloat) && good(v, n, at::kFloat);
      TORCH_CHECK_VALUE(fits, "FusedAdamW: the state of a parameter of ", p.sizes(),
                        " is not what this optimizer made: contiguous float32 moments of its size, or float8_e4m3fn codes padded "
                        "to blocks of ", RK_ADAMW_BLOCK, " with a float32 scale for each");
      torch::autograd::impl::bump_version(p);
      table.push_back({p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), q8 ? ms.data_ptr<float>() : nullptr,
                       q8 ? vs.data_ptr<float>() : nullptr, n, pd, gd, group_index, 0});
    }
    ++group_index;
  }
  if (table.empty()) return 0;
  const size_t need = abi.rk_adamw_ws_bytes((int32_t)table.size());
  if (ws.nbytes() < need) return (int64_t)need;
  c10::DeviceGuard guard(dev);
  check(abi.rk_adamw_step(table.data(), (int32_t)table.size(), constants.data(), (int32_t)constants.size(),
                          step.data_ptr<int64_t>(), lr.data_ptr<float>(), (float)max_norm, norm.data_ptr<float>(),
                          ws.data_ptr(), ws.nbytes(), stream_of(dev)));
  return 0;
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.def("bind", &bind);
  m.def("held_by_default_stream", [](const Tensor &leaf) {
    HANDLE_TH_ERRORS
    return waits_on_default(torch::autograd::impl::try_get_grad_accumulator(leaf).get());
    END_HANDLE_TH_ERRORS_PYBIND
  });
  m.def("embedding_lookup", [](const Tensor &w, const Tensor &ids, double scale, std::optional<int64_t> padding_idx) {
    HANDLE_TH_ERRORS
    return embedding_lookup(w, ids, scale, padding_idx);
    END_HANDLE_TH_ERRORS_PYBIND
  });
  m.def("list_logps", [](const Tensor &scores, const Tensor &items, int64_t ignore, bool average) {
    HANDLE_TH_ERRORS
    return list_logps(scores, items, ignore, average);
    END_HANDLE_TH_ERRORS_PYBIND
  });
  m.def("preference_loss", [](const Tensor &scores, const Tensor &items, const Tensor &ref, double beta, double smoothing,
                              const std::string &kind, int64_t ignore, bool average) {
    HANDLE_TH_ERRORS
    return preference_loss(scores, items, ref, beta, smoothing, kind, ignore, average);
    END_HANDLE_TH_ERRORS_PYBIND
  });
  m.def("adamw_step", [](const py::list &groups, const py::dict &state, int64_t min_8bit, const py::object &new_state,
                         const py::object &refuse, const Tensor &step, const Tensor &lr, double max_norm, const Tensor &norm,
                         const Tensor &ws) {
    HANDLE_TH_ERRORS
    return adamw_step(groups, state, min_8bit, new_state, refuse, step, lr, max_norm, norm, ws);
    END_HANDLE_TH_ERRORS_PYBIND
  });
}
