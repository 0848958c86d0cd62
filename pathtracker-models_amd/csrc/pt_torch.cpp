// pt_torch.cpp — the tensors' side of pt_scan.h and pt_clip.h (ptamd/_native.so).
//
// Argument checks, layouts, buffers and the autograd node of ptamd.scan and
// ptamd.clip.  These calls are made once a token or once a step and run for a
// few microseconds on the device; in Python the checks and the node alone took
// 15 us (a step), 65 us (30 gradients) and 140 us (a forward and backward), so
// they are here.  The kernels stay behind the C ABI: both libraries are opened
// by path and called through their headers' functions.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <optional>
#include <string>
#include <unordered_set>
#include <vector>

#include "pt_clip.h"
#include "pt_scan.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// ------------------------------------------------------------------ the libraries

struct Libs {
  decltype(&pt_scan_saved_bytes) scan_saved;
  decltype(&pt_scan_workspace_bytes) scan_work;
  decltype(&pt_scan_forward) scan_forward;
  decltype(&pt_scan_backward) scan_backward;
  decltype(&pt_scan_step) scan_step;
  decltype(&pt_scan_last_error) scan_error;
  decltype(&pt_clip_workspace_bytes) clip_work;
  decltype(&pt_clip_norm) clip_norm;
  decltype(&pt_clip_grads) clip_grads;
  decltype(&pt_clip_last_error) clip_error;
};
Libs lib;
PyObject* scan_error_type = nullptr;
PyObject* clip_error_type = nullptr;

template <typename F> void find(void* so, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(so, name));
  TORCH_CHECK(f, "the library lacks ", name);
}

void* open_lib(const std::string& path) {
  void* so = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(so, path, " cannot be opened: ", dlerror());
  return so;
}

void open_scan(const std::string& path, py::object error) {
  void* so = open_lib(path);
  find(so, "pt_scan_saved_bytes", lib.scan_saved);
  find(so, "pt_scan_workspace_bytes", lib.scan_work);
  find(so, "pt_scan_forward", lib.scan_forward);
  find(so, "pt_scan_backward", lib.scan_backward);
  find(so, "pt_scan_step", lib.scan_step);
  find(so, "pt_scan_last_error", lib.scan_error);
  scan_error_type = error.release().ptr();
}

void open_clip(const std::string& path, py::object error) {
  void* so = open_lib(path);
  find(so, "pt_clip_workspace_bytes", lib.clip_work);
  find(so, "pt_clip_norm", lib.clip_norm);
  find(so, "pt_clip_grads", lib.clip_grads);
  find(so, "pt_clip_last_error", lib.clip_error);
  clip_error_type = error.release().ptr();
}

// The module's own exception where Python is calling; the autograd engine's
// threads hold no interpreter lock and pass a RuntimeError on.
[[noreturn]] void raise(PyObject* type, const std::string& msg) {
  if (type && PyGILState_Check()) {
    PyErr_SetString(type, msg.c_str());
    throw py::error_already_set();
  }
  throw std::runtime_error(msg);
}

void check_scan(int rc) {
  if (rc) raise(scan_error_type, "pt_scan error " + std::to_string(rc) + ": " + lib.scan_error());
}
void check_clip(int rc) {
  if (rc) raise(clip_error_type, "pt_clip error " + std::to_string(rc) + ": " + lib.clip_error());
}

template <typename S> S stream_of(const Tensor& t) {
  return (S)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int type_code(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

// ------------------------------------------------------------------ layouts

using Dims = at::DimVector;
constexpr size_t KINDS = 4;              // kinds of tensors of a call (gates, their gradients, y): strides differ

struct Fold {
  int64_t b, c, n;
  pt_scan_view views[KINDS];             // strides; no pointers yet
};

// Dimensions lo..hi-1 as one axis of every kind: its size and strides.
// Axes of one element drop out.
bool merge(const Dims& size, const Dims* st, size_t kinds, size_t lo, size_t hi, int64_t& n, int64_t (&out)[KINDS]) {
  n = 1;
  std::fill(std::begin(out), std::end(out), 0);
  bool first = true;
  for (size_t k = hi; k-- > lo;) {
    if (size[k] == 1) continue;
    for (size_t i = 0; i < kinds; ++i) {
      if (first) out[i] = st[i][k];
      else if (st[i][k] != out[i] * n) return false;
    }
    first = false;
    n *= size[k];
  }
  return true;
}

// How tensors of one shape (their strides differing) fold into [batch][channels]
// [steps][inner], time at `dim` (-1: no time axis).  The batch is the first `lead`
// of the other dimensions (row ends need dimension 0 alone, and forward and
// backward, whose tensors may be laid out differently, have to agree on how the
// columns are cut), or as many as it takes (-1).
std::optional<Fold> fold(at::IntArrayRef sizes, int64_t dim, at::ArrayRef<at::IntArrayRef> strides, int64_t lead) {
  const size_t kinds = strides.size();
  TORCH_CHECK(kinds <= KINDS, "too many kinds of tensors");
  Dims size, st[KINDS];
  Fold f;
  for (size_t k = 0; k < sizes.size(); ++k) {
    if ((int64_t)k == dim) continue;
    size.push_back(sizes[k]);
    for (size_t i = 0; i < kinds; ++i) st[i].push_back(strides[i][k]);
  }
  for (size_t i = 0; i < kinds; ++i) f.views[i] = {nullptr, 0, 0, dim < 0 ? 0 : strides[i][dim]};
  const size_t first = lead < 0 ? 0 : lead;
  size_t inner = size.size();
  f.n = 1;
  while (inner > first) {                // every trailing axis that all tensors hold densely
    bool dense = true;
    for (size_t i = 0; i < kinds; ++i) dense = dense && (size[inner - 1] == 1 || st[i][inner - 1] == f.n);
    if (!dense) break;
    f.n *= size[--inner];
  }
  int64_t bs[KINDS], cs[KINDS];
  for (size_t cut = first; cut <= (lead < 0 ? inner : first); ++cut)    // dimensions cut..inner-1: channels
    if (merge(size, st, kinds, 0, cut, f.b, bs) && merge(size, st, kinds, cut, inner, f.c, cs)) {
      for (size_t i = 0; i < kinds; ++i) {
        f.views[i].sb = bs[i];
        f.views[i].sc = cs[i];
      }
      return f;
    }
  return std::nullopt;
}

// Whether no two elements share memory, for strides that nest.
bool disjoint(at::IntArrayRef sizes, at::IntArrayRef strides) {
  std::vector<std::pair<int64_t, int64_t>> v;
  for (size_t k = 0; k < sizes.size(); ++k)
    if (sizes[k] > 1) v.emplace_back(strides[k], sizes[k]);
  std::sort(v.begin(), v.end());
  int64_t reach = 1;
  for (const auto& [st, n] : v) {
    if (st < reach) return false;
    reach += st * (n - 1);
  }
  return true;
}

// The bytes from a tensor's first element to its last.
std::pair<uintptr_t, uintptr_t> span_of(const Tensor& t) {
  int64_t reach = 1;
  for (int64_t k = 0; k < t.dim(); ++k) reach += (t.size(k) - 1) * t.stride(k);
  const uintptr_t at = (uintptr_t)t.data_ptr();
  return {at, at + (uintptr_t)reach * t.element_size()};
}
bool meet(const Tensor& a, const Tensor& b) {
  const auto x = span_of(a), y = span_of(b);
  return x.first < y.second && y.first < x.second;
}

// Whether an address difference lo .. hi plus step times x, x in its axis' range, over
// all axes, can be 0.  Exact for strided tensors (views that interleave do not meet); it
// gives up as "yes" where the axes nest so little that the search takes long.
struct Axis {
  int64_t step, lo, hi;
};
struct Reach {
  std::vector<Axis> axes;                // the widest step first
  std::vector<int64_t> least, most;      // of the axes from k on
  int budget = 10000;

  explicit Reach(std::vector<Axis> ax) : axes(std::move(ax)), least(axes.size() + 1), most(axes.size() + 1) {
    std::sort(axes.begin(), axes.end(), [](const Axis& a, const Axis& b) { return a.step > b.step; });
    for (size_t k = axes.size(); k-- > 0;) {
      least[k] = least[k + 1] + axes[k].step * axes[k].lo;
      most[k] = most[k + 1] + axes[k].step * axes[k].hi;
    }
  }
  bool zero(int64_t lo, int64_t hi, size_t k = 0) {
    if (k == axes.size()) return lo <= 0 && 0 <= hi;
    const Axis& a = axes[k];
    const int64_t from = std::max(a.lo, (int64_t)std::ceil((double)-(hi + most[k + 1]) / (double)a.step));
    const int64_t to = std::min(a.hi, (int64_t)std::floor((double)-(lo + least[k + 1]) / (double)a.step));
    for (int64_t x = from; x <= to; ++x)
      if (--budget < 0 || zero(lo + a.step * x, hi + a.step * x, k + 1)) return true;
    return false;
  }
};

// Whether two tensors have a byte in common.
bool intersect(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0 || !meet(a, b)) return false;
  std::map<int64_t, Axis> ax;            // i steps of a and j of the same in b: i - j steps
  auto axes_of = [&ax](const Tensor& t, int sign) {
    for (int64_t k = 0; k < t.dim(); ++k) {
      const int64_t st = t.stride(k) * (int64_t)t.element_size();
      if (st == 0) continue;
      Axis& x = ax.emplace(st, Axis{st, 0, 0}).first->second;
      (sign > 0 ? x.hi : x.lo) += sign * (t.size(k) - 1);
    }
  };
  axes_of(a, 1);
  axes_of(b, -1);
  std::vector<Axis> list;
  for (const auto& [st, x] : ax) list.push_back(x);
  const int64_t d = (int64_t)((intptr_t)a.data_ptr() - (intptr_t)b.data_ptr());
  return Reach(list).zero(d - (int64_t)b.element_size() + 1, d + (int64_t)a.element_size() - 1);
}

// Whether two elements of one tensor share memory: places that differ, first in axis k.
bool meets_itself(const Tensor& t) {
  if (t.numel() == 0 || disjoint(t.sizes(), t.strides())) return false;
  std::vector<Axis> ax;
  for (int64_t k = 0; k < t.dim(); ++k)
    if (t.size(k) > 1) {
      if (t.stride(k) == 0) return true;
      ax.push_back({t.stride(k), 1 - t.size(k), t.size(k) - 1});
    }
  for (; !ax.empty(); ax.pop_back()) {
    auto some = ax;
    some.back().lo = 1;
    if (Reach(some).zero(0, 0)) return true;
  }
  return false;
}

// What autograd has to know of a tensor that a kernel wrote in place.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// What a call cannot take, looked at once a call and once a tensor.
struct Inputs {
  const char* op;
  PyObject* error;
  bool tangents;                         // they live in a level alone (a view's is looked up in its base: 30 ns)

  // The operators are unknown to whatever records calls instead of making them: a trace
  // would hold the outputs' allocation alone and replay whatever stands in that memory.
  Inputs(const char* op, PyObject* error)
      : op(op), error(error), tangents(torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr) {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    bool recorded = torch::jit::tracer::isTracing();
    for (auto k : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
      recorded = recorded || TorchDispatchModeTLS::get_mode(k).has_value();
    if (recorded) raise(error, std::string(op) + " cannot be traced");
  }
  // Forward-mode derivatives: the kernels carry no tangents, and an input whose tangent is
  // passed over would look like a constant.  Tensors of a Python dispatch (traced, sharded,
  // wrapping others): their address is none, or not that of their values.
  void check(const Tensor& t) const {
    if (tangents && t._fw_grad(/*level=*/0).defined())
      raise(error, std::string(op) + " has no forward-mode derivative: an input carries a tangent");
    if (t.key_set().has(c10::DispatchKey::Python))
      raise(error, std::string(op) +
                       " takes plain tensors: one with a Python dispatch has no memory that a kernel could read");
  }
};

// Whether a backward that has come to `from` goes on to a node of the default stream:
// the accumulator of a leaf that another graph, built there, keeps alive.  The engine
// makes that stream wait for the present one, which no capture allows; in a captured
// backward the process ends there.
bool waits_on_default_stream(const torch::autograd::Node* from) {
  const auto* exec = torch::autograd::get_current_graph_task_exec_info();   // null outside, empty: every node runs
  std::vector<const torch::autograd::Node*> open{from};
  std::unordered_set<const torch::autograd::Node*> seen{from};
  while (!open.empty()) {
    const auto* node = open.back();
    open.pop_back();
    for (const auto& edge : node->next_edges()) {
      auto* next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (exec && !exec->empty()) {
        const auto it = exec->find(next);
        if (it == exec->end() || !it->second.should_execute()) continue;
      }
      const auto stream = next->stream();
      if (stream && stream->device_type() != c10::kCPU && stream->id() == 0) return true;
      open.push_back(next);
    }
  }
  return false;
}

bool expanded(const Tensor& t) {
  for (int64_t k = 0; k < t.dim(); ++k)
    if (t.stride(k) == 0 && t.size(k) > 1) return true;
  return false;
}

// ------------------------------------------------------------------ the scan

using Gates = std::vector<Tensor>;

struct Form {
  int code;
  int gates;
  bool lstm() const { return code == PT_SCAN_LSTM; }
};

Form form_of(const std::string& name) {
  if (name == "leaky") return {PT_SCAN_LEAKY, 2};
  TORCH_CHECK_VALUE(name == "lstm", "unknown form '", name, "': one of leaky, lstm");
  return {PT_SCAN_LSTM, 4};
}

Gates chunks(const Tensor& x, int gates, int64_t gate_dim) {
  const int64_t w = x.size(gate_dim) / gates;
  Gates out;
  for (int g = 0; g < gates; ++g) out.push_back(x.narrow(gate_dim, g * w, w));
  return out;
}

// The gates of a call as the library reads them: one shape, one set of strides,
// a pointer each.  Of stacked gates no views are made (a token's call is short).
struct Side {
  Dims shape, strides;
  void* p[4];
  int count;
  Gates hold;                            // copies that the pointers belong to

  // stacked along gate_dim, or (-1) a tensor each; copied where their strides differ
  Side(const Gates& xs, int gates, int64_t gate_dim) : count(gates) {
    if (gate_dim < 0) {
      take(xs);
      return;
    }
    const Tensor& x = xs[0];
    shape = Dims(x.sizes().begin(), x.sizes().end());
    strides = Dims(x.strides().begin(), x.strides().end());
    shape[gate_dim] /= gates;
    const int64_t step = shape[gate_dim] * strides[gate_dim] * (int64_t)x.element_size();
    for (int g = 0; g < gates; ++g) p[g] = (char*)x.data_ptr() + g * step;
  }
  void take(const Gates& xs) {
    hold = xs;
    for (const auto& g : xs)
      if (g.strides() != xs[0].strides()) {
        for (auto& h : hold) h = h.contiguous();
        break;
      }
    shape = Dims(xs[0].sizes().begin(), xs[0].sizes().end());
    strides = Dims(hold[0].strides().begin(), hold[0].strides().end());
    for (int g = 0; g < count; ++g) p[g] = hold[g].data_ptr();
  }
  void views(const pt_scan_view& like, pt_scan_view* out) const {
    for (int g = 0; g < count; ++g) {
      out[g] = like;
      out[g].data = p[g];
    }
  }
};

Gates apart(const Gates& xs, int gates, int64_t gate_dim) {
  return gate_dim >= 0 ? chunks(xs[0], gates, gate_dim) : xs;
}

void dense_copies(Gates& gates) {
  for (auto& g : gates) g = g.contiguous();
}

pt_scan_view at_data(pt_scan_view v, const Tensor& t) {
  v.data = t.data_ptr();
  return v;
}

std::vector<int64_t> without(at::IntArrayRef sizes, int64_t dim) {
  std::vector<int64_t> out(sizes.begin(), sizes.end());
  out.erase(out.begin() + dim);
  return out;
}

template <typename T> T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }

Tensor bytes(size_t n, const Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

struct Scanned {
  Tensor y, h_last, c_last, saved;
  int64_t lead;                          // dimensions that the columns' batch took (fold)
};

Scanned forward(Form form, int64_t dim, int64_t gate_dim, bool want_seq, const Tensor& lengths, const Tensor& h0,
                const Gates& xs, bool keep) {
  const c10::DeviceGuard guard(xs[0].device());
  const auto opts = xs[0].options().requires_grad(false);
  Side x(xs, form.gates, gate_dim);
  const auto end = without(x.shape, dim);
  Scanned r;
  if (want_seq) r.y = at::empty(x.shape, opts);
  auto folded = [&](int64_t lead) {
    at::IntArrayRef st[] = {x.strides, want_seq ? r.y.strides() : at::IntArrayRef()};
    r.lead = lead;
    return fold(x.shape, dim, at::ArrayRef<at::IntArrayRef>(st, want_seq ? 2 : 1), lead);
  };
  // Rows without ends of their own are columns like the others.  Taken together
  // they leave no lane idle where a row's columns do not fill the last 64: lstm
  // bf16 300 x 500 x 20 28 us and 30 in the backward, 40 and 60 row by row; at a
  // thousand columns a row both take the same.
  std::optional<Fold> f;
  const int64_t cols = c10::multiply_integers(end) / x.shape[0];
  if (dim != 0 && !lengths.defined() && cols % 64 != 0) f = folded(0);
  if (!f) f = folded(dim != 0);
  if (!f) {                              // no common layout: dense copies have one
    Gates gates = apart(xs, form.gates, gate_dim);
    dense_copies(gates);
    x.take(gates);
    f = folded(dim != 0);
  }
  pt_scan_view xv[4], yv;
  x.views(f->views[0], xv);
  if (want_seq) yv = at_data(f->views[1], r.y);
  const pt_scan_desc d{form.code, type_code(xs[0].scalar_type()), f->b, f->c, x.shape[dim], f->n};
  r.h_last = at::empty(end, opts.dtype(at::kFloat));
  if (form.lstm()) r.c_last = at::empty(end, opts.dtype(at::kFloat));
  if (keep) r.saved = bytes(lib.scan_saved(&d), xs[0]);
  const Tensor work = bytes(lib.scan_work(&d), xs[0]);
  check_scan(lib.scan_forward(&d, xv, ptr<float>(h0), ptr<int64_t>(lengths), want_seq ? &yv : nullptr,
                              ptr<float>(r.h_last), ptr<float>(r.c_last), ptr<void>(r.saved), ptr<void>(work),
                              stream_of<pt_scan_stream_t>(xs[0])));
  return r;
}

// y, h_last, c_last = scan(gates; h0); x: one tensor with the gates stacked along
// gate_dim, or up to four tensors (gate_dim -1).
struct ScanFn : torch::autograd::Function<ScanFn> {
  using Opt = std::optional<Tensor>;
  static constexpr int kArgs = 11;

  static variable_list forward(AutogradContext* ctx, int64_t code, int64_t count, int64_t dim, int64_t gate_dim,
                               bool want_seq, const Opt& lengths, const Opt& h0, const Opt& x0, const Opt& x1,
                               const Opt& x2, const Opt& x3) {
    const Form form{(int)code, (int)count};
    Gates xs;
    for (const Opt* x : {&x0, &x1, &x2, &x3})
      if (x->has_value()) xs.push_back(**x);
    const Tensor len = lengths.value_or(Tensor()), h = h0.value_or(Tensor());
    Scanned r = ::forward(form, dim, gate_dim, want_seq, len, h, xs, true);
    variable_list keep{len, h, r.saved};
    keep.insert(keep.end(), xs.begin(), xs.end());
    ctx->save_for_backward(keep);
    ctx->saved_data["args"] = std::vector<int64_t>{code, count, dim, gate_dim, want_seq, r.lead};
    ctx->set_materialize_grads(false);
    variable_list out;
    if (want_seq) out.push_back(r.y);
    out.push_back(r.h_last);
    if (form.lstm()) out.push_back(r.c_last);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto args = ctx->saved_data["args"].toIntVector();
    const Form form{(int)args[0], (int)args[1]};
    const int64_t dim = args[2], gate_dim = args[3];
    const bool want_seq = args[4] != 0;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &lengths = saved[0], &h0 = saved[1], &states = saved[2];
    const Gates xs(saved.begin() + 3, saved.end());
    const c10::DeviceGuard guard(xs[0].device());
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None &&
        waits_on_default_stream(torch::autograd::get_current_node().get()))
      raise(scan_error_type,
            "gated_scan: a backward cannot be captured while a graph of the same leaves from the default stream "
            "lives (a loss of an earlier pass, for one): release it first");
    const Inputs in("gated_scan", scan_error_type);
    for (const auto& g : grads)          // (of no address they would pass for absent)
      if (g.defined()) in.check(g);
    variable_list out;
    {
      at::NoGradGuard no_grad;
      out = run(form, dim, gate_dim, want_seq, args[5], lengths, h0, states, xs, grads);
    }
    if (at::GradMode::is_enabled()) {    // the gradients have no derivative of their own
      for (auto& v : out)                // (of gradients that need none the error would leave no trace)
        if (v.defined()) v = v.detach().set_requires_grad(true);
      auto err = std::make_shared<torch::autograd::DelayedError>(
          "gated_scan is differentiable once: its gradients have no derivative", (int)out.size());
      return (*err)(std::move(out));
    }
    return out;
  }

  static variable_list run(Form form, int64_t dim, int64_t gate_dim, bool want_seq, int64_t lead,
                           const Tensor& lengths, const Tensor& h0, const Tensor& states, const Gates& xs,
                           const variable_list& grads) {
    Tensor dy = want_seq ? grads[0] : Tensor(), dh = grads[want_seq ? 1 : 0];
    Tensor dc = form.lstm() ? grads[want_seq ? 2 : 1] : Tensor();
    if (dy.defined()) dy = (expanded(dy) ? dy.contiguous() : dy).resolve_neg();  // (of a sum, a mean) no dense axis
    if (dh.defined()) dh = dh.contiguous().resolve_neg();
    if (dc.defined()) dc = dc.contiguous().resolve_neg();
    Side x(xs, form.gates, gate_dim);
    Gates dxs;                           // stacked as x is, or one a gate
    if (gate_dim >= 0) dxs.push_back(at::empty_like(xs[0]));
    else
      for (const auto& g : x.hold) dxs.push_back(at::empty_like(g));
    Side dx(dxs, form.gates, gate_dim);
    auto folded = [&] {
      at::IntArrayRef st[] = {x.strides, dx.strides, dy.defined() ? dy.strides() : at::IntArrayRef()};
      return fold(x.shape, dim, at::ArrayRef<at::IntArrayRef>(st, dy.defined() ? 3 : 2), lead);
    };
    auto f = folded();
    const bool copied = !f;
    if (copied) {                        // no common layout: dense tensors have one
      Gates gates = apart(xs, form.gates, gate_dim);
      dense_copies(gates);
      x.take(gates);
      dxs.clear();
      for (const auto& g : gates) dxs.push_back(at::empty_like(g));
      dx.take(dxs);
      if (dy.defined()) dy = dy.contiguous();
      f = folded();
    }
    pt_scan_view xv[4], dv[4], yv;
    x.views(f->views[0], xv);
    dx.views(f->views[1], dv);
    if (dy.defined()) yv = at_data(f->views[2], dy);
    const pt_scan_desc d{form.code, type_code(xs[0].scalar_type()), f->b, f->c, x.shape[dim], f->n};
    const Tensor dh0 = h0.defined() && h0.requires_grad() ? at::empty_like(h0) : Tensor();
    const Tensor work = bytes(lib.scan_work(&d), xs[0]);
    check_scan(lib.scan_backward(&d, xv, ptr<float>(h0), ptr<int64_t>(lengths), dy.defined() ? &yv : nullptr,
                                 ptr<float>(dh), ptr<float>(dc), ptr<void>(states), dv, ptr<float>(dh0),
                                 ptr<void>(work), stream_of<pt_scan_stream_t>(xs[0])));
    variable_list out(kArgs);
    out[6] = dh0;
    if (gate_dim >= 0) {
      out[7] = copied ? at::cat(dxs, gate_dim) : dxs[0];
    } else {
      for (int g = 0; g < form.gates; ++g) out[7 + g] = dxs[g];
    }
    return out;
  }
};

// The gates as passed on, gate_dim (-1: one tensor per gate) and a gate's shape.
struct Taken {
  Gates xs;
  int64_t gate_dim;
  std::vector<int64_t> shape;
};

Taken take(const py::object& x, Form form, int64_t gate_dim, int64_t least, const Inputs& in) {
  Taken t;
  if (THPVariable_Check(x.ptr())) {
    const Tensor v = THPVariable_Unpack(x.ptr());
    TORCH_CHECK_VALUE(v.dim() > least, "stacked gates need at least ", least + 1, " dimensions, got ", v.sizes());
    t.gate_dim = gate_dim < 0 ? gate_dim + v.dim() : gate_dim;
    TORCH_CHECK_VALUE(t.gate_dim >= 0 && t.gate_dim < v.dim(), "gate_dim ", gate_dim, " is outside the tensor's ",
                      v.dim(), " dimensions");
    TORCH_CHECK_VALUE(v.size(t.gate_dim) % form.gates == 0, "dimension ", t.gate_dim, " holds ", form.gates,
                      " gates, its size ", v.size(t.gate_dim), " is no multiple");
    t.shape = v.sizes().vec();
    t.shape[t.gate_dim] /= form.gates;
    t.xs.push_back(v);
  } else {
    t.gate_dim = -1;
    for (const py::handle& h : x) {
      TORCH_CHECK_TYPE(THPVariable_Check(h.ptr()), "the gates must be tensors");
      t.xs.push_back(THPVariable_Unpack(h.ptr()));
    }
    TORCH_CHECK_VALUE((int)t.xs.size() == form.gates, "the form takes ", form.gates, " gates, got ", t.xs.size());
    t.shape = t.xs[0].sizes().vec();
    for (const auto& v : t.xs)
      TORCH_CHECK_VALUE((int64_t)t.shape.size() >= least && v.sizes() == t.xs[0].sizes(),
                        "the gates need one shape of at least ", least, " dimensions");
  }
  const Tensor& v0 = t.xs[0];
  for (const auto& v : t.xs) {
    TORCH_CHECK_TYPE(v.layout() == at::kStrided && type_code(v.scalar_type()) >= 0, "gates of type ", v.scalar_type(),
                     ": dense float32, bfloat16 or float16");
    TORCH_CHECK_TYPE(v.scalar_type() == v0.scalar_type() && v.device() == v0.device(),
                     "the gates must have one type and one device");
    in.check(v);
  }
  for (auto& v : t.xs) v = v.resolve_neg();
  if (!v0.is_cuda()) raise(scan_error_type, "the gated scan runs on a ROCm device only (no CPU fallback)");
  return t;
}

py::tuple gated_scan(const py::object& x, std::optional<Tensor> h0, const std::string& form_name, int64_t dim,
                     int64_t gate_dim, std::optional<Tensor> lengths, bool want_seq) {
  const Form form = form_of(form_name);
  const Inputs in("gated_scan", scan_error_type);
  if (h0) in.check(*h0);
  Taken t = take(x, form, gate_dim, 2, in);
  const int64_t nd = t.shape.size(), k = dim < 0 ? dim + nd : dim;
  TORCH_CHECK_VALUE(k >= 0 && k < nd, "dim ", dim, " is outside the tensor's ", nd, " dimensions");
  TORCH_CHECK_VALUE(k != t.gate_dim, "the gates cannot be stacked along the time dimension");
  const auto device = t.xs[0].device();
  const auto end = without(t.shape, k);
  Tensor h, len;
  if (h0) {
    TORCH_CHECK_VALUE(h0->sizes() == at::IntArrayRef(end), "h0 has shape ", h0->sizes(), ", the state ",
                      at::IntArrayRef(end));
    TORCH_CHECK_TYPE(h0->device() == device && h0->is_floating_point(),
                     "h0 must be a floating-point tensor on the gates' device");
    h = h0->to(at::kFloat).contiguous().resolve_neg();
  }
  if (lengths) {
    in.check(*lengths);
    TORCH_CHECK_VALUE(k != 0, "lengths need the batch in dimension 0, which is the time dimension here");
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == t.shape[0], "lengths has shape ", lengths->sizes(),
                      ", expected [", t.shape[0], "]");
    TORCH_CHECK_TYPE(lengths->device() == device &&
                         at::isIntegralType(lengths->scalar_type(), /*includeBool=*/false),
                     "lengths must be an integer tensor on the gates' device");
    len = lengths->to(at::kLong).contiguous().resolve_neg();
  }
  auto give = [&](const Tensor& y, const Tensor& hl, const Tensor& cl) -> py::tuple {
    py::object seq = want_seq ? py::cast(y) : py::none();
    return form.lstm() ? py::make_tuple(seq, hl, cl) : py::make_tuple(seq, hl);
  };
  for (int64_t n : t.shape)
    if (n == 0) {                        // no step or no column: nothing to launch
      Tensor zero = at::zeros(end, t.xs[0].options().dtype(at::kFloat).requires_grad(false));
      for (const auto& g : t.xs)         // a gradient to the gates has a place to go, as with steps
        if (g.requires_grad()) zero = zero + g.sum(at::kFloat);
      const Tensor c = !h.defined() ? zero : zero.requires_grad() ? h + zero : h.clone();
      Tensor y;
      if (want_seq)
        for (const auto& g : t.gate_dim >= 0 ? chunks(t.xs[0], form.gates, t.gate_dim) : t.xs)
          y = y.defined() ? y + g : g.clone();
      return form.lstm() ? give(y, zero.clone(), c) : give(y, c, Tensor());
    }
  int64_t back = -1;
  if (k == nd - 1 && nd > 2 && t.shape[k] > 1 && t.shape[k - 1] > 1) {
    // time innermost ([B, D, T]): a lane's steps would lie together and the
    // lanes apart; two copies cost less than reading memory that way
    Gates g = t.gate_dim >= 0 ? chunks(t.xs[0], form.gates, t.gate_dim) : t.xs;
    for (auto& v : g) v = v.movedim(k, 1).contiguous();
    t.xs = g;
    t.gate_dim = -1;
    back = k;
  }
  const int64_t at_dim = back >= 0 ? 1 : k;
  bool grad = h.defined() && h.requires_grad();
  for (const auto& v : t.xs) grad = grad || v.requires_grad();
  Tensor y, hl, cl;
  if (grad && at::GradMode::is_enabled()) {
    std::optional<Tensor> a[4];
    for (size_t g = 0; g < t.xs.size(); ++g) a[g] = t.xs[g];
    auto opt = [](const Tensor& v) { return v.defined() ? std::optional<Tensor>(v) : std::nullopt; };
    variable_list r = ScanFn::apply((int64_t)form.code, (int64_t)form.gates, at_dim, t.gate_dim, want_seq, opt(len),
                                    opt(h), a[0], a[1], a[2], a[3]);
    size_t i = 0;
    if (want_seq) y = r[i++];
    hl = r[i++];
    if (form.lstm()) cl = r[i];
  } else {
    at::NoGradGuard no_grad;
    Scanned r = forward(form, at_dim, t.gate_dim, want_seq, len, h, t.xs, false);
    y = r.y;
    hl = r.h_last;
    cl = r.c_last;
  }
  if (back >= 0 && want_seq) y = y.movedim(1, back);
  return give(y, hl, cl);
}

Tensor gated_scan_step(const py::object& x, const Tensor& state, const std::string& form_name, int64_t gate_dim) {
  const Form form = form_of(form_name);
  const Inputs in("gated_scan_step", scan_error_type);
  in.check(state);
  if (state.is_neg()) raise(scan_error_type, "state is a negated view: it cannot be updated in place");
  Taken t = take(x, form, gate_dim, 1, in);
  TORCH_CHECK_TYPE(state.scalar_type() == at::kFloat && state.device() == t.xs[0].device(),
                   "state must be a float32 tensor on the gates' device");
  TORCH_CHECK_VALUE(state.sizes() == at::IntArrayRef(t.shape), "state has shape ", state.sizes(), ", expected ",
                    at::IntArrayRef(t.shape));
  if (at::GradMode::is_enabled()) {
    bool grad = state.requires_grad();
    for (const auto& v : t.xs) grad = grad || v.requires_grad();
    if (grad)
      raise(scan_error_type,
            "gated_scan_step has no backward: call it under torch.no_grad(), or use gated_scan");
  }
  at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(state.device());
  const Tensor y = at::empty(t.shape, t.xs[0].options().requires_grad(false));
  if (y.numel() == 0) return y;
  TORCH_CHECK_VALUE(disjoint(state.sizes(), state.strides()),
                    "state's elements share memory: it cannot be updated in place");
  for (auto& v : t.xs)                   // gates in the state's own memory: read before it is written
    if (meet(v, state)) v = v.clone(at::MemoryFormat::Contiguous);
  Side gates(t.xs, form.gates, t.gate_dim);
  Tensor s = state;
  auto folded = [&] {
    at::IntArrayRef st[] = {gates.strides, s.strides(), y.strides()};
    return fold(gates.shape, -1, st, -1);
  };
  auto f = folded();
  if (!f) {
    Gates copies = apart(t.xs, form.gates, t.gate_dim);
    dense_copies(copies);
    gates.take(copies);
    s = state.contiguous();
    f = folded();
  }
  pt_scan_view xv[4];
  gates.views(f->views[0], xv);
  const pt_scan_view sv = at_data(f->views[1], s), yv = at_data(f->views[2], y);
  const pt_scan_desc d{form.code, type_code(y.scalar_type()), f->b, f->c, 1, f->n};
  check_scan(lib.scan_step(&d, xv, &sv, &yv, stream_of<pt_scan_stream_t>(y)));
  if (s.data_ptr() != state.data_ptr()) state.copy_(s);
  else written(state);
  return y;
}

// ------------------------------------------------------------------ clipping

// Whether every element has a place of its own and the places are one run: the
// order of the axes does not matter to a norm.
bool dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

void check_tensors(const std::vector<Tensor>& ts, const char* what) {
  for (const auto& t : ts) {
    TORCH_CHECK_TYPE(t.layout() == at::kStrided && type_code(t.scalar_type()) >= 0, what, " of type ",
                     t.scalar_type(), ": dense float32, bfloat16 or float16");
    if (!t.is_cuda()) raise(clip_error_type, "clipping runs on a ROCm device only (no CPU fallback)");
    if (t.device() != ts[0].device())
      raise(clip_error_type, std::string(what) + " are on several devices: one process per GPU");
  }
}

// The library checks the memory that it is given.  Where a copy stands for a gradient or an
// output there (`aside`), the tensors themselves have to be apart from all others.
void check_aside(const std::vector<Tensor>& grads, const std::optional<std::vector<Tensor>>& out,
                 const std::vector<size_t>& aside) {
  struct Span {
    uintptr_t lo, hi, before;            // before: the furthest end of the spans in front
    size_t i;
    const Tensor* t;
    bool written;
  };
  std::vector<Span> all;
  auto add = [&all](const Tensor& t, size_t i, bool written) {
    if (t.numel() == 0) return;
    const auto [lo, hi] = span_of(t);
    all.push_back({lo, hi, 0, i, &t, written});
  };
  for (size_t i = 0; i < grads.size(); ++i) {
    add(grads[i], i, !out);
    if (out) add((*out)[i], i, true);
  }
  std::sort(all.begin(), all.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
  for (size_t k = 1; k < all.size(); ++k) all[k].before = std::max(all[k - 1].before, all[k - 1].hi);
  auto apart = [](const Span& a, const Span& b) {
    if (a.i != b.i && (a.written || b.written) && intersect(*a.t, *b.t))
      raise(clip_error_type, "a tensor that is written shares memory with another tensor of the call");
  };
  std::vector<bool> is_aside(grads.size());
  for (size_t i : aside) is_aside[i] = true;
  for (size_t k = 0; k < all.size(); ++k) {
    if (!is_aside[all[k].i]) continue;
    for (size_t j = k + 1; j < all.size() && all[j].lo < all[k].hi; ++j) apart(all[k], all[j]);
    for (size_t j = k; j > 0 && all[j].before > all[k].lo; --j) apart(all[k], all[j - 1]);
  }
}

// The norm of `grads`; with max_norm >= 0 they are clipped, into `out` or in place.
Tensor clip(const std::vector<Tensor>& grads, double norm_type, double max_norm,
            const std::optional<std::vector<Tensor>>& out) {
  int code = -1;
  if (std::isinf(norm_type) && norm_type > 0) code = PT_CLIP_INF;
  else if (norm_type == 1.0) code = PT_CLIP_L1;
  else if (norm_type == 2.0) code = PT_CLIP_L2;
  TORCH_CHECK_VALUE(code >= 0, "norm_type ", norm_type, ": 1, 2 or inf");
  const bool scale = max_norm >= 0.0;
  TORCH_CHECK_VALUE(!out || out->size() == grads.size(), out->size(), " outputs for ", grads.size(), " gradients");
  const Inputs in("clipping", clip_error_type);
  for (const auto& t : grads) in.check(t);
  if (out)
    for (const auto& t : *out) in.check(t);
  if (out)
    for (size_t i = 0; i < grads.size(); ++i)
      if ((*out)[i].is_neg() && !(*out)[i].is_same(grads[i]))
        raise(clip_error_type, "an output is a negated view: it cannot be written");
  check_tensors(grads, "gradients");
  if (out) {
    check_tensors(*out, "outputs");
    for (size_t i = 0; i < grads.size(); ++i) {
      const Tensor &g = grads[i], &o = (*out)[i];
      TORCH_CHECK_VALUE(o.sizes() == g.sizes(), "an output of shape ", o.sizes(), " for a gradient of shape ",
                        g.sizes());
      TORCH_CHECK_TYPE(o.scalar_type() == g.scalar_type() || o.scalar_type() == at::kFloat, "an output of type ",
                       o.scalar_type(), " for a gradient of type ", g.scalar_type());
      if (o.device() != g.device()) raise(clip_error_type, "outputs are not on the gradients' device");
      if (!dense(o) && meets_itself(o))
        raise(clip_error_type, "an output's elements share memory");
    }
  }
  if (grads.empty()) return Tensor();
  at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(grads[0].device());
  std::vector<pt_clip_tensor> table(grads.size());
  std::vector<Tensor> hold;                              // dense copies
  std::vector<std::pair<Tensor, Tensor>> back;           // (tensor, dense copy): outputs to copy back
  std::vector<size_t> aside;                             // where a copy stands for a tensor in the table
  for (size_t i = 0; i < grads.size(); ++i) {
    Tensor g = grads[i];
    const Tensor& o = out ? (*out)[i] : grads[i];
    const bool place = scale && (!out || o.is_same(g) ||                 // (in place the sign does not matter)
                                 (!g.is_neg() && o.data_ptr() == g.data_ptr() && o.scalar_type() == g.scalar_type() &&
                                  o.strides() == g.strides()));
    const bool strided = !dense(g), copied = strided || (!place && g.is_neg());
    if (place && strided && meets_itself(g))
      raise(clip_error_type,
            "a gradient's elements share memory (an expanded tensor): it cannot be clipped in place");
    if (scale && copied) aside.push_back(i);
    if (strided) g = g.contiguous();
    if (!place) g = g.resolve_neg();
    if (copied) hold.push_back(g);
    pt_clip_tensor& e = table[i];
    e.grad = g.data_ptr();
    e.n = g.numel();
    e.grad_type = type_code(g.scalar_type());
    e.out = g.data_ptr();
    e.out_type = e.grad_type;
    if (!scale) continue;
    if (place) {
      if (copied) back.emplace_back(grads[i], g);
    } else if (o.strides() == g.strides() && dense(o)) {
      e.out = o.data_ptr();
      e.out_type = type_code(o.scalar_type());
    } else {                                             // another order of the axes: through a copy
      Tensor d = at::empty_like(g, g.options().dtype(o.scalar_type()));
      e.out = d.data_ptr();
      e.out_type = type_code(o.scalar_type());
      back.emplace_back(o, d);
      if (!copied) aside.push_back(i);
    }
  }
  if (!aside.empty()) check_aside(grads, out, aside);
  const int64_t n = (int64_t)table.size();
  const size_t size = lib.clip_work(table.data(), n);
  if (!size) check_clip(PT_CLIP_ERR_ARG);
  const Tensor work = bytes(size, grads[0]);
  const Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  const auto stream = stream_of<pt_clip_stream_t>(grads[0]);
  if (scale)
    check_clip(lib.clip_grads(table.data(), n, code, max_norm, (float*)norm.data_ptr(), work.data_ptr(), stream));
  else
    check_clip(lib.clip_norm(table.data(), n, code, (float*)norm.data_ptr(), work.data_ptr(), stream));
  if (scale)
    for (size_t i = 0; i < grads.size(); ++i) written(out ? (*out)[i] : grads[i]);
  for (auto& [o, d] : back) o.copy_(d);
  return norm;
}

py::object py_fold(const std::vector<int64_t>& sizes, int64_t dim, const std::vector<std::vector<int64_t>>& strides,
                   int64_t lead) {
  std::vector<at::IntArrayRef> st(strides.begin(), strides.end());
  const auto f = fold(sizes, dim, st, lead);
  if (!f) return py::none();
  py::list v;
  for (size_t i = 0; i < st.size(); ++i) v.append(py::make_tuple(f->views[i].sb, f->views[i].sc, f->views[i].st));
  return py::make_tuple(f->b, f->c, f->n, v);
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.def("open_scan", torch::wrap_pybind_function(open_scan));
  m.def("open_clip", torch::wrap_pybind_function(open_clip));
  m.def("gated_scan", torch::wrap_pybind_function(gated_scan));
  m.def("gated_scan_step", torch::wrap_pybind_function(gated_scan_step));
  m.def("clip", torch::wrap_pybind_function(clip));
  m.def("fold", torch::wrap_pybind_function(py_fold));
  m.def("waits_on_default_stream",
        [](const Tensor& t) { return t.grad_fn() && waits_on_default_stream(t.grad_fn().get()); });
  m.def("intersect", torch::wrap_pybind_function(intersect));
  m.def("meets_itself", torch::wrap_pybind_function(meets_itself));
  m.def("disjoint", [](const std::vector<int64_t>& sizes, const std::vector<int64_t>& strides) {
    return disjoint(sizes, strides);
  });
}
