// dgnn_torch.cpp -- what spmm_cpp's training operators do on the host, per call: checks, outputs, workspace, stream, autograd
// node, C entry. The same in Python costs 40 to 100 us a call, several times what small kernels take on the GPU. No
// arithmetic here; the C ABI's functions come from the library that spmm_cpp loaded (bind()).

#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "dgnn_train.h"

namespace {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;

struct Api {
  decltype(&dgnn_last_error) last_error;
  decltype(&dgnn_linear_workspace) workspace;
  decltype(&dgnn_linear_forward) forward;
  decltype(&dgnn_linear_slope) slope;
  decltype(&dgnn_linear_grad_input) grad_input;
  decltype(&dgnn_linear_grad_weight) grad_weight;
  decltype(&dgnn_linear_backward_workspace) backward_workspace;
  decltype(&dgnn_linear_backward) backward;
  decltype(&dgnn_adamw) adamw;
} api;

void bind(const std::vector<uintptr_t>& f) {
  if (f.size() != sizeof(Api) / sizeof(void*)) throw std::runtime_error("spmm_cpp: the torch binding and the library do not fit");
  uintptr_t* to = reinterpret_cast<uintptr_t*>(&api);
  for (size_t i = 0; i < f.size(); ++i) to[i] = f[i];
}

[[noreturn]] void refuse(const std::string& what) { throw std::runtime_error(what); }

void check(int rc, const char* what) {
  if (rc) refuse(std::string(what) + ": " + api.last_error() + " (status " + std::to_string(rc) + ")");
}

std::string text(const Tensor& t) { return std::string(c10::toString(t.scalar_type())) + " on " + t.device().str(); }
std::string shape(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return DGNN_F32;
    case at::kBFloat16: return DGNN_BF16;
    case at::kHalf: return DGNN_F16;
    default: return -1;
  }
}

void* stream_of(const Tensor& t) { return (void*)at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;

// ------------------------------------------------------------------------------------------- layer transform
struct Rows { void* p; int64_t ld; };

// The kernels take plain addresses: what else a tensor carries would be dropped without a word.
void plain(const Tensor& t, const std::string& who) {
  if (t._fw_grad(0).defined()) refuse(who + " is a dual tensor; this operator has no forward-mode derivative");
  if (t.is_neg()) refuse(who + " is a view whose values are stored negated (of a conjugate's imaginary part); call resolve_neg()");
  if (torch::jit::tracer::isTracing()) refuse(who + " is traced; torch.jit.trace cannot record this operator");
}

// a 2-D operand with unit-stride rows; `like`: the operand whose type and device it has to have
Rows rows(const Tensor& t, const char* name, const Tensor* like = nullptr) {
  const std::string who = std::string("spmm_cpp.linear: ") + name;
  if (!t.defined()) refuse(who + " is missing");
  plain(t, who);
  if (!t.is_cuda()) refuse(who + " is on " + t.device().str() + "; this operator has no CPU path");
  if (t.layout() != at::kStrided) refuse(who + " must be dense");
  if (code_of(t.scalar_type()) < 0) refuse(who + " must be fp32, bf16 or fp16, got " + c10::toString(t.scalar_type()));
  if (t.dim() != 2) refuse(who + " must have 2 dims, got " + std::to_string(t.dim()));
  if (like && (t.scalar_type() != like->scalar_type() || t.device() != like->device()))
    refuse(who + " is " + text(t) + ", the other operands are " + text(*like));
  const int64_t n = t.size(0), f = t.size(1);
  if (f > 1 && t.stride(1) != 1) refuse(who + " must be row-major (stride(1) == 1)");
  if (n > 1 && t.stride(0) < f) refuse(who + " has overlapping rows");
  return {t.data_ptr(), n > 1 ? t.stride(0) : std::max<int64_t>(f, 1)};
}

Rows rows(const MaybeTensor& t, const char* name, const Tensor& like, int64_t m, int64_t n) {
  if (!t || !t->defined()) return {nullptr, 0};
  const Rows r = rows(*t, name, &like);
  if (t->size(0) != m || t->size(1) != n)
    refuse(std::string("spmm_cpp.linear: ") + name + " is " + shape(*t) + ", expected (" + std::to_string(m) + ", " + std::to_string(n) + ")");
  return r;
}

void* vector(const MaybeTensor& t, const char* name, int64_t n, const Tensor& like) {
  if (!t || !t->defined()) return nullptr;
  plain(*t, std::string("spmm_cpp.linear: ") + name);
  if (t->dim() != 1 || t->numel() != n || t->scalar_type() != like.scalar_type() || t->device() != like.device() || !t->is_contiguous())
    refuse(std::string("spmm_cpp.linear: ") + name + " must be a contiguous vector of " + std::to_string(n) + " " + text(like));
  return t->data_ptr();
}

// Workspaces come from the caching allocator at every call: calls on different streams, and captured graphs, each have theirs.
Tensor room(int64_t bytes, const Tensor& like) { return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor(); }
void* at_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor workspace(int pass, int64_t M, int64_t K, int64_t N, const Tensor& like, int64_t* bytes) {
  check(api.workspace(pass, M, K, N, code_of(like.scalar_type()), bytes), "linear_workspace");
  return room(*bytes, like);
}

std::pair<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w, const MaybeTensor& bias, int64_t act, const MaybeTensor& residual, bool save) {
  const Rows a = rows(x, "x"), b = rows(w, "weight", &x);
  const int64_t M = x.size(0), K = x.size(1), N = w.size(1);
  if (w.size(0) != K) refuse("spmm_cpp.linear: shape mismatch x" + shape(x) + " weight" + shape(w));
  void* const v = vector(bias, "bias", N, x);
  const Rows r = rows(residual, "residual", x, M, N);
  const Guard guard(x.device());
  Tensor y = at::empty({M, N}, x.options()), saved;
  if (save && act) saved = act == DGNN_ACT_RELU ? at::empty({M, (N + 31) / 32}, x.options().dtype(at::kInt)) : at::empty({M, N}, x.options().dtype(at::kFloat));
  if (M && N) {
    int64_t bytes;
    const Tensor ws = workspace(DGNN_LINEAR_FORWARD, M, K, N, x, &bytes);
    check(api.forward(a.p, a.ld, b.p, b.ld, v, r.p, r.ld, y.data_ptr(), N, at_of(saved), saved.defined() ? saved.size(1) : 0, M, K, N,
                      code_of(x.scalar_type()), (int32_t)act, at_of(ws), bytes, stream_of(x)), "linear_forward");
  }
  return {y, saved};
}

std::pair<Tensor, Tensor> linear_slope(const Tensor& dy, const MaybeTensor& saved, int64_t act, bool need_bias) {
  const Rows d = rows(dy, "dy");
  const int64_t M = dy.size(0), N = dy.size(1);
  if (act) {
    const int64_t wide = act == DGNN_ACT_RELU ? (N + 31) / 32 : N;
    const auto type = act == DGNN_ACT_RELU ? at::kInt : at::kFloat;
    if (!saved || !saved->defined() || saved->dim() != 2 || saved->size(0) != M || saved->size(1) != wide || saved->scalar_type() != type
        || saved->device() != dy.device() || !saved->is_contiguous())
      refuse("spmm_cpp.linear: saved must be what linear_forward returned for this activation and shape");
  }
  if (!act && !need_bias) return {dy, Tensor()};
  const Guard guard(dy.device());
  Tensor p = act ? at::empty({M, N}, dy.options()) : dy, db;
  int64_t bytes = 0;
  Tensor ws;
  if (need_bias) {
    db = at::empty({N}, dy.options());
    ws = workspace(DGNN_LINEAR_SLOPE, M, 0, N, dy, &bytes);
  }
  check(api.slope(d.p, d.ld, act ? saved->data_ptr() : nullptr, act ? std::max<int64_t>(saved->size(1), 1) : 0, act ? p.data_ptr() : nullptr,
                  std::max<int64_t>(N, 1), at_of(db), M, N, code_of(dy.scalar_type()), (int32_t)act, at_of(ws), bytes, stream_of(dy)), "linear_slope");
  return {p, db};
}

Tensor linear_grad_input(const Tensor& p, const Tensor& w, const MaybeTensor& add) {
  const Rows a = rows(p, "p"), b = rows(w, "weight", &p);
  const int64_t M = p.size(0), N = p.size(1), K = w.size(0);
  if (w.size(1) != N) refuse("spmm_cpp.linear: shape mismatch p" + shape(p) + " weight" + shape(w));
  const Rows r = rows(add, "add", p, M, K);
  const Guard guard(p.device());
  Tensor dx = at::empty({M, K}, p.options());
  if (M && K) {
    int64_t bytes;
    const Tensor ws = workspace(DGNN_LINEAR_GRAD_INPUT, M, K, N, p, &bytes);
    check(api.grad_input(a.p, a.ld, b.p, b.ld, r.p, r.ld, dx.data_ptr(), K, M, K, N, code_of(p.scalar_type()), at_of(ws), bytes, stream_of(p)),
          "linear_grad_input");
  }
  return dx;
}

Tensor linear_grad_weight(const Tensor& x, const Tensor& p) {
  const Rows a = rows(x, "x"), b = rows(p, "p", &x);
  const int64_t M = x.size(0), K = x.size(1), N = p.size(1);
  if (p.size(0) != M) refuse("spmm_cpp.linear: shape mismatch x" + shape(x) + " p" + shape(p));
  const Guard guard(x.device());
  Tensor dw = at::empty({K, N}, x.options());
  if (K && N) {
    int64_t bytes;
    const Tensor ws = workspace(DGNN_LINEAR_GRAD_WEIGHT, M, K, N, x, &bytes);
    check(api.grad_weight(a.p, a.ld, b.p, b.ld, dw.data_ptr(), N, M, K, N, code_of(x.scalar_type()), at_of(ws), bytes, stream_of(x)),
          "linear_grad_weight");
  }
  return dw;
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const MaybeTensor& bias, const MaybeTensor& residual, int64_t act) {
    const bool gx = x.requires_grad(), gw = w.requires_grad(), gb = bias && bias->defined() && bias->requires_grad();
    auto [y, saved] = linear_forward(x, w, bias, act, residual, gx || gw || gb);
    ctx->save_for_backward({gw ? x : Tensor(), gx ? w : Tensor(), saved});
    const bool gr = residual && residual->defined() && residual->requires_grad();
    ctx->saved_data["how"] = (int64_t)(act | gx << 4 | gw << 5 | gb << 6 | gr << 7) | x.size(1) << 8;
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (at::GradMode::is_enabled()) refuse("spmm_cpp.linear: no second derivative (create_graph=True)");
    const int64_t how = ctx->saved_data["how"].toInt(), K = how >> 8;
    const int act = how & 15;
    const bool gx = how >> 4 & 1, gw = how >> 5 & 1, gb = how >> 6 & 1, gr = how >> 7 & 1;
    const auto kept = ctx->get_saved_variables();
    Tensor dy = grads[0], dx, dw, db;
    const int64_t M = dy.size(0), N = dy.size(1);
    if (gx || gw || gb) {
      dy = dy.resolve_neg();
      if ((N > 1 && dy.stride(1) != 1) || (M > 1 && dy.stride(0) < N)) dy = dy.contiguous();       // expanded or transposed
      const Rows d = rows(dy, "the gradient");
      const Guard guard(dy.device());
      const int code = code_of(dy.scalar_type());
      int64_t bytes;
      check(api.backward_workspace(M, K, N, code, act, &bytes), "linear_backward");
      const Tensor ws = room(bytes, dy);
      Rows a{nullptr, 0}, b{nullptr, 0};
      if (gw) { a = rows(kept[0], "x", &dy); dw = at::empty({K, N}, dy.options()); }
      if (gx) { b = rows(kept[1], "weight", &dy); dx = at::empty({M, K}, dy.options()); }
      if (gb) db = at::empty({N}, dy.options());
      const Tensor& saved = kept[2];
      check(api.backward(a.p, a.ld, b.p, b.ld, d.p, d.ld, at_of(saved), saved.defined() ? std::max<int64_t>(saved.size(1), 1) : 0, at_of(dx),
                         std::max<int64_t>(K, 1), at_of(dw), std::max<int64_t>(N, 1), at_of(db), M, K, N, code, act, at_of(ws), bytes, stream_of(dy)),
            "linear_backward");
    }
    return {dx, dw, db, gr ? dy : Tensor(), Tensor()};
  }
};

Tensor linear(const Tensor& x, const Tensor& w, const MaybeTensor& bias, int64_t act, const MaybeTensor& residual) {
  const auto wants = [](const MaybeTensor& t) { return t && t->defined() && t->requires_grad(); };
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || wants(bias) || wants(residual)))
    return Linear::apply(x, w, bias, residual, act);
  return linear_forward(x, w, bias, act, residual, false).first;
}

// ------------------------------------------------------------------------------------------- AdamW
// The parameters of one optimiser segment and where their state lies; collect() reads and checks their gradients, launch()
// steps what it found.
struct AdamTable {
  std::vector<Tensor> params;
  std::vector<dgnn_adamw_tensor> table, live;
  std::vector<size_t> which;        // live's parameters
  std::vector<Tensor> kept;         // gradients that had to be made contiguous
  double lr = 0, b1 = 0, b2 = 0, eps = 0;
  dgnn_adamw_state state{};
  Tensor steps;                     // host counters, or the device's where the step can be captured
  bool capturable;
  int bits;
  at::ScalarType dtype;
  at::Device device;

  AdamTable(const std::vector<Tensor>& p, const std::vector<int64_t>& starts, int bits_, const Tensor& m, const Tensor& v, const MaybeTensor& ms,
            const MaybeTensor& vs, const MaybeTensor& master, const Tensor& steps_, const MaybeTensor& factors)
      : params(p), steps(steps_), capturable(factors.has_value()), bits(bits_), dtype(p.at(0).scalar_type()), device(p.at(0).device()) {
    state.exp_avg = m.data_ptr();
    state.exp_avg_sq = v.data_ptr();
    if (ms) state.exp_avg_scale = ms->data_ptr<float>();
    if (vs) state.exp_avg_sq_scale = vs->data_ptr<float>();
    if (master) state.master = master->data_ptr<float>();
    if (factors) {
      state.steps = steps.data_ptr<int64_t>();
      state.factors = factors->data_ptr<float>();
    }
    for (size_t i = 0; i < p.size(); ++i) {
      dgnn_adamw_tensor t{};
      t.numel = p[i].numel();
      t.start = starts.at(i);
      t.index = (int32_t)i;
      table.push_back(t);
    }
  }

  // the parameters that have a gradient; returns how many
  int64_t collect(double lr_, double b1_, double b2_, double eps_, double decay) {
    lr = lr_, b1 = b1_, b2 = b2_, eps = eps_;
    live.clear();
    which.clear();
    kept.clear();
    int64_t* const count = capturable ? nullptr : steps.data_ptr<int64_t>();
    int64_t last = -1;
    float rate = 0.f, root = 0.f;
    for (size_t i = 0; i < params.size(); ++i) {
      const Tensor& p = params[i];
      Tensor g = p.grad();
      if (!g.defined()) continue;
      if (p.scalar_type() != dtype || p.device() != device || p.numel() != table[i].numel || !p.is_contiguous())
        refuse("AdamW: parameter " + std::to_string(i) + " is not the contiguous " + c10::toString(dtype) + " tensor of " +
               std::to_string(table[i].numel) + " elements on " + device.str() + " any more that its state was made for");
      if (g.layout() != at::kStrided || g.scalar_type() != dtype || g.device() != device || g.sizes() != p.sizes())
        refuse("AdamW: the gradient of parameter " + std::to_string(i) + " is not a dense " + c10::toString(dtype) + " tensor of its shape on " + device.str());
      if (!g.is_contiguous() || g.is_neg()) {
        g = g.resolve_neg().contiguous();
        kept.push_back(g);
      }
      dgnn_adamw_tensor t = table[i];
      t.param = p.data_ptr();
      t.grad = g.data_ptr();
      t.decay = (float)(1.0 - lr * decay);
      if (!capturable) {
        const int64_t turn = count[i] + 1;
        if (turn != last) {
          last = turn;
          rate = (float)(lr / (1.0 - std::pow(b1, (double)turn)));
          root = (float)(1.0 / std::sqrt(1.0 - std::pow(b2, (double)turn)));
        }
        t.rate = rate;
        t.root = root;
        t.turn = (uint32_t)turn;
      }
      live.push_back(t);
      which.push_back(i);
    }
    return (int64_t)live.size();
  }

  void launch() {
    int64_t* const count = capturable ? nullptr : steps.data_ptr<int64_t>();
    const Guard guard(device);
    check(api.adamw(live.data(), (int32_t)live.size(), code_of(dtype), bits, &state, lr, b1, b2, eps, stream_of(params[0])), "adamw");
    for (size_t i : which) {
      if (!capturable) ++count[i];
      // the kernel writes behind autograd's back: a graph that saved a parameter has to notice
      if (!params[i].is_inference()) params[i].unsafeGetTensorImpl()->bump_version();
    }
    kept.clear();
  }
};

// whether two sequences hold the same objects (comparing tensors would compare their elements)
bool same_objects(const py::object& a, const py::object& b) {
  const auto x = py::reinterpret_steal<py::object>(PySequence_Fast(a.ptr(), "AdamW: a sequence of parameters")),
             y = py::reinterpret_steal<py::object>(PySequence_Fast(b.ptr(), "AdamW: a sequence of parameters"));
  if (!x || !y) throw py::error_already_set();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(x.ptr());
  return n == PySequence_Fast_GET_SIZE(y.ptr()) && std::equal(PySequence_Fast_ITEMS(x.ptr()), PySequence_Fast_ITEMS(x.ptr()) + n, PySequence_Fast_ITEMS(y.ptr()));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("linear", &linear);
  m.def("linear_forward", &linear_forward);
  m.def("linear_slope", &linear_slope);
  m.def("linear_grad_input", &linear_grad_input);
  m.def("linear_grad_weight", &linear_grad_weight);
  m.def("same_objects", &same_objects);
  py::class_<AdamTable>(m, "AdamTable")
      .def(py::init<const std::vector<Tensor>&, const std::vector<int64_t>&, int, const Tensor&, const Tensor&, const MaybeTensor&, const MaybeTensor&,
                    const MaybeTensor&, const Tensor&, const MaybeTensor&>())
      .def("collect", &AdamTable::collect)
      .def("launch", &AdamTable::launch);
}
