// The head's operators for Python (keyed_dropout.py, vocab_loss.py, int8_linear.py): argument
// checks, allocations, the current stream and autograd around the C entries of advpatch.h.
//
// Compiled, where the other operators are called through ctypes, because these are also
// called on single rows: a call through ctypes costs 10 to 20 us of Python against kernels
// of 2 to 9, and a Python backward pass 50 us more (the engine's thread takes the
// interpreter for it).  The C entries are those of the library that _native.py loaded
// (bind() resolves them there), so that there is one library in a process.
#include <dlfcn.h>

#include <atomic>
#include <cmath>
#include <limits>
#include <string>
#include <unordered_set>
#include <vector>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/advpatch.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- the library -----------------------------------------------------------

struct Entries {
  decltype(&po_last_error) last_error;
  decltype(&po_device_check) device_check;
  decltype(&po_dropout) dropout;
  decltype(&po_linear_ce_fwd) ce_fwd;
  decltype(&po_linear_ce_bwd) ce_bwd;
  decltype(&po_linear_ce_workspace) ce_workspace;
  decltype(&po_linear_ce_frozen_fwd) ce_frozen_fwd;
  decltype(&po_linear_ce_frozen_bwd) ce_frozen_bwd;
  decltype(&po_linear_ce_frozen_workspace) ce_frozen_workspace;
  decltype(&po_int8_linear) int8_linear;
} lib{};

void bind(const std::string& path) {
  void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_NOLOAD);
  if (!h) h = dlopen(path.c_str(), RTLD_NOW);
  if (!h) throw py::import_error(dlerror());
  Entries e{};
  auto take = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(dlsym(h, name));
    if (!fn) throw py::import_error(std::string(path) + " has no " + name + ": rebuild it");
  };
  take(e.last_error, "po_last_error");
  take(e.device_check, "po_device_check");
  take(e.dropout, "po_dropout");
  take(e.ce_fwd, "po_linear_ce_fwd");
  take(e.ce_bwd, "po_linear_ce_bwd");
  take(e.ce_workspace, "po_linear_ce_workspace");
  take(e.ce_frozen_fwd, "po_linear_ce_frozen_fwd");
  take(e.ce_frozen_bwd, "po_linear_ce_frozen_bwd");
  take(e.ce_frozen_workspace, "po_linear_ce_frozen_workspace");
  take(e.int8_linear, "po_int8_linear");
  lib = e;
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == PO_OK, what, " failed (", rc, "): ", lib.last_error());
}

// The tensors' device made current (they must share one, a gfx950), and its current stream.
struct On {
  c10::OptionalDeviceGuard guard;
  po_stream_t stream;
  explicit On(std::initializer_list<const Tensor*> ts) {
    const c10::Device d = (*ts.begin())->device();
    for (const Tensor* t : ts) {
      if (!t->defined()) continue;
      TORCH_CHECK(t->is_cuda(), "advpatch HIP ops need CUDA (ROCm) tensors; got ", t->device());
      TORCH_CHECK(t->device() == d, "advpatch HIP ops need their tensors on one device; got ", d, " and ", t->device());
    }
    static std::atomic<bool> seen[64];                        // set under whatever thread: only ever to true
    guard.reset_device(d);
    if (d.index() >= 64 || !seen[d.index()]) {
      check(lib.device_check(d.index()), "po_device_check");
      if (d.index() < 64) seen[d.index()] = true;
    }
    stream = c10::hip::getCurrentHIPStream(d.index()).stream();
  }
};

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PO_F32;
    case at::kHalf: return PO_F16;
    case at::kBFloat16: return PO_BF16;
    default: return -1;
  }
}

// t as rows over its last dimension: a view where the elements of a row are neighbours and rows
// do not overlap (and start at most `most` elements apart), else a copy.
struct Rows {
  Tensor t;
  int64_t rows, cols, ld;
  explicit Rows(const Tensor& x, int64_t most = std::numeric_limits<int64_t>::max()) {
    cols = x.size(-1);
    rows = cols ? x.numel() / cols : 0;
    t = x;
    ld = cols;
    if (x.is_contiguous()) return;
    if (x.dim() != 2) t = x.reshape({rows, cols});
    ld = rows > 1 ? t.stride(0) : cols;
    if ((cols > 1 && t.stride(1) != 1) || ld < cols || ld > most) {
      t = t.contiguous();
      ld = cols;
    }
  }
};

const Tensor& tensor_of(const py::handle& h) { return THPVariable_Unpack(h.ptr()); }
bool is_tensor(const py::handle& h) { return THPVariable_Check(h.ptr()); }
bool is_float(const py::handle& h) { return is_tensor(h) && dtype_of(tensor_of(h)) >= 0; }

// a whole number of 64 bits; anything else: ValueError
uint64_t u64(const char* name, const py::handle& h) {
  const py::object i = py::reinterpret_steal<py::object>(PyNumber_Index(h.ptr()));
  if (!i) throw py::error_already_set();
  const uint64_t v = PyLong_AsUnsignedLongLong(i.ptr());
  if (PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_VALUE(false, "keyed_dropout: ", name, " must be in [0, 2^64)");
  }
  return v;
}

bool wants_grad(const Tensor& a, const Tensor& b) {
  return at::GradMode::is_enabled() && (a.requires_grad() || (b.defined() && b.requires_grad()));
}

// A dual tensor of forward-mode differentiation: its tangent would be lost, which counts as zero.
void check_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), what);
}

// A captured backward pass ends at the gradient accumulators of the leaves that its inputs come from.
// One that an eager graph of the same leaf keeps alive belongs to that graph's stream: the engine
// makes that stream wait for the captured one, which ends the process where it is the default
// stream.  Refused here, before anything is captured.
void check_capture(const char* what, std::initializer_list<const Tensor*> inputs) {
  const Tensor& first = **inputs.begin();
  if (!first.is_cuda()) return;                               // refused later
  const c10::OptionalDeviceGuard guard(first.device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto now = c10::hip::getCurrentHIPStream(first.device().index()).id();
  auto check = [&](torch::autograd::Node& accumulator) {
    const auto stream = accumulator.stream();
    if (!stream || stream->id() == now) return;
    const c10::Device device(c10::DeviceType::HIP, stream->device_index());
    const hipStream_t other =
        c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, c10::Stream(c10::Stream::UNSAFE, device, stream->id())).stream();
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;     // another stream of the capture will do
    if (other && hipStreamIsCapturing(other, &status) == hipSuccess && status == hipStreamCaptureStatusActive) return;
    TORCH_CHECK(false, what,
                ": a graph made outside this capture still holds one of its leaves (free that graph's outputs before capturing)");
  };
  std::unordered_set<torch::autograd::Node*> seen;
  std::vector<torch::autograd::Node*> left;
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad()) continue;
    if (t->is_leaf()) {
      if (const auto node = torch::autograd::impl::try_get_grad_accumulator(*t)) check(*node);
    } else if (seen.insert(t->grad_fn().get()).second) {
      left.push_back(t->grad_fn().get());
    }
  }
  while (!left.empty()) {
    torch::autograd::Node& node = *left.back();
    left.pop_back();
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(&node)) check(node);
    for (const auto& edge : node.next_edges())
      if (edge.function && seen.insert(edge.function.get()).second) left.push_back(edge.function.get());
  }
}

// ---- dropout ---------------------------------------------------------------

struct DropoutKey {
  int64_t drop, seed, step, row0;                             // seed and step as bits
};

// y, and in *used the step taken where it is on the device
Tensor dropout_run(const Tensor& x, const Tensor& residual, const DropoutKey& k, const Tensor& step, Tensor* used) {
  On on({&x, &residual, &step});
  const Rows xr(x);
  Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  if (step.defined()) *used = at::empty({1}, step.options());
  if (x.numel() == 0) {
    if (step.defined()) used->copy_(step.reshape({1}));
    return y;
  }
  std::optional<Rows> rr;
  if (residual.defined()) rr.emplace(residual);
  check(lib.dropout(xr.t.data_ptr(), xr.ld, rr ? rr->t.data_ptr() : nullptr, rr ? rr->ld : 0, dtype_of(x), xr.rows, xr.cols,
                    (uint64_t)k.seed, (uint64_t)k.step, step.defined() ? step.const_data_ptr<int64_t>() : nullptr,
                    step.defined() ? used->data_ptr<int64_t>() : nullptr, k.row0, (int)k.drop, y.data_ptr(), xr.cols,
                    on.stream),
        "po_dropout");
  return y;
}

std::optional<Tensor> some(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& residual,
                        const std::optional<Tensor>& step, int64_t drop, int64_t seed, int64_t at_step, int64_t row0) {
    Tensor used;
    Tensor y = dropout_run(x, residual.value_or(Tensor()), {drop, seed, at_step, row0}, step.value_or(Tensor()), &used);
    ctx->saved_data["key"] = std::vector<int64_t>{drop, seed, at_step, row0, residual.has_value()};
    // the caller may move its step on before the backward pass
    if (used.defined()) ctx->save_for_backward({used});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto k = ctx->saved_data["key"].toIntVector();
    const auto saved = ctx->get_saved_variables();
    const Tensor step = saved.empty() ? Tensor() : saved[0], &dy = grads[0];
    variable_list out(7);
    if (!dy.defined()) return out;
    if (ctx->needs_input_grad(0)) {
      // the same linear map; through apply where it has to be differentiable again
      Tensor used;
      out[0] = wants_grad(dy, Tensor()) ? apply(dy, std::optional<Tensor>(), some(step), k[0], k[1], k[2], k[3])
                                        : dropout_run(dy, Tensor(), {k[0], k[1], k[2], k[3]}, step, &used);
    }
    if (k[4]) out[1] = dy;
    return out;
  }
};

Tensor keyed_dropout(const py::object& x_, double p, const py::object& seed_, const py::object& step_,
                     const py::object& row0_, const py::object& residual_) {
  TORCH_CHECK_TYPE(is_float(x_), "keyed_dropout: x must be a float32, float16 or bfloat16 tensor");
  const Tensor& x = tensor_of(x_);
  TORCH_CHECK_VALUE(x.dim() >= 1, "keyed_dropout: x needs at least one dimension");
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "keyed_dropout: p must be in [0, 1], got ", p);
  Tensor residual, step;
  if (!residual_.is_none()) {
    TORCH_CHECK_VALUE(is_tensor(residual_) && tensor_of(residual_).sizes() == x.sizes() &&
                          tensor_of(residual_).scalar_type() == x.scalar_type(),
                      "keyed_dropout: residual must have x's shape and type");
    residual = tensor_of(residual_);
  }
  DropoutKey k{};
  if (is_tensor(step_)) {
    step = tensor_of(step_);
    TORCH_CHECK_TYPE(step.scalar_type() == at::kLong && step.numel() == 1, "keyed_dropout: a step on the device is one int64");
  } else {
    k.step = (int64_t)u64("step", step_);
  }
  k.seed = (int64_t)u64("seed", seed_);
  // half a step of the probability's 2^-16 goes to the even neighbour
  k.drop = (int64_t)std::nearbyint(p * 65536.0);
  const int64_t rows = x.size(-1) ? x.numel() / x.size(-1) : 0;
  const uint64_t row0 = u64("row0", row0_);
  TORCH_CHECK_VALUE(row0 <= (1ULL << 32) && row0 + (uint64_t)rows <= (1ULL << 32),
                    "keyed_dropout: rows row0 .. row0 + rows must stay within 2^32");
  k.row0 = (int64_t)row0;
  check_tangents("keyed_dropout has no forward-mode derivative", {&x, &residual});
  py::gil_scoped_release free;
  if (wants_grad(x, residual)) {
    check_capture("keyed_dropout", {&x, &residual});
    return Dropout::apply(x, some(residual), some(step), k.drop, k.seed, k.step, k.row0);
  }
  Tensor used;
  return dropout_run(x, residual, k, step, &used);
}

// ---- cross entropy ---------------------------------------------------------

constexpr int64_t kMostStride = 1 << 21;

struct CeForward {
  Tensor loss, target, stat;                                  // stat: [3 N] statistics, then the count
  Tensor dhu;                                                 // frozen: the embeddings' gradient, [N][D up to a multiple of 4]
};

CeForward ce_forward(const Tensor& hidden, const Tensor& weight, const Tensor& target, int64_t ignore, int64_t reduction,
                     double scale, bool frozen = false) {
  On on({&hidden, &weight, &target});
  const Rows h(hidden, kMostStride), w(weight, kMostStride);
  const auto f32 = hidden.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous);
  CeForward r;
  r.target = target.reshape({-1}).contiguous();
  r.loss = reduction == 0 ? at::empty(target.sizes(), f32) : at::empty({}, f32);
  r.stat = at::empty({frozen ? 1 : 3 * h.rows + 1}, f32);
  if (frozen) r.dhu = at::empty({h.rows, (h.cols + 3) / 4 * 4}, f32);
  if (h.rows == 0) {
    if (reduction) r.loss.fill_(reduction == 2 ? std::numeric_limits<double>::quiet_NaN() : 0.0);
    return r;
  }
  int64_t bytes = 0;
  const int dt = dtype_of(hidden);
  if (frozen) {
    check(lib.ce_frozen_workspace(h.t.data_ptr(), h.ld, w.t.data_ptr(), w.ld, dt, h.rows, w.rows, h.cols, &bytes),
          "po_linear_ce_frozen_workspace");
    const Tensor ws = at::empty({bytes}, f32.dtype(at::kByte));
    check(lib.ce_frozen_fwd(h.t.data_ptr(), h.ld, w.t.data_ptr(), w.ld, dt, h.rows, w.rows, h.cols,
                            r.target.const_data_ptr<int64_t>(), ignore, (float)scale, (int)reduction, ws.data_ptr(), bytes,
                            r.loss.data_ptr<float>(), r.stat.data_ptr<float>(), r.dhu.data_ptr<float>(), on.stream),
          "po_linear_ce_frozen_fwd");
    return r;
  }
  check(lib.ce_workspace(h.t.data_ptr(), h.ld, w.t.data_ptr(), w.ld, dt, h.rows, w.rows, h.cols, 0, 0, &bytes, nullptr),
        "po_linear_ce_workspace");
  const Tensor ws = at::empty({bytes}, f32.dtype(at::kByte));
  float* stat = r.stat.data_ptr<float>();
  check(lib.ce_fwd(h.t.data_ptr(), h.ld, w.t.data_ptr(), w.ld, dt, h.rows, w.rows, h.cols, r.target.const_data_ptr<int64_t>(),
                   ignore, (float)scale, (int)reduction, ws.data_ptr(), bytes, stat, r.loss.data_ptr<float>(),
                   stat + 3 * h.rows, on.stream),
        "po_linear_ce_fwd");
  return r;
}

struct LinearCe : torch::autograd::Function<LinearCe> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& target,
                        int64_t ignore, int64_t reduction, double scale) {
    // of few rows a second pass over the vocabulary is the quicker one (1 x 65536 x 1024 bf16: 67 us against 126), and of
    // fp32 up to 128, which are multiplied as they are (100 x 30000 x 1024: 262 against 424; 192: 376 and 355)
    const bool fp32 = hidden.scalar_type() == at::kFloat;
    const bool frozen = !weight.requires_grad() && target.numel() > (fp32 ? 128 : weight.size(1) > 2048 ? 0 : 8);
    CeForward r = ce_forward(hidden, weight, target, ignore, reduction, scale, frozen);
    ctx->save_for_backward({hidden, weight, r.target, r.stat, r.dhu});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["scale"] = scale;
    return r.loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &hidden = saved[0], &weight = saved[1], &target = saved[2], &stat = saved[3];
    const bool need_h = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool again = wants_grad(grads[0], hidden) || wants_grad(weight, Tensor());
    {
      at::AutoGradMode off(false);
      const int64_t ignore = ctx->saved_data["ignore"].toInt(), reduction = ctx->saved_data["reduction"].toInt();
      if (saved[4].defined())
        out[0] = scaled(hidden, saved[4], target, stat, grads[0], ignore, reduction);
      else
        run(hidden, weight, target, stat, grads[0], ignore, reduction, ctx->saved_data["scale"].toDouble(),
            need_h ? &out[0] : nullptr, need_w ? &out[1] : nullptr);
    }
    if (again) {                                              // gradients of second order: refused where they are asked for
      auto no = std::make_shared<torch::autograd::DelayedError>("linear_cross_entropy has no gradient of second order", 4);
      variable_list marked = (*no)({out[0], out[1], hidden, weight});
      out[0] = marked[0];
      out[1] = marked[1];
    }
    return out;
  }
  // a frozen vocabulary's gradient of the embeddings: made in the forward pass
  static Tensor scaled(const Tensor& hidden, const Tensor& dhu, const Tensor& target, const Tensor& count, const Tensor& grad,
                       int64_t ignore, int64_t reduction) {
    On on({&hidden, &dhu, &grad});
    Tensor dh = at::empty(hidden.sizes(), hidden.options().memory_format(at::MemoryFormat::Contiguous));
    if (target.numel() == 0) return dh;
    const Tensor g = grad.reshape({-1}).contiguous();
    const int64_t D = hidden.size(-1);
    check(lib.ce_frozen_bwd(dhu.data_ptr<float>(), dtype_of(hidden), target.numel(), D, target.const_data_ptr<int64_t>(), ignore,
                            (int)reduction, count.data_ptr<float>(), g.const_data_ptr<float>(), dh.data_ptr(), D, on.stream),
          "po_linear_ce_frozen_bwd");
    return dh;
  }
  static void run(const Tensor& hidden, const Tensor& weight, const Tensor& target, const Tensor& stat, const Tensor& grad,
                  int64_t ignore, int64_t reduction, double scale, Tensor* dh, Tensor* dw) {
    On on({&hidden, &weight, &grad});
    const Rows h(hidden, kMostStride), w(weight, kMostStride);
    const auto contiguous = hidden.options().memory_format(at::MemoryFormat::Contiguous);
    if (dh) *dh = at::empty(hidden.sizes(), contiguous);
    if (dw) *dw = at::empty(weight.sizes(), contiguous);
    if (h.rows == 0) {
      if (dw) dw->zero_();
      return;
    }
    const Tensor g = grad.reshape({-1}).contiguous();
    const int dt = dtype_of(hidden);
    int64_t bytes = 0;
    check(lib.ce_workspace(h.t.data_ptr(), h.ld, w.t.data_ptr(), w.ld, dt, h.rows, w.rows, h.cols, dh != nullptr,
                           dw != nullptr, nullptr, &bytes),
          "po_linear_ce_workspace");
    const Tensor ws = at::empty({bytes}, contiguous.dtype(at::kByte));
    float* st = stat.data_ptr<float>();
    check(lib.ce_bwd(h.t.data_ptr(), h.ld, w.t.data_ptr(), w.ld, dt, h.rows, w.rows, h.cols, target.const_data_ptr<int64_t>(),
                     ignore, (float)scale, (int)reduction, st, st + 3 * h.rows, g.const_data_ptr<float>(), ws.data_ptr(),
                     bytes, dh ? dh->data_ptr() : nullptr, h.cols, dw ? dw->data_ptr() : nullptr, h.cols, on.stream),
          "po_linear_ce_bwd");
  }
};

Tensor linear_cross_entropy(const py::object& hidden_, const py::object& weight_, const py::object& target_, int64_t ignore,
                            const std::string& reduction, double scale) {
  TORCH_CHECK_TYPE(is_float(hidden_), "linear_cross_entropy: hidden must be a float32, float16 or bfloat16 tensor");
  TORCH_CHECK_TYPE(is_float(weight_), "linear_cross_entropy: weight must be a float32, float16 or bfloat16 tensor");
  const Tensor &hidden = tensor_of(hidden_), &weight = tensor_of(weight_);
  TORCH_CHECK_TYPE(hidden.scalar_type() == weight.scalar_type(), "linear_cross_entropy: hidden is ", hidden.scalar_type(),
                   ", weight ", weight.scalar_type());
  TORCH_CHECK_VALUE(hidden.dim() >= 1 && weight.dim() == 2 && hidden.size(-1) == weight.size(1),
                    "linear_cross_entropy: hidden [..., D] and weight [V, D] expected, got ", hidden.sizes(), " and ",
                    weight.sizes());
  TORCH_CHECK_VALUE(weight.size(0) >= 1 && weight.size(1) >= 1, "linear_cross_entropy: the vocabulary is empty");
  TORCH_CHECK_VALUE(is_tensor(target_) && tensor_of(target_).scalar_type() == at::kLong &&
                        tensor_of(target_).sizes() == hidden.sizes().slice(0, hidden.dim() - 1),
                    "linear_cross_entropy: target must be int64 of hidden's shape without its last dimension");
  const int64_t red = reduction == "none" ? 0 : reduction == "sum" ? 1 : reduction == "mean" ? 2 : -1;
  TORCH_CHECK_VALUE(red >= 0, "linear_cross_entropy: reduction must be one of none, sum, mean");
  TORCH_CHECK_VALUE(scale > 0.0 && std::isfinite(scale), "linear_cross_entropy: scale must be positive and finite, got ", scale);
  const Tensor& target = tensor_of(target_);
  check_tangents("linear_cross_entropy has no forward-mode derivative", {&hidden, &weight});
  py::gil_scoped_release free;
  if (wants_grad(hidden, weight)) {
    check_capture("linear_cross_entropy", {&hidden, &weight});
    return LinearCe::apply(hidden, weight, target, ignore, red, scale);
  }
  return ce_forward(hidden, weight, target, ignore, red, scale).loss;
}

// ---- 8-bit linear layer ----------------------------------------------------

constexpr int64_t kMaxInner = (1 << 17) - 1;

// int8 [out][K] as a view of rows that start on 128 bytes, zeros behind them, and long ones not on 256: rows a
// power of two apart fall on few memory channels (one token of 4096 x 4096 6.3 -> 5.8 us, 8192^3 507 -> 496)
Tensor lay_out(const Tensor& w) {
  int64_t ld = (w.size(1) + 127) / 128 * 128;
  if (ld >= 1024 && ld % 256 == 0) ld += 128;
  Tensor store = at::zeros({w.size(0), ld}, w.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor rows = store.narrow(1, 0, w.size(1));
  rows.copy_(w);
  return rows;
}

Tensor int8_linear(const py::object& x_, const py::object& wq_, const py::object& wscale_, const py::object& bias_) {
  TORCH_CHECK_TYPE(is_float(x_) && tensor_of(x_).dim() >= 1, "int8_linear: x must be a float32, float16 or bfloat16 tensor of rows");
  const Tensor& x = tensor_of(x_);
  const int64_t K = x.size(-1);
  TORCH_CHECK_VALUE(K >= 1 && K <= kMaxInner, "int8_linear: the inner dimension must be in [1, ", kMaxInner, "], got ", K);
  TORCH_CHECK_VALUE(is_tensor(wq_) && tensor_of(wq_).scalar_type() == at::kChar && tensor_of(wq_).dim() == 2 &&
                        tensor_of(wq_).size(1) == K && tensor_of(wq_).size(0) >= 1,
                    "int8_linear: the weights must be int8 [out, ", K, "]");
  const Tensor& wq = tensor_of(wq_);
  const int64_t N = wq.size(0);
  auto vector = [&](const py::object& o) {
    return is_tensor(o) && tensor_of(o).scalar_type() == at::kFloat && tensor_of(o).dim() == 1 && tensor_of(o).size(0) == N;
  };
  TORCH_CHECK_VALUE(vector(wscale_), "int8_linear: the weight scales must be float32 [", N, "]");
  TORCH_CHECK_VALUE(bias_.is_none() || vector(bias_), "int8_linear: the bias must be float32 [", N, "]");
  const Tensor& wscale = tensor_of(wscale_);
  const Tensor bias = bias_.is_none() ? Tensor() : tensor_of(bias_);
  TORCH_CHECK(!wants_grad(x, bias) && !wants_grad(wscale, Tensor()),
              "int8_linear has no gradient: call it under torch.no_grad() or on detached tensors");
  check_tangents("int8_linear has no gradient, nor a forward-mode derivative: call it on detached tensors", {&x, &wscale, &bias});
  py::gil_scoped_release free;
  On on({&x, &wq, &wscale, &bias});
  const Rows r(x);
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  Tensor y = at::empty(shape, x.options().memory_format(at::MemoryFormat::Contiguous));
  if (r.rows == 0) return y;
  // rows that start on 16 bytes and are laid out to a multiple of 16; else a copy
  Tensor w = wq;
  int64_t ldw = N > 1 ? w.stride(0) : (K + 15) / 16 * 16;
  if ((K > 1 && w.stride(1) != 1) || ldw % 16 || ldw < K || ldw > (1 << 22) || (uintptr_t)w.data_ptr() % 16 ||
      (N == 1 && K % 16)) {
    w = lay_out(wq);
    ldw = w.stride(0);
  }
  const Tensor sw = wscale.contiguous(), b = bias.defined() ? bias.contiguous() : bias;
  const int64_t bytes = r.rows * (K + 260);
  const Tensor ws = at::empty({bytes}, y.options().dtype(at::kByte));
  check(lib.int8_linear(r.t.data_ptr(), r.ld, w.const_data_ptr<int8_t>(), ldw, sw.const_data_ptr<float>(),
                        b.defined() ? b.const_data_ptr<float>() : nullptr, r.rows, N, K, ws.data_ptr(), bytes, y.data_ptr(), N,
                        dtype_of(x), on.stream),
        "po_int8_linear");
  return y;
}

}  // namespace

PYBIND11_MODULE(_head, m) {
  m.def("bind", &bind);
  m.def("keyed_dropout", &keyed_dropout);
  m.def("linear_cross_entropy", &linear_cross_entropy);
  m.def("int8_linear", &int8_linear);
  m.def("lay_out", [](const py::object& w) {
    TORCH_CHECK_VALUE(is_tensor(w) && tensor_of(w).scalar_type() == at::kChar && tensor_of(w).dim() == 2,
                      "lay_out: the weights must be int8 [out, K]");
    return lay_out(tensor_of(w));
  });
}
