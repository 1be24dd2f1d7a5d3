// Host side of sgpo_amd.train_ops: argument checks, memory from torch's allocator, the autograd tape, and one call into libsgpo_hip.so per
// operator.  In C++ because the smallest of these kernels take 3 us and the same steps in Python 10 to 25, and because autograd runs a backward
// pass on a thread of its own, where Python code costs two to three times as much again (measured on the training step of 7616 tokens with 31
// classes: forward and backward 128 us through torch.autograd.Function, 70 to 82 so).
//
// The library's functions are handed over by address (bind), so that this module uses the one library that sgpo_amd._lib loaded.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <atomic>
#include <map>
#include <optional>
#include <sstream>
#include <string>

#include "../../include/sgpo_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw Refused(s.str());
}
#define REQUIRE(cond, ...)         \
  do {                             \
    if (!(cond)) refuse(__VA_ARGS__); \
  } while (0)

struct Library {
  decltype(&sgpo_init) init;
  decltype(&sgpo_last_error) last_error;
  decltype(&sgpo_rotary) rotary;
  decltype(&sgpo_linear_ce_workspace_bytes) ce_bytes;
  decltype(&sgpo_linear_ce_forward) ce_forward;
  decltype(&sgpo_linear_ce_backward) ce_backward;
  decltype(&sgpo_newton_schulz_workspace_bytes) ns_bytes;
  decltype(&sgpo_newton_schulz) newton_schulz;
  decltype(&sgpo_muon_step) muon_step;
} lib = {};

void check(int rc, const char* what) {
  if (rc) refuse(what, " failed (", rc, "): ", lib.last_error());
}

std::atomic<int> bound{-1};   // the device this process has been bound to

// A call's tensors, all on one GPU, which is (or becomes) the one the process is bound to and is current while the object lives.
struct Call {
  c10::Device dev;
  c10::DeviceGuard guard;
  static c10::Device device_of(std::initializer_list<const Tensor*> ts) {
    REQUIRE(!torch::jit::tracer::isTracing(), "a trace would hold this call's result as a constant: trace around it");
    for (const Tensor* t : ts)
      if (t && t->defined()) REQUIRE(t->has_storage() && !t->_is_zerotensor(), "a tensor without memory of its own ", t->sizes(), " ", t->dtype(), " (of a torch.func transform, say, or sparse)");
    for (const Tensor* t : ts)
      if (t && t->defined()) REQUIRE(!t->is_neg(), "a lazily negated view ", t->sizes(), " ", t->dtype(), ": resolve_neg() it first");
    const Tensor* first = nullptr;
    for (const Tensor* t : ts) {
      if (!t || !t->defined()) continue;
      REQUIRE(t->is_cuda(), "host tensor ", t->sizes(), " ", t->dtype(), " passed where the library expects device memory");
      if (!first) first = t;
      REQUIRE(t->device() == first->device(), "tensors on ", first->device(), " and on ", t->device());
    }
    return first->device();
  }
  explicit Call(std::initializer_list<const Tensor*> ts) : dev(device_of(ts)), guard(dev) {
    if (bound.load(std::memory_order_relaxed) != dev.index()) {
      check(lib.init(dev.index()), "sgpo_init");
      bound = dev.index();
    }
  }
  void* stream() const { return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream(); }
};

const Tensor* opt(const OptTensor& t) { return t && t->defined() ? &*t : nullptr; }

int dtype_of(const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kFloat) return SGPO_DTYPE_F32;
  REQUIRE(t.scalar_type() == at::kBFloat16, what, " must be float32 or bfloat16, got ", t.dtype());
  return SGPO_DTYPE_BF16;
}

// scratch of one call, 256-byte aligned; from torch's allocator, which keeps streams and captured graphs apart
struct Scratch {
  Tensor buf;
  void* at;
  Scratch(size_t bytes, c10::Device dev) : buf(at::empty({(int64_t)bytes + 256}, at::TensorOptions().dtype(at::kByte).device(dev))) {
    at = (void*)(((uintptr_t)buf.data_ptr() + 255) & ~(uintptr_t)255);
  }
};

bool records(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t && t->defined() && t->requires_grad()) return true;
  return false;
}

// a gradient or tangent as memory that holds its values: autograd may hand over lazily negated views, and zeros that have none
Tensor resolved(const Tensor& t) { return t._is_zerotensor() ? at::zeros(t.sizes(), at::TensorOptions().dtype(t.scalar_type()).device(t.device())) : t.resolve_neg(); }

bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
void no_tangents(std::initializer_list<const Tensor*> ts, const char* what) {
  for (const Tensor* t : ts)
    if (t && t->defined()) REQUIRE(!has_tangent(*t), what, " has no forward-mode derivative: detach its inputs");
}

// ------------------------------------------------------------------------------------------------------------- rotation
variable_list rotate(Tensor q, Tensor k, const Tensor& freq, const Tensor& pos, bool interleaved, double scale, bool inverse, bool in_place) {
  const Call call({&q, &k, &freq, &pos});
  sgpo_rotary_args a = {};
  a.dtype = dtype_of(q, "q");
  REQUIRE(q.dim() == 4, "heads are (batch, tokens, heads, head_dim), got ", q.sizes());
  const int64_t B = q.size(0), L = q.size(1), D = q.size(3), rot = 2 * freq.numel();
  if (k.defined())
    REQUIRE(k.dim() == 4 && k.scalar_type() == q.scalar_type() && k.size(0) == B && k.size(1) == L && k.size(3) == D, "k ", k.sizes(), " ", k.dtype(), " does not match q ",
            q.sizes(), " ", q.dtype());
  REQUIRE(freq.scalar_type() == at::kDouble && freq.dim() == 1 && freq.is_contiguous(), "frequencies must be a contiguous float64 vector");
  REQUIRE(rot <= D, rot, " rotated elements in heads of ", D);
  REQUIRE(B < INT_MAX && L < INT_MAX && D <= 4096 && q.size(2) < INT_MAX && (!k.defined() || k.size(2) < INT_MAX), "heads ", q.sizes(), " over the supported range");
  if (pos.defined()) {
    const int64_t n = pos.dim();
    REQUIRE(pos.scalar_type() == at::kLong && (n == 1 || n == 2) && pos.size(-1) == L && (n == 1 || pos.size(0) == B || pos.size(0) == 1), "positions must be int64 for ", B, " x ", L,
            " tokens, got ", pos.sizes(), " ", pos.dtype());
    a.positions = pos.const_data_ptr<int64_t>();
    a.pos_stride_l = pos.stride(-1);
    a.pos_stride_b = n == 2 && pos.size(0) > 1 ? pos.stride(0) : 0;
  }
  Tensor out[2];
  for (int w = 0; w < 2; ++w) {
    Tensor& x = w ? k : q;
    if (!x.defined()) continue;
    if (in_place) {
      REQUIRE(D <= 1 || x.stride(3) == 1, "in place, the elements of a head must be contiguous");
      out[w] = x;
    } else {
      if (D > 1 && x.stride(3) != 1) x = x.contiguous();
      out[w] = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    }
    for (int i = 0; i < 3; ++i) {
      (w ? a.k_stride : a.q_stride)[i] = x.stride(i);
      (w ? a.k_out_stride : a.q_out_stride)[i] = out[w].stride(i);
    }
    (w ? a.k : a.q) = x.const_data_ptr();
    (w ? a.k_out : a.q_out) = out[w].data_ptr();
    (w ? a.heads_k : a.heads_q) = (int)x.size(2);
  }
  a.frequencies = freq.const_data_ptr<double>();
  a.B = (int)B; a.L = (int)L; a.head_dim = (int)D; a.rot = (int)rot;
  a.interleaved = interleaved; a.inverse = inverse; a.scale = (float)scale;
  check(lib.rotary(&a, call.stream()), "sgpo_rotary");
  return {out[0], out[1]};
}

// rotate, with the derivatives of both modes in q and k
variable_list turn(const Tensor& q, const Tensor& k, const Tensor& freq, const Tensor& pos, bool interleaved, double scale, bool inverse);

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& freq, const OptTensor& pos, bool interleaved, double scale, bool inverse) {
    const Tensor none, kk = k.value_or(none), pp = pos.value_or(none);
    ctx->save_for_backward({freq, pp});
    ctx->saved_data["how"] = (int64_t)((interleaved ? 1 : 0) | (inverse ? 2 : 0) | (kk.defined() ? 4 : 0));
    ctx->saved_data["scale"] = scale;
    variable_list out = rotate(q, kk, freq, pp, interleaved, scale, inverse, false);
    if (!kk.defined()) out.pop_back();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const int64_t how = ctx->saved_data["how"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    // the transposed rotation, itself differentiable where a second derivative is asked for
    const variable_list d = turn(resolved(g[0]), how & 4 ? resolved(g[1]) : Tensor(), saved[0], saved[1], how & 1, scale, !(how & 2));
    return {d[0], d[1], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

variable_list turn(const Tensor& q, const Tensor& k, const Tensor& freq, const Tensor& pos, bool interleaved, double scale, bool inverse) {
  const bool dq = has_tangent(q), dk = k.defined() && has_tangent(k);
  if (dq || dk) {   // linear: a tangent turns like its heads
    Tensor value[2] = {q, k}, tangent[2];
    for (int w = 0; w < 2; ++w) {
      if (!(w ? dk : dq)) continue;
      std::tie(value[w], tangent[w]) = at::_unpack_dual(value[w], 0);
      tangent[w] = resolved(tangent[w]);
    }
    variable_list out = turn(value[0], value[1], freq, pos, interleaved, scale, inverse);
    const variable_list t = turn(tangent[dq ? 0 : 1], dq ? tangent[1] : Tensor(), freq, pos, interleaved, scale, inverse);
    if (dq) out[0] = at::_make_dual(out[0], t[0], 0);
    if (dk) out[1] = at::_make_dual(out[1], t[dq ? 1 : 0], 0);
    return out;
  }
  if (!records({&q, &k})) return rotate(q, k, freq, pos, interleaved, scale, inverse, false);
  variable_list out = Rotary::apply(q, k.defined() ? OptTensor(k) : std::nullopt, freq, pos.defined() ? OptTensor(pos) : std::nullopt, interleaved, scale, inverse);
  out.resize(2);
  return out;
}

std::pair<Tensor, OptTensor> rotary_positions(const Tensor& q, const OptTensor& k, const Tensor& freq, const OptTensor& pos, bool interleaved, double scale) {
  REQUIRE(!records({&freq}), "rotary_positions has no gradient for the frequencies: detach them");
  REQUIRE(!has_tangent(freq), "rotary_positions has no derivative for the frequencies: detach them");
  Call::device_of({&q, opt(k), &freq, opt(pos)});
  const variable_list out = turn(q, k.value_or(Tensor()), freq, pos.value_or(Tensor()), interleaved, scale, false);
  return {out[0], opt(k) ? OptTensor(out[1]) : std::nullopt};
}

void rotary_positions_(const Tensor& q, const OptTensor& k, const Tensor& freq, const OptTensor& pos, bool interleaved, double scale) {
  REQUIRE(!records({&freq}), "rotary_positions has no gradient for the frequencies: detach them");
  REQUIRE(!records({&q, opt(k)}), "rotary_positions_ has no gradient: use rotary_positions");
  no_tangents({&q, opt(k), &freq}, "rotary_positions_");
  rotate(q, k.value_or(Tensor()), freq, pos.value_or(Tensor()), interleaved, scale, false, true);
  // what autograd saved of them is stale now
  if (!q.is_inference()) q.unsafeGetTensorImpl()->bump_version();
  if (opt(k) && !k->is_inference()) k->unsafeGetTensorImpl()->bump_version();
}

// ----------------------------------------------------------------------------------------------------------------- loss
Tensor rows(const Tensor& t) {   // contiguous rows that do not overlap, of a pitch that the library takes
  return t.stride(1) == 1 && (t.size(0) <= 1 || (t.stride(0) >= t.size(1) && t.stride(0) < 1 << 22)) ? t : t.contiguous();
}

sgpo_linear_ce_args ce_args(const Tensor& h, const Tensor& w, const Tensor& t, const Tensor& b, int64_t ignore, int64_t reduction) {
  sgpo_linear_ce_args a = {};
  a.hidden = h.const_data_ptr(); a.weight = w.const_data_ptr(); a.targets = t.const_data_ptr<int64_t>();
  a.bias = b.defined() ? b.const_data_ptr<float>() : nullptr;
  a.N = (int)h.size(0); a.H = (int)h.size(1); a.V = (int)w.size(0);
  a.ld_hidden = a.N > 1 ? h.stride(0) : a.H;
  a.ld_weight = a.V > 1 ? w.stride(0) : a.H;
  a.ignore_index = ignore; a.dtype = dtype_of(h, "hidden"); a.reduction = (int)reduction;
  return a;
}

// (loss or losses, state of the backward pass: the tokens' log-sums, the gradient's factor, and losses that are only summed)
std::pair<Tensor, Tensor> ce_forward(const Tensor& h, const Tensor& w, const Tensor& t, const Tensor& b, int64_t ignore, int64_t reduction) {
  const Call call({&h, &w, &t, &b});
  const sgpo_linear_ce_args a = ce_args(h, w, t, b, ignore, reduction);
  const size_t need = lib.ce_bytes(&a, 0);
  const Scratch ws(need, call.dev);
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(call.dev);
  const int64_t N = a.N;
  Tensor state = at::empty({reduction ? 2 * N + 1 : N + 1}, f32);
  Tensor out = reduction ? at::empty({}, f32) : at::empty({N}, f32);
  float *lse = state.data_ptr<float>(), *inv = lse + N, *o = out.data_ptr<float>();
  check(lib.ce_forward(&a, reduction ? inv + 1 : o, lse, o, inv, ws.at, need, call.stream()), "sgpo_linear_ce_forward");
  return {out, state};
}

// first derivatives, tied to what they depend on by a node that refuses to be differentiated
struct NoSecond : torch::autograd::Function<NoSecond> {
  static variable_list forward(AutogradContext*, const Tensor& g, const Tensor& h, const Tensor& w, const OptTensor& b, const variable_list& d) {
    variable_list out;
    for (const Tensor& x : d) out.push_back(x.detach());
    return out;
  }
  [[noreturn]] static variable_list backward(AutogradContext*, variable_list) { refuse("linear_cross_entropy can be differentiated once"); }
};

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& w, const Tensor& t, const OptTensor& b, int64_t ignore, int64_t reduction) {
    const Tensor bias = b.value_or(Tensor());
    auto [out, state] = ce_forward(h, w, t, bias, ignore, reduction);
    ctx->save_for_backward({h, w, t, bias, state});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["how"] = (int64_t)(reduction | (h.requires_grad() ? 4 : 0) | (w.requires_grad() ? 8 : 0) | (bias.defined() && bias.requires_grad() ? 16 : 0));
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool again = at::GradMode::is_enabled();
    variable_list d(3);
    {
      at::AutoGradMode off(false);
      const auto s = ctx->get_saved_variables();
      const int64_t how = ctx->saved_data["how"].toInt();
      no_tangents({&grads[0]}, "the gradient of linear_cross_entropy");
      const Call call({&s[0]});
      const sgpo_linear_ce_args a = ce_args(s[0], s[1], s[2], s[3], ctx->saved_data["ignore"].toInt(), how & 3);
      const Tensor g = resolved(grads[0]).contiguous();
      void* out[3] = {nullptr, nullptr, nullptr};
      const Tensor* like[3] = {&s[0], &s[1], &s[3]};
      for (int i = 0; i < 3; ++i)
        if (how & (4 << i)) {
          d[i] = at::empty(like[i]->sizes(), like[i]->options().memory_format(at::MemoryFormat::Contiguous));
          out[i] = d[i].data_ptr();
        }
      const size_t need = lib.ce_bytes(&a, 1);
      const Scratch ws(need, call.dev);
      const float* lse = s[4].const_data_ptr<float>();
      check(lib.ce_backward(&a, lse, g.const_data_ptr<float>(), lse + a.N, out[0], out[1], (float*)out[2], ws.at, need, call.stream()), "sgpo_linear_ce_backward");
    }
    if (again) {   // a graph of this pass is asked for: going through it is an error
      const auto s = ctx->get_saved_variables();
      variable_list live;
      for (const Tensor& x : d) if (x.defined()) live.push_back(x);
      live = NoSecond::apply(grads[0], s[0], s[1], s[3].defined() ? OptTensor(s[3]) : std::nullopt, live);
      size_t k = 0;
      for (Tensor& x : d) if (x.defined()) x = live[k++];
    }
    return {d[0], d[1], Tensor(), d[2], Tensor(), Tensor()};
  }
};

Tensor linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& targets, const OptTensor& bias, int64_t ignore, const std::string& reduction) {
  no_tangents({&hidden, &weight, opt(bias)}, "linear_cross_entropy");
  Call::device_of({&hidden, &weight, &targets, opt(bias)});
  dtype_of(hidden, "hidden");
  REQUIRE(hidden.dim() >= 1 && weight.dim() == 2 && hidden.size(-1) == weight.size(1) && weight.numel() > 0, "hidden ", hidden.sizes(), " does not match weight ", weight.sizes());
  REQUIRE(weight.scalar_type() == hidden.scalar_type(), "hidden is ", hidden.dtype(), " and weight ", weight.dtype());
  REQUIRE(targets.scalar_type() == at::kLong && targets.sizes() == hidden.sizes().slice(0, hidden.dim() - 1), "targets ", targets.sizes(), " ", targets.dtype(), " for hidden ", hidden.sizes());
  REQUIRE(!opt(bias) || ((bias->scalar_type() == at::kFloat || bias->scalar_type() == weight.scalar_type()) && bias->dim() == 1 && bias->size(0) == weight.size(0)),
          "bias must be float32 or of weight's type, with one value per class");
  const int64_t red = reduction == "none" ? SGPO_REDUCE_NONE : reduction == "mean" ? SGPO_REDUCE_MEAN : reduction == "sum" ? SGPO_REDUCE_SUM : -1;
  REQUIRE(red >= 0, "unknown reduction '", reduction, "'");
  REQUIRE(targets.numel() <= (1 << 30) && weight.size(0) <= (1 << 30) && weight.size(1) <= (1 << 20), "hidden ", hidden.sizes(), " and weight ", weight.sizes(), " over the supported range");
  const Tensor h = rows(hidden.dim() == 2 ? hidden : hidden.reshape({-1, hidden.size(-1)})), w = rows(weight);
  const Tensor t = targets.dim() == 1 && targets.is_contiguous() ? targets : targets.reshape({-1}).contiguous();
  const OptTensor b = opt(bias) ? OptTensor(bias->to(at::kFloat).contiguous()) : std::nullopt;   // bf16: its gradient is rounded by the same step on the tape
  Tensor out = records({&hidden, &weight, opt(bias)}) ? LinearCrossEntropy::apply(h, w, t, b, ignore, red) : ce_forward(h, w, t, b.value_or(Tensor()), ignore, red).first;
  return red == SGPO_REDUCE_NONE && targets.dim() != 1 ? out.view(targets.sizes()) : out;
}

// -------------------------------------------------------------------------------------------------------------- updates
void check_table(const std::vector<float>& c, int64_t steps) {
  REQUIRE(steps >= 1 && steps <= 64 && (int64_t)c.size() == 3 * steps, steps, " steps need ", steps, " coefficient triples (1 to 64)");
}

Tensor newton_schulz(const Tensor& update, int64_t steps, const std::vector<float>& table, double eps) {
  REQUIRE(!records({&update}), "newton_schulz has no gradient: detach the update, or call it under torch.no_grad()");
  no_tangents({&update}, "newton_schulz");
  const Call call({&update});
  const int dt = dtype_of(update, "update");
  REQUIRE(update.dim() >= 2, "an update is a matrix or a batch of them, got ", update.sizes());
  check_table(table, steps);
  at::AutoGradMode off(false);
  const int64_t m = update.size(-2), n = update.size(-1);
  Tensor out = at::empty(update.sizes(), at::TensorOptions().dtype(at::kBFloat16).device(call.dev));
  if (!update.numel()) return out;
  const int64_t batch = update.numel() / (m * n);
  REQUIRE(m < INT_MAX && n < INT_MAX && batch < INT_MAX, "updates ", update.sizes(), " over the supported range");
  Tensor u = update.dim() == 3 ? update : update.reshape({batch, m, n});
  if ((n > 1 && u.stride(2) != 1) || (m > 1 && u.stride(1) < n)) u = u.contiguous();
  const size_t need = lib.ns_bytes((int)batch, (int)m, (int)n);
  const Scratch ws(need, call.dev);
  check(lib.newton_schulz(u.const_data_ptr(), dt, (int)batch, (int)m, (int)n, u.stride(0), u.stride(1), table.data(), (int)steps, (float)eps, out.data_ptr(), ws.at, need,
                          call.stream()), "sgpo_newton_schulz");
  return out;
}

void muon_step(const Tensor& weight, const Tensor& grad, const Tensor& buffer, double lr, double momentum, bool nesterov, double weight_decay, int64_t steps,
               const std::vector<float>& table, double eps) {
  for (const Tensor* t : {&weight, &buffer})
    REQUIRE(!records({t}) || t->is_leaf(), "weight or momentum_buffer is part of a graph: a step updates leaves");
  no_tangents({&weight, &grad, &buffer}, "muon_step");
  const Call call({&weight, &grad, &buffer});
  const int wd = dtype_of(weight, "weight"), gd = dtype_of(grad, "grad");
  REQUIRE(weight.dim() >= 2 && weight.sizes() == grad.sizes() && weight.sizes() == buffer.sizes(), "weight ", weight.sizes(), ", grad ", grad.sizes(), " and buffer ", buffer.sizes(),
          " must agree");
  REQUIRE(buffer.scalar_type() == at::kFloat, "momentum_buffer must be float32");
  REQUIRE(weight.is_contiguous() && buffer.is_contiguous(), "weight and momentum_buffer are updated in place and must be contiguous");
  check_table(table, steps);
  if (!weight.numel()) return;
  at::AutoGradMode off(false);
  const Tensor g = grad.contiguous();
  const int64_t m = weight.size(-2), n = weight.size(-1), batch = weight.numel() / (m * n);
  REQUIRE(m < INT_MAX && n < INT_MAX && batch < INT_MAX, "weights ", weight.sizes(), " over the supported range");
  const size_t need = lib.ns_bytes((int)batch, (int)m, (int)n);
  const Scratch ws(need, call.dev);
  check(lib.muon_step(weight.data_ptr(), wd, g.const_data_ptr(), gd, buffer.data_ptr<float>(), (int)batch, (int)m, (int)n, (float)lr, (float)momentum, nesterov, (float)weight_decay,
                      table.data(), (int)steps, (float)eps, ws.at, need, call.stream()), "sgpo_muon_step");
  // what autograd saved of them is stale now
  if (!weight.is_inference()) weight.unsafeGetTensorImpl()->bump_version();
  if (!buffer.is_inference()) buffer.unsafeGetTensorImpl()->bump_version();
}

template <typename F>
void take(F& f, const std::map<std::string, uintptr_t>& from, const char* name) {
  f = reinterpret_cast<F>(from.at(name));
}

}  // namespace

PYBIND11_MODULE(_sgpo_torch, m) {
  m.def("bind", [](const std::map<std::string, uintptr_t>& from, pybind11::object error) {
    take(lib.init, from, "sgpo_init");
    take(lib.last_error, from, "sgpo_last_error");
    take(lib.rotary, from, "sgpo_rotary");
    take(lib.ce_bytes, from, "sgpo_linear_ce_workspace_bytes");
    take(lib.ce_forward, from, "sgpo_linear_ce_forward");
    take(lib.ce_backward, from, "sgpo_linear_ce_backward");
    take(lib.ns_bytes, from, "sgpo_newton_schulz_workspace_bytes");
    take(lib.newton_schulz, from, "sgpo_newton_schulz");
    take(lib.muon_step, from, "sgpo_muon_step");
    static pybind11::handle raised;
    raised = error.release();   // lives as long as the process
    pybind11::register_exception_translator([](std::exception_ptr p) {
      try {
        if (p) std::rethrow_exception(p);
      } catch (const Refused& e) {
        PyErr_SetString(raised.ptr(), e.what());
      }
    });
  });
  m.def("rotary_positions", &rotary_positions);
  m.def("rotary_positions_", &rotary_positions_);
  m.def("linear_cross_entropy", &linear_cross_entropy);
  m.def("newton_schulz", &newton_schulz);
  m.def("muon_step", &muon_step);
}
